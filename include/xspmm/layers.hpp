// xspmm/layers.hpp -- the operators of the layer around the sparse product, over the C ABI: layer norm,
// dropout and the gated feed-forward block, each with its gradient (xspmm_layer_norm_*, xspmm_dropout_*,
// xspmm_gated_ffn_* in include/xspmm_b200.h, which states what each computes). The reference has none.
//
// Rows are nodes or tokens, features are contiguous; a Rows<T> is a device matrix with its row stride in
// elements. Calls enqueue on the executor's stream and throw as the other calls do.
#pragma once

#include <cstdint>
#include <memory>

#include "core/executor.hpp"
#include "detail/abi.hpp"

namespace xspmm {

enum class Activation { Silu = XSPMM_ACT_SILU, Gelu = XSPMM_ACT_GELU, Relu = XSPMM_ACT_RELU, Sigmoid = XSPMM_ACT_SIGMOID };

template <typename T>
struct Rows {
    T* data = nullptr;
    int64_t ld = 0;
};

namespace detail {

template <typename X, typename Y>
struct NormAbi;
#define XSPMM_NORM_ROW(X, Y, S)                                                  \
    template <>                                                                  \
    struct NormAbi<X, Y> {                                                       \
        static constexpr auto forward = xspmm_layer_norm_##S;                    \
        static constexpr auto backward = xspmm_layer_norm_backward_##S;          \
    };
XSPMM_NORM_ROW(__half, __half, f16f16)
XSPMM_NORM_ROW(__nv_bfloat16, __nv_bfloat16, bf16bf16)
XSPMM_NORM_ROW(float, float, f32f32)
XSPMM_NORM_ROW(float, __half, f32f16)
XSPMM_NORM_ROW(float, __nv_bfloat16, f32bf16)
#undef XSPMM_NORM_ROW

template <typename T>
struct DropoutAbi;
template <> struct DropoutAbi<__half> { static constexpr auto call = xspmm_dropout_f16; };
template <> struct DropoutAbi<__nv_bfloat16> { static constexpr auto call = xspmm_dropout_bf16; };
template <> struct DropoutAbi<float> { static constexpr auto call = xspmm_dropout_f32; };

template <typename T>
struct GatedAbi;
template <> struct GatedAbi<__half> {
    static constexpr auto forward = xspmm_gated_ffn_f16;
    static constexpr auto backward = xspmm_gated_ffn_backward_f16;
};
template <> struct GatedAbi<__nv_bfloat16> {
    static constexpr auto forward = xspmm_gated_ffn_bf16;
    static constexpr auto backward = xspmm_gated_ffn_backward_bf16;
};

}  // namespace detail

// y = (x - mean) * rstd * weight + bias over each row. weight, bias, mean, rstd may be null.
template <typename X, typename Y>
void layer_norm(std::shared_ptr<const Executor> exec, int64_t rows, int64_t cols, Rows<const X> x,
                const float* weight, const float* bias, float eps, Rows<Y> y, float* mean = nullptr,
                float* rstd = nullptr) {
    detail::check(detail::NormAbi<X, Y>::forward(detail::handle_of(exec), rows, cols, x.data, x.ld, weight,
                                                 bias, eps, y.data, y.ld, mean, rstd));
}

// Gradients of layer_norm; outputs that are null are not computed.
template <typename X, typename Y>
void layer_norm_backward(std::shared_ptr<const Executor> exec, int64_t rows, int64_t cols,
                         Rows<const Y> dy, Rows<const X> x, const float* weight, const float* mean,
                         const float* rstd, Rows<Y> dx, float* dweight, float* dbias) {
    detail::check(detail::NormAbi<X, Y>::backward(detail::handle_of(exec), rows, cols, dy.data, dy.ld,
                                                  x.data, x.ld, weight, mean, rstd, dx.data, dx.ld,
                                                  dweight, dbias));
}

// y = residual + keep * x / (1 - p); residual may be null. The gradient is the same call on dy without it.
template <typename T>
void dropout(std::shared_ptr<const Executor> exec, int64_t n, const T* x, const T* residual, double p,
             uint64_t seed, uint64_t offset, T* y) {
    detail::check(detail::DropoutAbi<T>::call(detail::handle_of(exec), n, x, residual, p, seed, offset, y));
}

// y = act(x w_gate^T) * (x w_up^T); gate and up (rows x F, contiguous) receive the projections if not null.
template <typename T>
void gated_ffn(std::shared_ptr<const Executor> exec, int64_t rows, int64_t K, int64_t F, Activation act,
               Rows<const T> x, Rows<const T> w_gate, Rows<const T> w_up, Rows<T> y, T* gate = nullptr,
               T* up = nullptr) {
    detail::check(detail::GatedAbi<T>::forward(detail::handle_of(exec), rows, K, F, static_cast<int>(act),
                                               x.data, x.ld, w_gate.data, w_gate.ld, w_up.data, w_up.ld,
                                               y.data, y.ld, gate, up));
}

// Gradients of gated_ffn from the kept projections. dx may be null; dw_gate and dw_up both, too.
template <typename T>
void gated_ffn_backward(std::shared_ptr<const Executor> exec, int64_t rows, int64_t K, int64_t F,
                        Activation act, Rows<const T> dy, Rows<const T> x, Rows<const T> w_gate,
                        Rows<const T> w_up, const T* gate, const T* up, Rows<T> dx, T* dw_gate, T* dw_up) {
    detail::check(detail::GatedAbi<T>::backward(detail::handle_of(exec), rows, K, F, static_cast<int>(act),
                                                dy.data, dy.ld, x.data, x.ld, w_gate.data, w_gate.ld,
                                                w_up.data, w_up.ld, gate, up, dx.data, dx.ld, dw_gate, dw_up));
}

}  // namespace xspmm
