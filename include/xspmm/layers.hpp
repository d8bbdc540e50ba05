// xspmm/layers.hpp -- the operators of the layer around the sparse product, over the C ABI: layer norm,
// group norm, dropout and the gated feed-forward block, each with its gradient, 8-bit rows and their product,
// and the orthogonalised update of a weight (xspmm_layer_norm_*, xspmm_group_norm_*, xspmm_dropout_*,
// xspmm_gated_ffn_*, xspmm_quantize_rows_*, xspmm_linear_int8_*, xspmm_orthogonalize_* in
// include/xspmm_b200.h, which states what each computes). The reference has none.
//
// Rows are nodes or tokens, features are contiguous; a Rows<T> is a device matrix with its row stride in
// elements. Calls enqueue on the executor's stream and throw as the other calls do.
#pragma once

#include <cstdint>
#include <memory>

#include "core/executor.hpp"
#include "detail/abi.hpp"

namespace xspmm {

enum class Activation { Silu = XSPMM_ACT_SILU, Gelu = XSPMM_ACT_GELU, Relu = XSPMM_ACT_RELU, Sigmoid = XSPMM_ACT_SIGMOID, None = XSPMM_ACT_NONE };

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
        static constexpr auto group_forward = xspmm_group_norm_##S;              \
        static constexpr auto group_backward = xspmm_group_norm_backward_##S;    \
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

template <typename T>
struct Int8Abi;
template <> struct Int8Abi<__half> {
    static constexpr auto quantize = xspmm_quantize_rows_f16;
    static constexpr auto linear = xspmm_linear_int8_f16;
};
template <> struct Int8Abi<__nv_bfloat16> {
    static constexpr auto quantize = xspmm_quantize_rows_bf16;
    static constexpr auto linear = xspmm_linear_int8_bf16;
};
template <> struct Int8Abi<float> {
    static constexpr auto quantize = xspmm_quantize_rows_f32;
    static constexpr auto linear = xspmm_linear_int8_f32;
};

template <typename X, typename Y>
struct UpdateAbi;
template <> struct UpdateAbi<__half, __half> { static constexpr auto call = xspmm_orthogonalize_f16f16; };
template <> struct UpdateAbi<__nv_bfloat16, __nv_bfloat16> { static constexpr auto call = xspmm_orthogonalize_bf16bf16; };
template <> struct UpdateAbi<float, __half> { static constexpr auto call = xspmm_orthogonalize_f32f16; };
template <> struct UpdateAbi<float, __nv_bfloat16> { static constexpr auto call = xspmm_orthogonalize_f32bf16; };

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

// A packed batch for the group norm: sample i is rows [offsets[i], offsets[i + 1]) (device, samples + 1).
// The default is one sample of all rows.
struct Samples {
    int64_t count = 1;
    const int64_t* offsets = nullptr;
};

// y = act((x - mean) * rstd * weight + bias) over each sample's rows and group of neighbouring channels.
// weight, bias, mean, rstd may be null.
template <typename X, typename Y>
void group_norm(std::shared_ptr<const Executor> exec, int64_t rows, int64_t cols, int64_t groups, Samples samples,
                Rows<const X> x, const float* weight, const float* bias, float eps, Activation act, Rows<Y> y,
                float* mean = nullptr, float* rstd = nullptr) {
    detail::check(detail::NormAbi<X, Y>::group_forward(detail::handle_of(exec), rows, cols, groups, samples.count,
                                                       samples.offsets, x.data, x.ld, weight, bias, eps,
                                                       static_cast<int>(act), y.data, y.ld, mean, rstd));
}

// Gradients of group_norm; outputs that are null are not computed.
template <typename X, typename Y>
void group_norm_backward(std::shared_ptr<const Executor> exec, int64_t rows, int64_t cols, int64_t groups,
                         Samples samples, Rows<const Y> dy, Rows<const X> x, const float* weight, const float* bias,
                         const float* mean, const float* rstd, Activation act, Rows<Y> dx, float* dweight,
                         float* dbias) {
    detail::check(detail::NormAbi<X, Y>::group_backward(detail::handle_of(exec), rows, cols, groups, samples.count,
                                                        samples.offsets, dy.data, dy.ld, x.data, x.ld, weight, bias,
                                                        mean, rstd, static_cast<int>(act), dx.data, dx.ld, dweight,
                                                        dbias));
}

// Rows of x as 8-bit integers q with a scale each.
template <typename T>
void quantize_rows(std::shared_ptr<const Executor> exec, int64_t rows, int64_t cols, Rows<const T> x, Rows<int8_t> q,
                   float* scale) {
    detail::check(detail::Int8Abi<T>::quantize(detail::handle_of(exec), rows, cols, x.data, x.ld, q.data, q.ld, scale));
}

// y = x_scale * w_scale * (x w^T) + bias of 8-bit x (rows x K) and w (F x K); bias may be null.
template <typename T>
void linear_int8(std::shared_ptr<const Executor> exec, int64_t rows, int64_t K, int64_t F, Rows<const int8_t> x,
                 const float* x_scale, Rows<const int8_t> w, const float* w_scale, Rows<T> y,
                 const float* bias = nullptr) {
    detail::check(detail::Int8Abi<T>::linear(detail::handle_of(exec), rows, K, F, x.data, x.ld, x_scale, w.data, w.ld,
                                             w_scale, bias, y.data, y.ld));
}

// The orthogonalised update y of a weight matrix from its gradient or momentum g.
template <typename X, typename Y>
void orthogonalize(std::shared_ptr<const Executor> exec, int64_t rows, int64_t cols, Rows<const X> g, Rows<Y> y,
                   int steps = 5, float eps = 1e-7f) {
    detail::check(detail::UpdateAbi<X, Y>::call(detail::handle_of(exec), rows, cols, g.data, g.ld, steps, eps, y.data,
                                                y.ld));
}

}  // namespace xspmm
