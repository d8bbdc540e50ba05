// capi_layers.cu -- extern "C" entry points of the layer operators (include/xspmm_b200.h): layer
// norm, dropout, gated feed-forward. Validates arguments; the kernels see only valid ones.
#include "layers.cuh"

#include <cmath>

using namespace xspmm_b200;

namespace {

// A matrix argument: present (unless it has no elements), aligned to its type, rows apart.
template <typename T>
const T* matrix(const void* p, int64_t rows, int64_t cols, int64_t ld, const char* name) {
    need(ld >= cols, (std::string("row stride of ") + name + " smaller than its columns").c_str());
    need(rows == 0 || ld <= INT64_MAX / (int64_t)sizeof(T) / rows,
         (std::string(name) + " too large").c_str());
    need(p != nullptr || rows == 0 || cols == 0, (std::string("null ") + name).c_str());
    need(aligned_to(p, sizeof(T)), (std::string(name) + " not aligned to its type").c_str());
    return static_cast<const T*>(p);
}
template <typename T>
T* out_matrix(void* p, int64_t rows, int64_t cols, int64_t ld, const char* name) {
    return const_cast<T*>(matrix<T>(p, rows, cols, ld, name));
}
const float* vec(const float* p, const char* name) {
    need(aligned_to(p, sizeof(float)), (std::string(name) + " not aligned to its type").c_str());
    return p;
}

template <typename T>
GatedArgs<T> gated_args(int64_t rows, int64_t K, int64_t F, int act, const void* x, int64_t ldx,
                        const void* wg, int64_t ldwg, const void* wu, int64_t ldwu) {
    need(rows >= 0 && K >= 0 && F >= 0, "negative dimension");
    need(act >= XSPMM_ACT_SILU && act <= XSPMM_ACT_SIGMOID, "unknown activation");
    return GatedArgs<T>{rows, K, F, static_cast<Activation>(act),
                        matrix<T>(x, rows, K, ldx, "x"), ldx,
                        matrix<T>(wg, F, K, ldwg, "w_gate"), ldwg,
                        matrix<T>(wu, F, K, ldwu, "w_up"), ldwu};
}

}  // namespace

#define XS_LAYER_NORM(SUF, TX, TY)                                                                \
    XS_API xspmm_status_t xspmm_layer_norm_##SUF(                                                 \
        xspmm_handle_t hh, int64_t rows, int64_t D, const void* x, int64_t ldx, const float* w,   \
        const float* b, float eps, void* y, int64_t ldy, float* mean, float* rstd) {              \
        return guarded([&] {                                                                      \
            Handle& h = H(hh);                                                                    \
            need(rows >= 0 && D >= 1, "rows must be non-negative and cols positive");             \
            need(std::isfinite(eps) && eps >= 0.0f, "eps must be finite and non-negative");       \
            const TX* px = matrix<TX>(x, rows, D, ldx, "x");                                      \
            TY* py = out_matrix<TY>(y, rows, D, ldy, "y");                                        \
            vec(w, "weight"), vec(b, "bias"), vec(mean, "mean"), vec(rstd, "rstd");               \
            DeviceGuard g(h.device);                                                              \
            layer_norm<TX, TY>(h, rows, D, px, ldx, w, b, eps, py, ldy, mean, rstd);              \
        });                                                                                       \
    }                                                                                             \
    XS_API xspmm_status_t xspmm_layer_norm_backward_##SUF(                                        \
        xspmm_handle_t hh, int64_t rows, int64_t D, const void* dy, int64_t lddy, const void* x,  \
        int64_t ldx, const float* w, const float* mean, const float* rstd, void* dx,              \
        int64_t lddx, float* dw, float* db) {                                                     \
        return guarded([&] {                                                                      \
            Handle& h = H(hh);                                                                    \
            need(rows >= 0 && D >= 1, "rows must be non-negative and cols positive");             \
            const TY* pdy = matrix<TY>(dy, rows, D, lddy, "dy");                                  \
            const TX* px = matrix<TX>(x, rows, D, ldx, "x");                                      \
            need(rows == 0 || (mean && rstd), "null mean or rstd");                               \
            TY* pdx = dx ? out_matrix<TY>(dx, rows, D, lddx, "dx") : nullptr;                     \
            vec(w, "weight"), vec(mean, "mean"), vec(rstd, "rstd"), vec(dw, "dweight"),           \
                vec(db, "dbias");                                                                 \
            DeviceGuard g(h.device);                                                              \
            layer_norm_backward<TX, TY>(h, rows, D, pdy, lddy, px, ldx, w, mean, rstd, pdx, lddx, \
                                        dw, db);                                                  \
        });                                                                                       \
    }
XS_LAYER_NORM(f16f16, __half, __half)
XS_LAYER_NORM(bf16bf16, __nv_bfloat16, __nv_bfloat16)
XS_LAYER_NORM(f32f32, float, float)
XS_LAYER_NORM(f32f16, float, __half)
XS_LAYER_NORM(f32bf16, float, __nv_bfloat16)

#define XS_DROPOUT(SUF, T)                                                                        \
    XS_API xspmm_status_t xspmm_dropout_##SUF(xspmm_handle_t hh, int64_t n, const void* x,        \
                                              const void* residual, double p, uint64_t seed,      \
                                              uint64_t offset, void* y) {                         \
        return guarded([&] {                                                                      \
            Handle& h = H(hh);                                                                    \
            need(n >= 0, "negative dimension");                                                   \
            need(p >= 0.0 && p <= 1.0, "p must lie in [0, 1]");                                   \
            const T* px = matrix<T>(x, 1, n, n, "x");                                             \
            T* py = out_matrix<T>(y, 1, n, n, "y");                                               \
            const T* pr = residual ? matrix<T>(residual, 1, n, n, "residual") : nullptr;          \
            DeviceGuard g(h.device);                                                              \
            dropout<T>(h, n, px, pr, p, seed, offset, py);                                        \
        });                                                                                       \
    }
XS_DROPOUT(f16, __half)
XS_DROPOUT(bf16, __nv_bfloat16)
XS_DROPOUT(f32, float)

#define XS_GATED_FFN(SUF, T)                                                                      \
    XS_API xspmm_status_t xspmm_gated_ffn_##SUF(                                                  \
        xspmm_handle_t hh, int64_t rows, int64_t K, int64_t F, int act, const void* x,            \
        int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu, void* y,         \
        int64_t ldy, void* gate, void* up) {                                                      \
        return guarded([&] {                                                                      \
            Handle& h = H(hh);                                                                    \
            const GatedArgs<T> a = gated_args<T>(rows, K, F, act, x, ldx, wg, ldwg, wu, ldwu);    \
            T* py = out_matrix<T>(y, rows, F, ldy, "y");                                          \
            T* pg = gate ? out_matrix<T>(gate, rows, F, F, "gate") : nullptr;                     \
            T* pu = up ? out_matrix<T>(up, rows, F, F, "up") : nullptr;                           \
            DeviceGuard g(h.device);                                                              \
            gated_ffn<T>(h, a, py, ldy, pg, pu);                                                  \
        });                                                                                       \
    }                                                                                             \
    XS_API xspmm_status_t xspmm_gated_ffn_backward_##SUF(                                         \
        xspmm_handle_t hh, int64_t rows, int64_t K, int64_t F, int act, const void* dy,           \
        int64_t lddy, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,   \
        int64_t ldwu, const void* gate, const void* up, void* dx, int64_t lddx, void* dwg,        \
        void* dwu) {                                                                              \
        return guarded([&] {                                                                      \
            Handle& h = H(hh);                                                                    \
            const GatedArgs<T> a = gated_args<T>(rows, K, F, act, x, ldx, wg, ldwg, wu, ldwu);    \
            const T* pdy = matrix<T>(dy, rows, F, lddy, "dy");                                    \
            const T* pg = matrix<T>(gate, rows, F, F, "gate");                                    \
            const T* pu = matrix<T>(up, rows, F, F, "up");                                        \
            T* pdx = dx ? out_matrix<T>(dx, rows, K, lddx, "dx") : nullptr;                       \
            need((dwg == nullptr) == (dwu == nullptr),                                            \
                 "dw_gate and dw_up are wanted both or neither");                                 \
            T* pdwg = dwg ? out_matrix<T>(dwg, F, K, K, "dw_gate") : nullptr;                     \
            T* pdwu = dwu ? out_matrix<T>(dwu, F, K, K, "dw_up") : nullptr;                       \
            DeviceGuard g(h.device);                                                              \
            gated_ffn_backward<T>(h, a, pdy, lddy, pg, pu, pdx, lddx, pdwg, pdwu);                \
        });                                                                                       \
    }
XS_GATED_FFN(f16, __half)
XS_GATED_FFN(bf16, __nv_bfloat16)
