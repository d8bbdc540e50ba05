// layer_norm.cu -- layer norm over the features of each row, forward and backward.
//
// Forward: mean = sum(x) / D, var = sum((x - mean)^2) / D, rstd = 1 / sqrt(var + eps),
// y = (x - mean) * rstd * w + b. Backward, with xh = (x - mean) * rstd and t = dy * w:
// dx = rstd * (t - mean(t) - xh * mean(t * xh)), dw = sum over rows of dy * xh, db = sum of dy.
// Every sum is held in fp32 in an order fixed by the sizes alone.
#include "layers.cuh"

namespace xspmm_b200 {
namespace {

constexpr int LN_THREADS = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < LN_THREADS / 32; ++w) s += red[w];
    return s;
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(LN_THREADS)
layer_norm_kernel(int64_t rows, int64_t D, const TX* x, int64_t ldx, const float* w, const float* b,
                  float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    __shared__ float red[LN_THREADS / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const TX* xr = x + r * ldx;
        float s = 0.0f;
        for (int64_t c = threadIdx.x; c < D; c += LN_THREADS) s += to_float(xr[c]);
        const float m = block_sum(s, red) / (float)D;
        float q = 0.0f;
        for (int64_t c = threadIdx.x; c < D; c += LN_THREADS) {
            const float d = to_float(xr[c]) - m;
            q += d * d;
        }
        const float rs = 1.0f / sqrtf(block_sum(q, red) / (float)D + eps);
        for (int64_t c = threadIdx.x; c < D; c += LN_THREADS) {
            const float xh = (to_float(xr[c]) - m) * rs;
            y[r * ldy + c] = from_float<TY>(xh * (w ? w[c] : 1.0f) + (b ? b[c] : 0.0f));
        }
        if (threadIdx.x == 0) {
            if (mean) mean[r] = m;
            if (rstd) rstd[r] = rs;
        }
    }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(LN_THREADS)
layer_norm_dx_kernel(int64_t rows, int64_t D, const TY* dy, int64_t lddy, const TX* x, int64_t ldx,
                     const float* w, const float* mean, const float* rstd, TY* dx, int64_t lddx) {
    __shared__ float red[LN_THREADS / 32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float m = mean[r], rs = rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = threadIdx.x; c < D; c += LN_THREADS) {
            const float t = to_float(dy[r * lddy + c]) * (w ? w[c] : 1.0f);
            s1 += t;
            s2 += t * ((to_float(x[r * ldx + c]) - m) * rs);
        }
        const float c1 = block_sum(s1, red) / (float)D, c2 = block_sum(s2, red) / (float)D;
        for (int64_t c = threadIdx.x; c < D; c += LN_THREADS) {
            const float t = to_float(dy[r * lddy + c]) * (w ? w[c] : 1.0f);
            const float xh = (to_float(x[r * ldx + c]) - m) * rs;
            dx[r * lddx + c] = from_float<TY>(rs * (t - c1 - xh * c2));
        }
    }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(LN_THREADS)
layer_norm_dw_kernel(int64_t rows, int64_t D, const TY* dy, int64_t lddy, const TX* x, int64_t ldx,
                     const float* mean, const float* rstd, float* dw, float* db) {
    __shared__ float red[LN_THREADS / 32];
    for (int64_t c = blockIdx.x; c < D; c += gridDim.x) {
        float sw = 0.0f, sb = 0.0f;
        for (int64_t r = threadIdx.x; r < rows; r += LN_THREADS) {
            const float g = to_float(dy[r * lddy + c]);
            sw += g * ((to_float(x[r * ldx + c]) - mean[r]) * rstd[r]);
            sb += g;
        }
        sw = block_sum(sw, red);
        sb = block_sum(sb, red);
        if (threadIdx.x == 0) {
            if (dw) dw[c] = sw;
            if (db) db[c] = sb;
        }
    }
}

unsigned ln_grid(Handle& h, int64_t n) {
    return (unsigned)std::min(n, (int64_t)sm_count(h.device) * 8);
}

}  // namespace

template <typename TX, typename TY>
void layer_norm(Handle& h, int64_t rows, int64_t D, const TX* x, int64_t ldx, const float* w,
                const float* b, float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    if (rows == 0) return;
    layer_norm_kernel<TX, TY><<<ln_grid(h, rows), LN_THREADS, 0, h.stream>>>(
        rows, D, x, ldx, w, b, eps, y, ldy, mean, rstd);
    after_launch(h, "layer_norm");
}

template <typename TX, typename TY>
void layer_norm_backward(Handle& h, int64_t rows, int64_t D, const TY* dy, int64_t lddy,
                         const TX* x, int64_t ldx, const float* w, const float* mean,
                         const float* rstd, TY* dx, int64_t lddx, float* dw, float* db) {
    if (dx && rows > 0) {
        layer_norm_dx_kernel<TX, TY><<<ln_grid(h, rows), LN_THREADS, 0, h.stream>>>(
            rows, D, dy, lddy, x, ldx, w, mean, rstd, dx, lddx);
        after_launch(h, "layer_norm_dx");
    }
    if (dw || db) {
        layer_norm_dw_kernel<TX, TY><<<ln_grid(h, D), LN_THREADS, 0, h.stream>>>(
            rows, D, dy, lddy, x, ldx, mean, rstd, dw, db);
        after_launch(h, "layer_norm_dw");
    }
}

#define XS_INST_LN(TX, TY)                                                                        \
    template void layer_norm<TX, TY>(Handle&, int64_t, int64_t, const TX*, int64_t, const float*, \
                                     const float*, float, TY*, int64_t, float*, float*);          \
    template void layer_norm_backward<TX, TY>(Handle&, int64_t, int64_t, const TY*, int64_t,      \
                                              const TX*, int64_t, const float*, const float*,     \
                                              const float*, TY*, int64_t, float*, float*);
XS_INST_LN(__half, __half)
XS_INST_LN(__nv_bfloat16, __nv_bfloat16)
XS_INST_LN(float, float)
XS_INST_LN(float, __half)
XS_INST_LN(float, __nv_bfloat16)

}  // namespace xspmm_b200
