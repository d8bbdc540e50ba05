// int8.cu -- rows in 8-bit integers with a scale each, and their product.
//
// Quantisation: scale = max|x| / 127, q = 127 x / max|x| rounded to the nearest whole number, ties to even, of
// the exact quotient. Product: y[r, f] = xs[r] * ws[f] * sum_k x[r, k] w[f, k] + bias[f], the sum exact in 32 bits.
#include "layers.cuh"

namespace xspmm_b200 {
namespace {

constexpr int Q_THREADS = 256;

// 127 v / most rounded to the nearest, ties to even. inv = 127 / most in fp32 puts the quotient within 2^-22 of
// itself, so only a product that close to a border can be on its wrong side; those are compared exactly in 64
// bits (127 v has 31 bits, (2 q + 1) most has 32). inv is infinite for the smallest subnormal `most`: 64 bits.
__device__ __forceinline__ int quantized(float v, float most, float inv) {
    const float p = v * inv, q = rintf(p);
    if (fabsf(fabsf(p - q) - 0.5f) > 1e-4f && fabsf(p) < 256.0f) return (int)q;
    return (int)rint(127.0 * (double)v / (double)most);
}

// A CTA per row.
template <typename T>
__global__ void __launch_bounds__(Q_THREADS)
quantize_kernel(int64_t cols, const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq, float* scale) {
    __shared__ float part[Q_THREADS / 32];
    __shared__ int odd;
    const int64_t r = blockIdx.x;
    if (threadIdx.x == 0) odd = 0;
    __syncthreads();
    float most = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += Q_THREADS) {
        const float v = fabsf(to_float(x[r * ldx + c]));
        if (!(v < INFINITY)) odd = 1;
        most = fmaxf(most, v);
    }
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
    __syncthreads();
    most = part[0];
    for (int i = 1; i < Q_THREADS / 32; ++i) most = fmaxf(most, part[i]);
    const bool zero = odd || most == 0.0f;
    const float inv = 127.0f / most;
    for (int64_t c = threadIdx.x; c < cols; c += Q_THREADS)
        q[r * ldq + c] = zero ? (int8_t)0 : (int8_t)quantized(to_float(x[r * ldx + c]), most, inv);
    if (threadIdx.x == 0) scale[r] = odd ? NAN : most / 127.0f;
}

// 16 x 16 outputs a CTA, one a thread.
template <typename T>
__global__ void __launch_bounds__(256) linear_int8_kernel(const Int8Args a, T* y, int64_t ldy) {
    __shared__ int8_t xs[16][65], ws[16][65];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t nf = (a.F + 15) / 16, r0 = blockIdx.x / nf * 16, f0 = blockIdx.x % nf * 16;
    int sum = 0;
    for (int64_t k0 = 0; k0 < a.K; k0 += 64) {
        for (int i = threadIdx.x; i < 16 * 64; i += 256) {
            const int64_t r = r0 + i / 64, f = f0 + i / 64, k = k0 + i % 64;
            xs[i / 64][i % 64] = r < a.rows && k < a.K ? a.x[r * a.ldx + k] : (int8_t)0;
            ws[i / 64][i % 64] = f < a.F && k < a.K ? a.w[f * a.ldw + k] : (int8_t)0;
        }
        __syncthreads();
        for (int k = 0; k < 64; ++k) sum += (int)xs[ty][k] * (int)ws[tx][k];
        __syncthreads();
    }
    const int64_t r = r0 + ty, f = f0 + tx;
    if (r < a.rows && f < a.F)
        y[r * ldy + f] = from_float<T>((float)sum * a.xs[r] * a.ws[f] + (a.bias ? a.bias[f] : 0.0f));
}

}  // namespace

template <typename T>
void quantize_rows(Handle& h, int64_t rows, int64_t cols, const T* x, int64_t ldx, int8_t* q, int64_t ldq,
                   float* scale) {
    if (rows == 0) return;
    XS_REQUIRE(rows < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "rows pass 2^31");
    quantize_kernel<T><<<(unsigned)rows, Q_THREADS, 0, h.stream>>>(cols, x, ldx, q, ldq, scale);
    after_launch(h, "quantize_rows");
}

template <typename T>
void linear_int8(Handle& h, const Int8Args& a, T* y, int64_t ldy) {
    if (a.rows == 0 || a.F == 0) return;
    const int64_t tiles = ceil_div(a.rows, 16) * ceil_div(a.F, 16);
    XS_REQUIRE(tiles < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "grid too large");
    linear_int8_kernel<T><<<(unsigned)tiles, 256, 0, h.stream>>>(a, y, ldy);
    after_launch(h, "linear_int8");
}

#define XS_INST_INT8(T)                                                                                        \
    template void quantize_rows<T>(Handle&, int64_t, int64_t, const T*, int64_t, int8_t*, int64_t, float*);     \
    template void linear_int8<T>(Handle&, const Int8Args&, T*, int64_t);
XS_INST_INT8(__half)
XS_INST_INT8(__nv_bfloat16)
XS_INST_INT8(float)

}  // namespace xspmm_b200
