// dropout.cu -- dropout whose mask is a function of (seed, offset, element) and is never stored.
//
// Element i takes word i mod 4 of the Philox4x32-10 block (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011) with the 64-bit counter offset + i / 4 (high counter
// words 0) and the 64-bit key seed. It is kept iff that word is at least p * 2^32 (rounded), so
// the mask is exact integer arithmetic: the backward pass calls the same function on the gradient
// and draws the same mask. A dropped element contributes exactly 0, also where x is Inf or NaN.
#include "layers.cuh"

#include <cmath>

namespace xspmm_b200 {
namespace {

constexpr int DROP_THREADS = 256;

__device__ __forceinline__ uint4 philox(uint64_t counter, uint2 key) {
    uint4 c = make_uint4((uint32_t)counter, (uint32_t)(counter >> 32), 0u, 0u);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ key.x, (uint32_t)p1,
                       (uint32_t)(p0 >> 32) ^ c.w ^ key.y, (uint32_t)p0);
        key.x += 0x9E3779B9u;
        key.y += 0xBB67AE85u;
    }
    return c;
}

template <typename T, bool RES>
__global__ void __launch_bounds__(DROP_THREADS)
dropout_kernel(int64_t n, const T* x, const T* res, uint32_t threshold, bool drop_all, float scale,
               uint2 key, uint64_t offset, T* y) {
    const int64_t blocks = (n + 3) / 4;
    for (int64_t b = (int64_t)blockIdx.x * DROP_THREADS + threadIdx.x; b < blocks;
         b += (int64_t)gridDim.x * DROP_THREADS) {
        const uint4 w = philox(offset + (uint64_t)b, key);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = b * 4 + j;
            if (i >= n) break;
            const bool keep = ws[j] >= threshold && !drop_all;
            float v = keep ? to_float(x[i]) * scale : 0.0f;
            if (RES) v += to_float(res[i]);
            y[i] = from_float<T>(v);
        }
    }
}

}  // namespace

template <typename T>
void dropout(Handle& h, int64_t n, const T* x, const T* residual, double p, uint64_t seed,
             uint64_t offset, T* y) {
    if (n == 0) return;
    // keep iff word >= threshold; p = 1 gives 2^32, which no word reaches
    const uint64_t threshold = (uint64_t)std::nearbyint(p * 4294967296.0);
    const bool all = threshold > 0xFFFFFFFFull;
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const unsigned grid = (unsigned)std::min(ceil_div(ceil_div(n, 4), DROP_THREADS),
                                             (int64_t)sm_count(h.device) * 8);
    if (residual)
        dropout_kernel<T, true><<<grid, DROP_THREADS, 0, h.stream>>>(
            n, x, residual, (uint32_t)threshold, all, scale, key, offset, y);
    else
        dropout_kernel<T, false><<<grid, DROP_THREADS, 0, h.stream>>>(
            n, x, nullptr, (uint32_t)threshold, all, scale, key, offset, y);
    after_launch(h, "dropout");
}

template void dropout<__half>(Handle&, int64_t, const __half*, const __half*, double, uint64_t,
                              uint64_t, __half*);
template void dropout<__nv_bfloat16>(Handle&, int64_t, const __nv_bfloat16*, const __nv_bfloat16*,
                                     double, uint64_t, uint64_t, __nv_bfloat16*);
template void dropout<float>(Handle&, int64_t, const float*, const float*, double, uint64_t,
                             uint64_t, float*);

}  // namespace xspmm_b200
