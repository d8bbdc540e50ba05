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

constexpr int DROP_THREADS = 128;

struct Keys {  // the key of each round: multiples of two constants added to the seed's halves
    uint32_t k0[10], k1[10];
};

__device__ __forceinline__ uint4 philox(uint64_t counter, const Keys& key) {
    uint4 c = make_uint4((uint32_t)counter, (uint32_t)(counter >> 32), 0u, 0u);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ key.k0[r], (uint32_t)p1,
                       (uint32_t)(p0 >> 32) ^ c.w ^ key.k1[r], (uint32_t)p0);
    }
    return c;
}

// V elements (V / 4 generator blocks) a thread; VEC: the pointers allow V-wide accesses. An element is
// dropped iff its word is at most `last`; draw is false where p rounds to 0 and nothing is dropped.
template <typename T, int V, bool RES, bool VEC>
__global__ void __launch_bounds__(DROP_THREADS)
dropout_kernel(int64_t n, const T* x, const T* res, bool draw, uint32_t last, float scale,
               const __grid_constant__ Keys key, uint64_t offset, T* y) {
    const int64_t g = (int64_t)blockIdx.x * DROP_THREADS + threadIdx.x, first = g * V;
    cudaGridDependencySynchronize();
    if (first >= n) return;
    float v[V], r[V];
    const bool whole = VEC && first + V <= n;
    if (whole) {
        load_pack<T, V>(x + first, v);
        if (RES) load_pack<T, V>(res + first, r);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            v[e] = first + e < n ? to_float(x[first + e]) : 0.0f;
            if (RES) r[e] = first + e < n ? to_float(res[first + e]) : 0.0f;
        }
    }
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        uint4 w = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (draw) w = philox(offset + (uint64_t)(g * (V / 4) + q), key);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float t = !draw || ws[e] > last ? v[q * 4 + e] * scale : 0.0f;
            v[q * 4 + e] = RES ? r[q * 4 + e] + t : t;
        }
    }
    if (whole) {
        store_pack<T, V>(y + first, v);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (first + e < n) y[first + e] = from_float<T>(v[e]);
    }
}

}  // namespace

template <typename T>
void dropout(Handle& h, int64_t n, const T* x, const T* residual, double p, uint64_t seed,
             uint64_t offset, T* y) {
    if (n == 0) return;
    // kept iff word >= threshold, which is word > threshold - 1; p = 1 gives 2^32, which no word reaches
    const uint64_t threshold = (uint64_t)std::nearbyint(p * 4294967296.0);
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    Keys key;
    for (int r = 0; r < 10; ++r) {
        key.k0[r] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u;
        key.k1[r] = (uint32_t)(seed >> 32) + (uint32_t)r * 0xBB67AE85u;
    }
    // 16 bits: 16 elements a thread interleave four generator blocks, whose multiplications bound the kernel
    // (2^27 fp16 with residual: 146 us against 162 with 8). fp32: 4, where memory does (224 us; 289 with
    // 8). Unaligned pointers: 4, so that a warp's accesses of single elements stay close together.
    constexpr int V = sizeof(T) == 2 ? 16 : 4;
    const bool vec = aligned_to(x, 16) && aligned_to(y, 16) && aligned_to(residual, 16);
    const int64_t grid = ceil_div(ceil_div(n, vec ? V : 4), DROP_THREADS);
    XS_REQUIRE(grid < (int64_t(1) << 31), XSPMM_STATUS_UNSUPPORTED, "grid too large");
    auto kern = residual ? (vec ? dropout_kernel<T, V, true, true> : dropout_kernel<T, 4, true, false>)
                         : (vec ? dropout_kernel<T, V, false, true> : dropout_kernel<T, 4, false, false>);
    launch_dependent(h.stream, kern, (unsigned)grid, DROP_THREADS, 0, 1, n, x, residual, threshold > 0,
                     (uint32_t)(threshold - 1), scale, key, offset, y);
    after_launch(h, "dropout");
}

template void dropout<__half>(Handle&, int64_t, const __half*, const __half*, double, uint64_t,
                              uint64_t, __half*);
template void dropout<__nv_bfloat16>(Handle&, int64_t, const __nv_bfloat16*, const __nv_bfloat16*,
                                     double, uint64_t, uint64_t, __nv_bfloat16*);
template void dropout<float>(Handle&, int64_t, const float*, const float*, double, uint64_t,
                             uint64_t, float*);

}  // namespace xspmm_b200
