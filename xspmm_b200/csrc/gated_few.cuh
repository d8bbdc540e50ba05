// gated_few.cuh -- the forward pass of the gated feed-forward block for a few rows (decoding): bound by
// the bytes of the weights, each used once.
//
// A CTA takes 16 features of both projections, its four warps interleaved 64-element slices of the sum.
// The weights go from memory straight to registers as the A operand of mma.sync m16n8k16 (16 features;
// the tokens are the 8 columns), with no shared memory and no barrier until the end. The sum's order is
// free, so a lane loads 16 contiguous elements of a weight row (four lanes: a 128-byte line) and hands
// them to four MMAs as if they were the k positions the fragment layout asks for; x is loaded in the same
// order. The warps' partial sums are added in warp order. One row of 4096 x 11008, 180 MB of weights:
// 34 us (83 % of the copy bandwidth; the tensor-core tiles take 50); with eight warps a CTA, which do not
// all fit the GPU at once, 12 rows take 45 us instead of 36.
#pragma once

#include "gated_tc.cuh"
#include "mma_sync.cuh"

namespace xspmm_b200 {
namespace gated {

constexpr int FEW_WARPS = 4, FEW_CTAS = 5;  // CTAs an SM should hold: 102 registers a thread

// 16 elements of a row from column k on as 8 words; zeros from column K on. VEC: the row starts on 16
// bytes and K is a multiple of 8.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(uint32_t (&w)[8], const T* row, int64_t k, int64_t K, bool live) {
    if constexpr (VEC) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (live && k + 8 * h < K) v = __ldg(reinterpret_cast<const uint4*>(row + k + 8 * h));
            w[4 * h] = v.x; w[4 * h + 1] = v.y; w[4 * h + 2] = v.z; w[4 * h + 3] = v.w;
        }
    } else {
        const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t lo = live && k + 2 * e < K ? __ldg(r + k + 2 * e) : 0u;
            const uint32_t hi = live && k + 2 * e + 1 < K ? __ldg(r + k + 2 * e + 1) : 0u;
            w[e] = lo | hi << 16;
        }
    }
}

// NT: tokens by eights.
template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS, FEW_CTAS)
few_rows_kernel(const GatedArgs<T> p, T* y, int64_t ldy, T* gate, T* up) {
    __shared__ float red[FEW_WARPS][2][NT * 8][16];
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int64_t f0 = (int64_t)blockIdx.x * 16;
    cudaGridDependencySynchronize();
    const T* rows[2][2];  // a lane's two features of each weight; past the last: the last, not stored
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t f = min(f0 + g + 8 * h, p.F - 1);
        rows[0][h] = p.wg + f * p.ldwg;
        rows[1][h] = p.wu + f * p.ldwu;
    }
    float acc[2][NT][4] = {};
    const int64_t slices = (p.K + 63) / 64;
#pragma unroll 2
    for (int64_t s = warp; s < slices; s += FEW_WARPS) {
        const int64_t k = s * 64 + q * 16;
        uint32_t a[2][2][8], x[NT][8];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) load16<T, VEC>(a[m][h], rows[m][h], k, p.K, true);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int n = t * 8 + g;
            load16<T, VEC>(x[t], p.x + (n < p.rows ? n : 0) * p.ldx, k, p.K, n < p.rows);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t f[4] = {a[m][0][2 * i], a[m][1][2 * i], a[m][0][2 * i + 1], a[m][1][2 * i + 1]};
                    warpmma::mma_16816<BF16>(acc[m][t], f, x[t][2 * i], x[t][2 * i + 1]);
                }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                red[warp][m][t * 8 + q * 2 + (i & 1)][g + (i >> 1) * 8] = acc[m][t][i];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * 16; i += 32 * FEW_WARPS) {
        const int n = i / 16, c = i % 16;
        if (n >= p.rows || f0 + c >= p.F) continue;
        float sg = 0.0f, su = 0.0f;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) {
            sg += red[w][0][n][c];
            su += red[w][1][n][c];
        }
        float v = 0.0f;
        with_activation(p.act, [&](auto act) { v = act_value<decltype(act)::value>(sg) * su; });
        y[n * ldy + f0 + c] = from_float<T>(v);
        if (gate) gate[n * p.F + f0 + c] = from_float<T>(sg);
        if (up) up[n * p.F + f0 + c] = from_float<T>(su);
    }
}

template <typename T>
void few_rows(Handle& h, const GatedArgs<T>& a, T* y, int64_t ldy, T* gate, T* up) {
    const bool vec = a.K % 8 == 0 && tma_ok(a.wg, a.F > 1 ? a.ldwg : 0) && tma_ok(a.wu, a.F > 1 ? a.ldwu : 0) &&
                     tma_ok(a.x, a.rows > 1 ? a.ldx : 0);
    auto kern = a.rows <= 8 ? (vec ? few_rows_kernel<T, 1, true> : few_rows_kernel<T, 1, false>)
                            : (vec ? few_rows_kernel<T, 2, true> : few_rows_kernel<T, 2, false>);
    launch_dependent(h.stream, kern, (unsigned)ceil_div(a.F, 16), 32 * FEW_WARPS, 0, 1, a, y, ldy, gate, up);
    after_launch(h, "gated_few_rows");
}

}  // namespace gated
}  // namespace xspmm_b200
