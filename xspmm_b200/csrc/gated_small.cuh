// gated_small.cuh -- the whole gradient of the gated feed-forward block in one pass over the rows, for
// K, F <= 128 (a graph layer's width): x, dy, gate and up are read once and dx written once, which is
// what bounds it (2^20 rows of 128: 1.34 GB, 208 us at the copy bandwidth).
//
// A persistent CTA per SM takes tiles of 128 rows. Sixteen warps compute dg and du of the tile from dy,
// gate and up (loaded straight to registers, one tile ahead) and write them to shared memory as the
// SWIZZLE_128B image of a [128 rows x 64 features] box. That image is at once dg as the A operand of
// dx = dg wg + du wu (K-major: rows are M, features are summed) and dg^T as the A operand of
// dwg = dg^T x (MN-major: features are M, rows are summed), so it is written once and feeds both. Both
// weights stay in shared memory, dwg and dwu accumulate in TMEM over all of the CTA's tiles, and dx has two
// TMEM accumulators in turn (512 columns in all). While the MMAs of a tile run, the same warps store
// the tile before's dx. At the end every CTA leaves its dwg and dwu as fp32 partials, which the join
// kernel adds in CTA order.
#pragma once

#include "gated_tc.cuh"

namespace xspmm_b200 {
namespace gated {

constexpr int SMALL = 128;                       // largest K and F
constexpr int SM_WORKERS = 16, SM_FIRST = 4;     // warps 4..19 compute, 0 issues MMAs, 1 loads, 2 TMEM
constexpr int SM_THREADS = 32 * (SM_FIRST + SM_WORKERS);
constexpr int SM_CHUNK = TM * 128;               // 64 columns of 128 rows
constexpr int SM_W = 0, SM_D = 4 * SM_CHUNK, SM_X = 8 * SM_CHUNK, SM_TURN = 12 * SM_CHUNK;
constexpr int SM_BARS = SM_TURN + SM_WORKERS * TURN;
constexpr size_t SM_BYTES = 1024 + SM_BARS + 256;
static_assert(SM_BYTES <= 232448, "shared memory per CTA");
constexpr uint32_t SM_DW = 256;                  // TMEM column of dwg; dwu 128 further

struct SmallArgs {
    TileArgs t;  // a[0]: x, b: the weights; out[0], out[1]: dwg, dwu (for the join), out[2]: dx
    const void *dy, *gate, *up;
    int64_t lddy;
    int F, K;
    int tiles;
    uint32_t idesc_dx, idesc_dw;
};

__device__ __forceinline__ uint64_t desc_mn_wide(uint32_t saddr) {  // 64-column chunks SM_CHUNK apart
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(SM_CHUNK >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS, 1) small_grad_kernel(const __grid_constant__ SmallArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* w_full = reinterpret_cast<uint64_t*>(smem + SM_BARS);
    uint64_t* x_full = w_full + 1;    // [2]
    uint64_t* x_empty = x_full + 2;   // [2]
    uint64_t* d_full = x_empty + 2;
    uint64_t* d_empty = d_full + 1;
    uint64_t* dx_full = d_empty + 1;  // [2]
    uint64_t* dx_empty = dx_full + 2; // [2]
    uint64_t* done = dx_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned* err = p.t.err;

    if (threadIdx.x == 0) {
        mbar_init(w_full, 1);
        mbar_init(d_full, SM_WORKERS);
        mbar_init(d_empty, 1);
        mbar_init(done, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&x_full[b], 1);
            mbar_init(&x_empty[b], 1);
            mbar_init(&dx_full[b], 1);
            mbar_init(&dx_empty[b], SM_WORKERS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_alloc_all<1>(tmem_slot);
    // columns of dg and du past F are never written: zeros for the last summed slice
    for (int i = threadIdx.x; i < 4 * SM_CHUNK / 16; i += SM_THREADS)
        reinterpret_cast<uint4*>(smem + SM_D)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    cudaGridDependencySynchronize();  // what came before wrote the operands

    const int kchunks = p.K > 64 ? 2 : 1;
    if (warp == 0) {
        if (lane == 0) {
            bool ok = mbar_wait(w_full, 0, err);
            for (int t = blockIdx.x, i = 0; t < p.tiles && ok; t += gridDim.x, ++i) {
                const int b = i & 1;
                ok = (i < 2 || mbar_wait(&dx_empty[b], ((i >> 1) - 1) & 1, err)) &&
                     mbar_wait(&x_full[b], (i >> 1) & 1, err) && mbar_wait(d_full, i & 1, err);
                if (!ok) break;
                tc_fence_after();
                const uint32_t sw = smem_u32(smem + SM_W), sd = smem_u32(smem + SM_D);
                const uint32_t sx = smem_u32(smem + SM_X + b * 2 * SM_CHUNK);
#pragma unroll
                for (int m = 0; m < 2; ++m)  // dx += d w, summed over the features
#pragma unroll
                    for (int s = 0; s < SMALL / 16; ++s)
                        if (s * 16 < p.F)
                            tc_mma(tmem + b * 128, desc_k(sd + m * 2 * SM_CHUNK + s / 4 * SM_CHUNK + s % 4 * 32),
                                   desc_mn_wide(sw + m * 2 * SM_CHUNK + s * 2048), p.idesc_dx, m > 0 || s > 0);
                tc_commit(&dx_full[b]);
#pragma unroll
                for (int m = 0; m < 2; ++m)  // dw += d^T x, summed over the rows
#pragma unroll
                    for (int s = 0; s < TM / 16; ++s)
                        tc_mma(tmem + SM_DW + m * 128, desc_mn_wide(sd + m * 2 * SM_CHUNK + s * 2048),
                               desc_mn_wide(sx + s * 2048), p.idesc_dw, i > 0 || s > 0);
                tc_commit(d_empty);
                tc_commit(&x_empty[b]);
            }
            tc_commit(done);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            mbar_expect_tx(w_full, (uint32_t)(2 * kchunks * SM_CHUNK));
            for (int m = 0; m < 2; ++m)
                for (int c = 0; c < kchunks; ++c)
                    tma_load_2d(smem + SM_W + (2 * m + c) * SM_CHUNK, &p.t.b[m], 64 * c, 0, w_full);
            // dy, gate and up of a tile, on their way to L2 while the warps have up to two tiles before it to do
            auto prefetch = [&](const void* m, int64_t ld, int t) {
                if (ld != p.F) return;
                const int64_t r = (int64_t)t * TM, n = min((int64_t)TM, p.t.M - r);
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                                 static_cast<const T*>(m) + r * p.F),
                             "r"((uint32_t)(n * p.F * sizeof(T)))
                             : "memory");
            };
            int i = 0;
            for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++i) {
                const int b = i & 1;
                if (i >= 2 && !mbar_wait(&x_empty[b], ((i >> 1) - 1) & 1, err)) break;
                prefetch(p.dy, p.lddy, t);
                prefetch(p.gate, p.F, t);
                prefetch(p.up, p.F, t);
                mbar_expect_tx(&x_full[b], (uint32_t)(kchunks * SM_CHUNK));
                for (int c = 0; c < kchunks; ++c)
                    tma_load_2d(smem + SM_X + (2 * b + c) * SM_CHUNK, &p.t.a[0], 64 * c, t * TM, &x_full[b]);
            }
            // no load may be in flight when the CTA ends (they have all landed unless a wait ran out)
            mbar_wait(w_full, 0, err);
            for (int j = max(0, i - 2); j < i; ++j) mbar_wait(&x_full[j & 1], (j >> 1) & 1, err);
        }
    } else if (warp >= SM_FIRST) {
        const int w = warp - SM_FIRST, tid = threadIdx.x - 32 * SM_FIRST;
        const int quarter = warp & 3, col0 = w / 4 * 32;  // this warp's rows and columns of an accumulator
        uint8_t* turn = smem + SM_TURN + w * TURN;
        int piece = 0;
        const T *dy = static_cast<const T*>(p.dy), *gate = static_cast<const T*>(p.gate),
                *up = static_cast<const T*>(p.up);
        // a thread's 16-byte pieces of a tile: piece j covers row[j], features 8 * pos[j] ...
        const int per_row = p.F / 8;
        int row[4], pos[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = tid + j * 32 * SM_WORKERS;
            row[j] = at / per_row;
            pos[j] = at - row[j] * per_row;
        }
        uint4 d[4], g[4], u[4];
        auto load = [&](int t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[j] = g[j] = u[j] = make_uint4(0, 0, 0, 0);
                const int64_t r = (int64_t)t * TM + row[j];
                if (row[j] < TM && r < p.t.M) {
                    d[j] = __ldg(reinterpret_cast<const uint4*>(dy + r * p.lddy + pos[j] * 8));
                    g[j] = __ldg(reinterpret_cast<const uint4*>(gate + r * p.F + pos[j] * 8));
                    u[j] = __ldg(reinterpret_cast<const uint4*>(up + r * p.F + pos[j] * 8));
                }
            }
        };
        auto store_dx = [&](int t, int i) {  // tile t, the CTA's i-th
            const int b = i & 1;
            if (!mbar_wait(&dx_full[b], (i >> 1) & 1, err)) return false;
            tc_fence_after();
            uint32_t words[16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t v[16];
                tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * 128 + col0 + 16 * h), v);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    words[8 * h + e] = pack2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]), T());
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&dx_empty[b]);
            const int64_t row0 = (int64_t)t * TM + quarter * 32;
            const int rows = (int)max((int64_t)0, min((int64_t)32, p.t.M - row0));
            if (col0 < p.K) store_group<T, false, 1>(p.t, 2, turn, piece, words, row0, col0, rows, min(32, p.K - col0));
            return true;
        };
        bool ok = true;
        int i = 0, t = blockIdx.x;
        load(t);
        for (; t < p.tiles && ok; t += gridDim.x, ++i) {
            // dg into d and du into g, under the MMAs of the tile before; only the stores wait for them
            with_activation(p.t.act, [&](auto act) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t dw[4] = {d[j].x, d[j].y, d[j].z, d[j].w}, gw[4] = {g[j].x, g[j].y, g[j].z, g[j].w};
                    const uint32_t uw[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
                    uint32_t a[4], b[4];
                    slope_words<decltype(act)::value, T>(a, b, dw, gw, uw);
                    d[j] = make_uint4(a[0], a[1], a[2], a[3]);
                    g[j] = make_uint4(b[0], b[1], b[2], b[3]);
                }
            });
            if (i > 0 && !mbar_wait(d_empty, (i - 1) & 1, err)) {
                ok = false;
                break;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (row[j] >= TM) continue;
                uint8_t* at = smem + SM_D + pos[j] / 8 * SM_CHUNK + row[j] * 128 + ((pos[j] ^ row[j]) & 7) * 16;
                *reinterpret_cast<uint4*>(at) = d[j];
                *reinterpret_cast<uint4*>(at + 2 * SM_CHUNK) = g[j];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(d_full);
            load(t + gridDim.x);  // past the last row: nothing is read
            if (i > 0) ok = store_dx(t - gridDim.x, i - 1);
        }
        if (ok && i > 0) ok = store_dx(t - gridDim.x, i - 1);
        if (ok && mbar_wait(done, 0, err)) {
            tc_fence_after();
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float4* dst = p.t.partial + ((int64_t)(blockIdx.x * 2 + m) * (ACC_COLS / 4) + col0 / 4) * TM +
                              quarter * 32 + lane;
                uint32_t v[32];
                tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + SM_DW + (uint32_t)(m * 128 + col0), v);
                tmem_wait();
                store_partial(dst, v, 32);
            }
            tc_fence_before();
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }
    __syncwarp();
    if (warp == 2) mbar_wait(done, 0, err);  // bounded; completes once the last MMA has
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 2) tmem_free_all<1>(tmem);
}

// Whether the one-pass gradient takes these arguments.
template <typename T>
bool small_grad_ok(const GatedArgs<T>& a, const T* dy, int64_t lddy, const T* gate, const T* up, const T* dx,
                   int64_t lddx, const T* dwg) {
    return dx && dwg && a.K <= SMALL && a.F <= SMALL && a.K % 8 == 0 && a.F % 8 == 0 && tma_ok(a.x, a.ldx) &&
           tma_ok(a.wg, a.ldwg) && tma_ok(a.wu, a.ldwu) && aligned_to(dy, 16) && lddy % 8 == 0 &&
           aligned_to(gate, 16) && aligned_to(up, 16) && tma_ok(dx, lddx);
}

template <typename T>
void small_grad(Handle& h, const GatedArgs<T>& a, const T* dy, int64_t lddy, const T* gate, const T* up, T* dx,
                int64_t lddx, T* dwg, T* dwu) {
    constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    SmallArgs s = {};
    TileArgs& t = s.t;
    s.dy = dy;
    s.gate = gate;
    s.up = up;
    s.lddy = lddy;
    s.F = (int)a.F;
    s.K = (int)a.K;
    s.tiles = (int)ceil_div(a.rows, TM);
    const int n = (s.K + 15) / 16 * 16;
    s.idesc_dx = make_idesc(bf16, false, true, TM, n);
    s.idesc_dw = make_idesc(bf16, true, true, TM, n);
    const int grid = std::min(s.tiles, sm_count(h.device));
    auto map = [](const T* p, int64_t ld, int64_t rows, int64_t cols) {
        return make_map_2d(p, (uint64_t)cols, (uint64_t)rows, (uint64_t)ld * 2, 64, TM, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    t.a[0] = map(a.x, a.ldx, a.rows, a.K);
    t.b[0] = map(a.wg, a.ldwg, a.F, a.K);
    t.b[1] = map(a.wu, a.ldwu, a.F, a.K);
    t.act = a.act;
    t.err = h.d_err;
    t.N = a.K;
    t.M = a.rows;
    set_output(t, 2, dx, lddx);
    DevBuf<float4> ws((size_t)grid * 2 * (ACC_COLS / 4) * TM, h.stream);
    t.partial = ws.get();
    allow_smem(small_grad_kernel<T>, SM_BYTES);
    launch_dependent(h.stream, small_grad_kernel<T>, (unsigned)grid, SM_THREADS, SM_BYTES, 1, s);
    after_launch(h, "gated_small_grad");
    // one shared tile for each weight, a slice a CTA
    t.M = a.F;
    t.mt = t.nt = 1;
    t.whole = 0;
    t.splits = grid;
    t.bn = n;
    set_output(t, 0, dwg, a.K);
    set_output(t, 1, dwu, a.K);
    launch_dependent(h.stream, join_kernel<T, Product::Dw, 2>, (unsigned)(2 * ((t.bn + 31) / 32) * (TM / 4)), 256, 0, 1, t);
    after_launch(h, "gated_join");
}

}  // namespace gated
}  // namespace xspmm_b200
