// tile_product.cuh -- matrix products on the 5th-generation tensor cores whose operands or results are not of
// one 16-bit type: one persistent kernel, two kinds.
//
//   Int8   D[m, n] = sum_k A[m, k] B[n, k] of 8-bit integers, exact in 32 bits (kind::i8).
//   Split  the same of numbers held as two fp16 parts, v = (hi + lo) 2^-14: hi hi' + (hi lo' + lo hi'), 22 bits of
//          each operand. The product of the low parts, below 2^-22 of the whole, is left out.
//
// A CTA's part of a tile is 128 rows by up to 256 columns; a stage holds 128 bytes of every row (64 fp16 or 128
// 8-bit elements), by TMA in the SWIZZLE_128B layout. Roles, barriers, pairs of CTAs (CG = 2) and slices of split
// tiles are those of the gated block's products (gated_tc.cuh).
//
// Split brings both parts of both operands once a stage and issues three MMAs on them: 64 KB of loads into an SM
// for 1536 clocks of MMA, where a pass over the sum for each of the three would need 96 KB. The two cross products
// are summed in an accumulator of their own and joined with the large one in fp32 afterwards: an addition in the
// tensor core truncates, and small terms on top of a large sum would triple the truncations of it. The two
// accumulators fill TMEM, so a tile's epilogue does not run under the next one's MMAs as it does for Int8.
// The large accumulator holds the sum of DRAIN stages at most: then the epilogue's warps add it to sums in their
// registers, where additions round, while the tensor core is at the cross products of the stages on both sides. An update
// of 11008 x 4096 normal numbers is 5e-6 off before its rounding, the iteration in fp32 8e-6; with all of the sum in the
// accumulator it was 1e-4 (at 1 % less time; DRAIN = 4: 9e-6; 768 x 1232: 3e-6 in 228 us, 5e-6 in 221, 7e-6 in 210).
//
// The entries of X, A and B' (orthogonalize.cu) are below 4 in magnitude, so 2^14 times them fits fp16, and parts
// down to 2^-38 are held. An X of small norm is held with a larger power of two.
#pragma once

#include "gated_tc.cuh"

namespace xspmm_b200 {
namespace product {

using namespace gated;

// What becomes of an accumulator: y of the 8-bit product; A = X X^T; B' = a I + b A + c A A; the next X; the
// update itself. Gram and Poly are symmetric: tiles on and above the diagonal are computed and stored twice.
enum class Epi { Int8, Gram, Poly, Next, Last };
constexpr bool symmetric(Epi e) { return e == Epi::Gram || e == Epi::Poly; }
constexpr bool split(Epi e) { return e != Epi::Int8; }

constexpr int DRAIN = 2;  // stages: 128 summed elements, 8 truncated additions

constexpr float SPLIT_SCALE = 16384.0f, SPLIT_INV = 1.0f / 16384.0f;
constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;

// a, b: Int8 [0]; Split [0] = hi, [1] = lo. out: y, or [0] = hi, [1] = lo in scratch, whose rows are padded to
// whole 16-byte words (N counts the padding, whose products are zeros).
struct Args : TileArgs {
    const float *xs, *ws, *bias;  // Int8
    const __half *ah, *al;        // Poly: A's parts, row stride lda
    int64_t lda;
    const float* mul;             // the others of Split: a power of two that the results are multiplied by
};

constexpr int COLUMN_BYTES = EPI_WARPS * 64 * 4;  // Int8: a warp's 32 column scales and biases

template <typename T>
constexpr int turn_bytes() { return EPI_WARPS * TURNS * 32 * 32 * (sizeof(T) == 4 ? 4 : 2); }
template <Epi E, typename T>
constexpr int stage_room() { return SMEM_MAX - turn_bytes<T>() - (E == Epi::Int8 ? COLUMN_BYTES : 0); }

template <Epi E, int CG>
__device__ __forceinline__ void issue(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (split(E)) {
        pair_mma<CG>(d, a, b, idesc, accumulate);
    } else if constexpr (CG == 2) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}

// Tile number to its place. Symmetric: the tiles on and above the diagonal, column by column.
template <Epi E>
__device__ __forceinline__ void place(const Args& p, int tile, int* mi, int* ni) {
    if constexpr (symmetric(E)) {
        int c = (int)((sqrtf(8.0f * (float)tile + 1.0f) - 1.0f) * 0.5f);
        while (c * (c + 1) / 2 > tile) --c;
        while ((c + 1) * (c + 2) / 2 <= tile) ++c;
        *ni = c;
        *mi = tile - c * (c + 1) / 2;
    } else {
        tile_place(p, tile, mi, ni);
    }
}
template <Epi E>
__host__ __device__ __forceinline__ int tiles_of(const TileArgs& p) {
    return symmetric(E) ? p.nt * (p.nt + 1) / 2 : p.mt * p.nt;
}
template <Epi E>
__device__ __forceinline__ Item item(const Args& p, int t) {
    Item it{0, 0, 0, p.ksteps, -1};
    int tile = t;
    if (t >= p.whole) {
        const int rest = tiles_of<E>(p) - p.whole, s = (t - p.whole) / rest;
        it.part = t - p.whole;
        tile = p.whole + it.part - s * rest;
        it.k0 = (int)((int64_t)p.ksteps * s / p.splits);
        it.k1 = (int)((int64_t)p.ksteps * (s + 1) / p.splits);
    }
    place<E>(p, tile, &it.mi, &it.ni);
    return it;
}

// v as fp16 parts of v 2^14, two values a word.
__device__ __forceinline__ void split2(float v0, float v1, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(v0, v1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(v0 - f.x, v1 - f.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// An accumulator's value (2^28 times the product's, before `mul`) as 2^14 times the result, for Last as the result itself;
// `a` is 2^14 times A's entry.
template <Epi E>
__device__ __forceinline__ float finish(float acc, float a, bool diagonal, float mul) {
    if constexpr (E == Epi::Poly)
        return fmaf(NS_B, a, NS_C * (acc * SPLIT_INV)) + (diagonal ? NS_A * SPLIT_SCALE : 0.0f);
    else if constexpr (E == Epi::Last) return acc * (SPLIT_INV * SPLIT_INV) * mul;
    else return acc * SPLIT_INV * mul;
}

// fp32 results (lane = row, 32 columns) to `out`, through a staging piece of 32 rows of 128 bytes.
template <bool ANY>
__device__ __forceinline__ void store_group32(const TileArgs& p, uint8_t* turn, int& piece, const uint32_t (&v)[32],
                                              int64_t row0, int64_t col0, int rows, int cols) {
    const int lane = threadIdx.x & 31;
    uint8_t* at = turn + piece * 4096;
    piece ^= 1;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(TURNS - 1) : "memory");
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i)  // SWIZZLE_128B: 16-byte pieces by the row's last three bits
        *reinterpret_cast<uint4*>(at + lane * 128 + ((i ^ (lane & 7)) * 16)) =
            make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    if ((!ANY || p.tma[0]) && cols == 32) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && rows > 0)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                             reinterpret_cast<uint64_t>(&p.omap[0])),
                         "r"((int)col0), "r"((int)row0), "r"(smem_u32(at))
                         : "memory");
    } else {
        __syncwarp();
        float* out = static_cast<float*>(p.out[0]) + row0 * p.ld[0] + col0 + lane;
        if (lane < cols)
#pragma unroll 8
            for (int r = 0; r < rows; ++r)
                out[r * p.ld[0]] = *reinterpret_cast<const float*>(at + r * 128 + (((lane >> 2) ^ (r & 7)) * 16) + (lane & 3) * 4);
        __syncwarp();
    }
    if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // one group a use, empty or not
}

// A warp's 32 x 32 fp16 words (lane = row) to the transposed place: lanes side by side.
__device__ __forceinline__ void store_mirror(__half* out, int64_t ld, const uint32_t (&w)[16], int64_t row0, int64_t col0,
                                             int rows, int cols) {
    const int lane = threadIdx.x & 31;
    if (lane >= rows) return;
    uint16_t* at = reinterpret_cast<uint16_t*>(out) + col0 * ld + row0 + lane;
#pragma unroll
    for (int c = 0; c < 32; ++c)
        if (c < cols) at[c * ld] = (uint16_t)(w[c / 2] >> (c % 2 * 16));
}

// A warp has read its part of an accumulator.
template <int CG>
__device__ __forceinline__ void taken(uint64_t* acc_empty) {
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
        if constexpr (CG == 2) arrive_cluster(first_cta_addr(acc_empty));
        else mbar_arrive(acc_empty);
    }
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
        "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
        "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
        : "memory");
}

// Takes a work item's large accumulator as often as it is filled, the u-th filling of all first, and returns with the last
// filling's wait done and the sum of all in the accumulator, false where a wait ran out. acc: the warp's lanes; it takes
// the 32-column groups half, half + 2, ... below ncols.
template <int CG>
__device__ __forceinline__ bool drain(const TileArgs& p, uint32_t acc, int half, int ncols, int stages, uint64_t* acc_full,
                                      uint64_t* acc_empty, int& u) {
    constexpr int GROUPS = ACC_COLS / 64;
    if (stages <= DRAIN) return mbar_wait(acc_full, u & 1, p.err);
    float sum[GROUPS][32] = {};
#pragma unroll 1
    for (int left = stages;; left -= DRAIN) {
        if (!mbar_wait(acc_full, u & 1, p.err)) return false;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            if (half * 32 + g * 64 >= ncols) continue;
#pragma unroll
            for (int h = 0; h < 32; h += 16) {  // 16 columns: the sums leave no room for more
                uint32_t v[16];
                tmem_ld16(acc + (uint32_t)(half * 32 + g * 64 + h), v);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    asm volatile("" : "+r"(v[e]));  // not before the wait
                    sum[g][h + e] += __uint_as_float(v[e]);
                }
            }
        }
        if (left <= DRAIN) break;
        taken<CG>(acc_empty);
        ++u;
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        if (half * 32 + g * 64 >= ncols) continue;
        uint32_t v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(sum[g][e]);
        tmem_st32(acc + (uint32_t)(half * 32 + g * 64), v);
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    return true;
}

// AMN, BMN: the operand's output index is contiguous in memory, not the summed one (Split only).
template <Epi E, typename T, int CG, bool AMN, bool BMN, bool ANY>
__global__ void __launch_bounds__(THREADS, 1) tile_product_kernel(const __grid_constant__ Args p) {
    constexpr bool SPLIT = split(E);
    constexpr int TKE = SPLIT ? 64 : 128;     // summed elements a stage
    constexpr int BUFFERS = SPLIT ? 1 : 2;    // accumulators used in turn
    constexpr int PARTS = SPLIT ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int part_bytes = A_BYTES + p.b_bytes, stage_bytes = PARTS * part_bytes;
    uint8_t* turn = smem + p.stages * stage_bytes;
    float* columns = reinterpret_cast<float*>(turn + turn_bytes<T>());
    uint64_t* full = reinterpret_cast<uint64_t*>(turn + turn_bytes<T>() + (SPLIT ? 0 : COLUMN_BYTES));
    uint64_t* empty = full + MAX_STAGES;
    uint64_t* acc_full = empty + MAX_STAGES;  // [2]
    uint64_t* acc_empty = acc_full + 2;       // [2]
    uint64_t* done = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 2 ? (int)cta_rank() : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);   // the first CTA's: its own expect_tx, both CTAs' bytes
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], CG * EPI_WARPS);  // the first CTA's: both epilogues
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_alloc_all<CG>(tmem_slot);
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync_all();  // the barriers of both CTAs are set up
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    cudaGridDependencySynchronize();  // what came before wrote the operands

    const int work = p.whole + (tiles_of<E>(p) - p.whole) * p.splits;
    const int group = blockIdx.x / CG, groups = gridDim.x / CG;

    if (warp == 0) {
        if (lane == 0 && rank == 0) {
            int s = 0, phase = 0;  // the next stage, and whether its ring has come round an odd number of times
            bool ok = true;
            int u = 0;  // accumulators filled
            for (int t = group; t < work && ok; t += groups, ++u) {
                const int b = u % BUFFERS;
                if (u >= BUFFERS && !mbar_wait(&acc_empty[b], (u / BUFFERS - 1) & 1, p.err)) break;
                tc_fence_after();
                const uint32_t acc = tmem + (uint32_t)(b * ACC_COLS), cross = tmem + ACC_COLS;
                const Item it = item<E>(p, t);
                for (int k = it.k0; k < it.k1; ++k) {
                    const uint32_t sa = smem_u32(smem + s * stage_bytes), sb = sa + PARTS * A_BYTES;
                    const uint64_t da = AMN ? desc_mn(sa) : desc_k(sa), db = BMN ? desc_mn(sb) : desc_k(sb);
                    const uint64_t la = AMN ? desc_mn(sa + A_BYTES) : desc_k(sa + A_BYTES);
                    const uint64_t lb = BMN ? desc_mn(sb + p.b_bytes) : desc_k(sb + p.b_bytes);
                    if (!mbar_wait(&full[s], phase, p.err)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    // an MMA's summed elements: 32 bytes along a K-major row, 2 KB of MN-major rows, in units of 16
                    auto each = [&](auto&& f) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) f(q, (uint64_t)(q * (AMN ? 128 : 2)), (uint64_t)(q * (BMN ? 128 : 2)));
                    };
                    const int in = SPLIT ? (k - it.k0) % DRAIN : k - it.k0;  // stages in the accumulator
                    auto large = [&] {
                        each([&](int q, uint64_t oa, uint64_t ob) { issue<E, CG>(acc, da + oa, db + ob, p.idesc, in > 0 || q > 0); });
                    };
                    auto small = [&] {
                        each([&](int q, uint64_t oa, uint64_t ob) {
                            issue<E, CG>(cross, da + oa, lb + ob, p.idesc, k > it.k0 || q > 0);
                            issue<E, CG>(cross, la + oa, db + ob, p.idesc, 1);
                        });
                    };
                    // the accumulator is drained under the cross products before its first stage and after its last
                    if constexpr (!SPLIT) {
                        large();
                    } else if (in > 0 || k == it.k0) {
                        large();
                        if (in == DRAIN - 1 && k + 1 < it.k1) pair_commit<CG>(&acc_full[b]);
                        small();
                    } else {
                        small();
                        if (!mbar_wait(&acc_empty[b], u & 1, p.err)) {
                            ok = false;
                            break;
                        }
                        ++u;
                        tc_fence_after();
                        large();
                    }
                    pair_commit<CG>(&empty[s]);
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
                if (ok) pair_commit<CG>(&acc_full[b]);
            }
            pair_commit<CG>(done);  // arrives at once where nothing was issued
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int s = 0, phase = 0, held = 0;  // held: stages filled, at most all
            bool ok = true;
            for (int t = group; t < work && ok; t += groups) {
                const Item it = item<E>(p, t);
                const int m0 = (it.mi * CG + rank) * TM, nb = it.ni * p.bn + rank * (p.acc_n / CG);
                for (int k = it.k0; k < it.k1; ++k) {
                    if (held == p.stages && !mbar_wait(&empty[s], phase ^ 1, p.err)) {
                        ok = false;
                        break;
                    }
                    if (held < p.stages) ++held;
                    if (rank == 0) mbar_expect_tx(&full[s], (uint32_t)(CG * stage_bytes));
                    const uint32_t bar = CG == 2 ? first_cta_addr(&full[s]) : smem_u32(&full[s]);
                    uint8_t* sa = smem + s * stage_bytes;
                    uint8_t* sb = sa + PARTS * A_BYTES;
#pragma unroll
                    for (int h = 0; h < PARTS; ++h, sa += A_BYTES, sb += p.b_bytes) {
                        if constexpr (AMN) {
                            for (int c = 0; c < TM / 64; ++c)
                                pair_load<CG>(sa + c * CHUNK, &p.a[h], m0 + 64 * c, k * TKE, bar);
                        } else {
                            pair_load<CG>(sa, &p.a[h], k * TKE, m0, bar);
                        }
                        if constexpr (BMN) {
                            for (int c = 0; c * CHUNK < p.b_bytes; ++c)
                                pair_load<CG>(sb + c * CHUNK, &p.b[h], nb + 64 * c, k * TKE, bar);
                        } else {
                            pair_load<CG>(sb, &p.b[h], k * TKE, nb, bar);
                        }
                    }
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
            }
            // No load may be in flight when the CTA ends. Each landed before its MMAs ran, and the commit
            // after those freed its stage (they have all done so unless a wait ran out).
            for (; held > 0; --held) {
                if (s-- == 0) s = p.stages - 1, phase ^= 1;
                mbar_wait(&empty[s], phase, p.err);
            }
        }
    } else if (warp >= FIRST_EPI) {
        const int quarter = warp & 3, half = (warp - FIRST_EPI) >> 2;
        uint8_t* my_turn = turn + (warp - FIRST_EPI) * (turn_bytes<T>() / EPI_WARPS);
        float* my_columns = columns + (warp - FIRST_EPI) * 64;
        int piece = 0;
        bool ok = true;
        float mul = 1.0f;
        if constexpr (SPLIT && E != Epi::Poly) mul = *p.mul;
        for (int t = group, u = 0; t < work; t += groups, ++u) {
            const int b = u % BUFFERS;
            const Item it = item<E>(p, t);
            const int64_t row0 = (int64_t)(it.mi * CG + rank) * TM + quarter * 32, n0 = (int64_t)it.ni * p.bn;
            const int rows = (int)max((int64_t)0, min((int64_t)32, p.M - row0));
            const int ncols = (int)min((int64_t)p.bn, p.N - n0);
            float scale = 0.0f;
            if constexpr (E == Epi::Int8)
                if (lane < rows) scale = p.xs[row0 + lane];
            if constexpr (SPLIT)
                ok = drain<CG>(p, tmem + ((uint32_t)(quarter * 32) << 16), half, ncols, it.k1 - it.k0, acc_full, acc_empty, u);
            else ok = mbar_wait(&acc_full[b], (u / BUFFERS) & 1, p.err);
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * ACC_COLS);
            float4* partial = p.partial + ((int64_t)it.part * CG + rank) * (ACC_COLS / 4) * TM + quarter * 32 + lane;
            for (int c = half * 32; c < ncols; c += 64) {
                const int cols = min(32, ncols - c);
                uint32_t v[32];
                tmem_ld32(acc + (uint32_t)c, v);
                if constexpr (SPLIT) {
                    uint32_t u[32];
                    tmem_ld32(acc + (uint32_t)(ACC_COLS + c), u);
                    tmem_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(u[e]));
                } else {
                    tmem_wait();
                }
                if (it.part >= 0) {
                    store_partial(partial + c / 4 * TM, v, p.bn - c);
                } else if constexpr (E == Epi::Int8) {
                    __syncwarp();  // the last group's columns are read
                    const int64_t at = n0 + c + min(lane, cols - 1);
                    my_columns[lane] = p.ws[at];
                    my_columns[32 + lane] = p.bias ? p.bias[at] : 0.0f;
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 ws = *reinterpret_cast<const float4*>(my_columns + e);
                        const float4 bs = *reinterpret_cast<const float4*>(my_columns + 32 + e);
                        v[e] = __float_as_uint(fmaf((float)(int)v[e] * scale, ws.x, bs.x));
                        v[e + 1] = __float_as_uint(fmaf((float)(int)v[e + 1] * scale, ws.y, bs.y));
                        v[e + 2] = __float_as_uint(fmaf((float)(int)v[e + 2] * scale, ws.z, bs.z));
                        v[e + 3] = __float_as_uint(fmaf((float)(int)v[e + 3] * scale, ws.w, bs.w));
                    }
                    if constexpr (sizeof(T) == 4) {
                        store_group32<ANY>(p, my_turn, piece, v, row0, n0 + c, rows, cols);
                    } else {
                        uint32_t w[16];
                        pack_words<T>(w, v);
                        store_group<T, ANY>(p, 0, my_turn, piece, w, row0, n0 + c, rows, cols);
                    }
                } else if constexpr (E == Epi::Last) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(finish<E>(__uint_as_float(v[e]), 0.0f, false, mul));
                    pack_words<T>(w, v);
                    store_group<T, ANY>(p, 0, my_turn, piece, w, row0, n0 + c, rows, cols);
                } else {
                    uint32_t hi[16], lo[16];
                    const int64_t row = row0 + lane;
                    if constexpr (E == Epi::Poly) {
                        const int64_t at = min(row, p.M - 1) * p.lda + n0 + c;  // rows of whole 16-byte words
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            uint4 h4 = make_uint4(0, 0, 0, 0), l4 = h4;
                            if (8 * e < cols) {
                                h4 = *reinterpret_cast<const uint4*>(p.ah + at + 8 * e);
                                l4 = *reinterpret_cast<const uint4*>(p.al + at + 8 * e);
                            }
                            hi[4 * e] = h4.x; hi[4 * e + 1] = h4.y; hi[4 * e + 2] = h4.z; hi[4 * e + 3] = h4.w;
                            lo[4 * e] = l4.x; lo[4 * e + 1] = l4.y; lo[4 * e + 2] = l4.z; lo[4 * e + 3] = l4.w;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 a = make_float2(0.0f, 0.0f);
                        if constexpr (E == Epi::Poly) a = add2(unpack2(hi[e], __half()), unpack2(lo[e], __half()));
                        const int64_t d = row - (n0 + c + 2 * e);
                        split2(finish<E>(__uint_as_float(v[2 * e]), a.x, d == 0, mul),
                               finish<E>(__uint_as_float(v[2 * e + 1]), a.y, d == 1, mul), &hi[e], &lo[e]);
                    }
                    store_group<__half, false>(p, 0, my_turn, piece, hi, row0, n0 + c, rows, cols);
                    store_group<__half, false>(p, 1, my_turn, piece, lo, row0, n0 + c, rows, cols);
                    if constexpr (symmetric(E))
                        if (it.mi != it.ni) {
                            const int real = (int)min((int64_t)cols, p.M - n0 - c);  // without the padding
                            store_mirror(static_cast<__half*>(p.out[0]), p.ld[0], hi, row0, n0 + c, rows, real);
                            store_mirror(static_cast<__half*>(p.out[1]), p.ld[1], lo, row0, n0 + c, rows, real);
                        }
                }
            }
            taken<CG>(&acc_empty[b]);
        }
        // the stores have read the shared memory they come from before the CTA gives it up
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }
    __syncwarp();
    if (warp == 2) mbar_wait(done, 0, p.err);  // bounded; completes once the last MMA has
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();  // neither CTA's shared memory or TMEM is in use any more
    tc_fence_after();
    if (warp == 2) tmem_free_all<CG>(tmem);
}

// Adds the slices of the split tiles in their order and finishes them. A CTA takes 32 x 32 elements: summed with a row a
// lane, as the slices lie (512 bytes a load), and through shared memory stored with a column a lane, and for the mirror
// image with a row a lane. (Stored from the sums' own places, 2 bytes here and there, the joining of a 1341 x 1341 product
// took 35 us, twice the product's time.)
template <Epi E, typename T, int CG>
__global__ void __launch_bounds__(256) tile_join_kernel(const __grid_constant__ Args p) {
    __shared__ float tile[32][33];
    cudaGridDependencySynchronize();
    const int rest = tiles_of<E>(p) - p.whole, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int groups = (p.bn + 31) / 32, slab = (int)(blockIdx.x % (TM / 32)), grp = (int)(blockIdx.x / (TM / 32) % groups);
    const int part = (int)(blockIdx.x / (TM / 32) / groups), rank = part % CG;
    const int64_t slice = (int64_t)rest * CG * (ACC_COLS / 4) * TM;
    int mi, ni;
    place<E>(p, p.whole + part / CG, &mi, &ni);
    const int64_t row0 = (int64_t)(mi * CG + rank) * TM + slab * 32, col0 = (int64_t)ni * p.bn + grp * 32;
    const int rows = (int)max((int64_t)0, min((int64_t)32, p.M - row0));
    const int cols = (int)max((int64_t)0, min((int64_t)min(32, p.bn - grp * 32), p.N - col0));
    if (rows == 0 || cols == 0) return;  // the same in all threads
    if (warp * 4 < cols) {  // a row a lane, 4 columns a warp
        const uint4* src = reinterpret_cast<const uint4*>(p.partial) + ((int64_t)part * (ACC_COLS / 4) + grp * 8 + warp) * TM +
                           slab * 32 + lane;
        uint4 s = src[0];
#pragma unroll 4
        for (int i = 1; i < p.splits; ++i) {
            const uint4 v = src[i * slice];
            auto one = [](uint32_t& a, uint32_t b) {
                if constexpr (split(E)) a = __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
                else a += b;
            };
            one(s.x, v.x), one(s.y, v.y), one(s.z, v.z), one(s.w, v.w);
        }
        const uint32_t v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[lane][warp * 4 + e] = split(E) ? __uint_as_float(v[e]) : (float)(int)v[e];
    }
    __syncthreads();
    const int64_t col = col0 + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = warp * 4 + i;
        const int64_t row = row0 + r;
        if (r >= rows || lane >= cols) continue;
        const float v = tile[r][lane];
        if constexpr (E == Epi::Int8) {
            static_cast<T*>(p.out[0])[row * p.ld[0] + col] =
                from_float<T>(fmaf(v * p.xs[row], p.ws[col], p.bias ? p.bias[col] : 0.0f));
        } else if constexpr (E == Epi::Last) {
            static_cast<T*>(p.out[0])[row * p.ld[0] + col] = from_float<T>(finish<E>(v, 0.0f, false, *p.mul));
        } else {
            float a = 0.0f;
            if constexpr (E == Epi::Poly) a = to_float(p.ah[row * p.lda + col]) + to_float(p.al[row * p.lda + col]);
            const float f = finish<E>(v, a, row == col, E == Epi::Poly ? 1.0f : *p.mul);
            const __half hi = __float2half_rn(f);
            static_cast<__half*>(p.out[0])[row * p.ld[0] + col] = hi;
            static_cast<__half*>(p.out[1])[row * p.ld[1] + col] = __float2half_rn(f - __half2float(hi));
            if constexpr (symmetric(E)) tile[r][lane] = f;
        }
    }
    if constexpr (symmetric(E)) {
        if (mi == ni) return;  // the same in all threads
        __syncthreads();
        for (int c = warp; c < cols && col0 + c < p.M; c += 8) {  // without the padding
            if (lane >= rows) continue;
            const float f = tile[lane][c];
            const __half hi = __float2half_rn(f);
            static_cast<__half*>(p.out[0])[(col0 + c) * p.ld[0] + row0 + lane] = hi;
            static_cast<__half*>(p.out[1])[(col0 + c) * p.ld[1] + row0 + lane] = __float2half_rn(f - __half2float(hi));
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------
// Instruction descriptor, kind::i8: 32-bit integer accumulator, signed operands.
inline uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Picks the tile width (a symmetric product's tiles are square) and how many slices the last wave's tiles are
// cut into: the model of the gated block's products (gated_ffn.cu), with this kernel's clocks a stage.
template <Epi E, int CG>
void choose(Handle& h, Args& t) {
    constexpr int UNIT = 32 * CG;
    const int slots = sm_count(h.device) / CG;
    const double mmas = split(E) ? 3.0 : 1.0, parts = split(E) ? 2.0 : 1.0;
    const double a_bytes = 128.0 * (double)std::min<int64_t>(t.M, TM);
    double least = -1.0;
    for (int bn = symmetric(E) ? TM * CG : UNIT; bn <= 256; bn += UNIT) {
        if (!symmetric(E) && bn < 128 && bn < t.N && bn % 64 != 0) continue;
        const double b_bytes = 128.0 * bn / CG;
        const double step = std::max({mmas * 2.0 * std::max(bn, 64), 2.0 * parts * (A_BYTES + b_bytes) / 128.0,
                                      parts * (a_bytes + b_bytes) / 56.0});
        const double ends = 1500.0 + (split(E) ? 20.0 : 6.0) * bn;
        const int64_t mt = ceil_div(t.M, TM * CG), nt = ceil_div(t.N, bn);
        const int64_t tiles = symmetric(E) ? nt * (nt + 1) / 2 : mt * nt;
        const int64_t whole = tiles / slots * slots, rest = tiles - whole;
        const double full = (double)(tiles / slots) * (t.ksteps * step + ends);
        const int64_t most = rest > 0 ? std::max<int64_t>(1, std::min<int64_t>(slots / rest, t.ksteps / 2)) : 1;
        for (int64_t sp = 1; sp <= most; ++sp) {
            double cost = full;
            if (rest > 0) cost += (double)ceil_div(t.ksteps, sp) * step + ends;
            if (sp > 1) cost += 6000.0 + (double)(rest * sp) * TM * CG * bn * 8.0 / 3000.0;
            if (least < 0.0 || cost < least) {
                least = cost;
                t.bn = bn;
                t.mt = (int)mt;
                t.nt = (int)nt;
                t.splits = (int)sp;
                t.whole = (int)(sp > 1 ? whole : tiles);
            }
        }
        if (bn >= t.N || symmetric(E)) break;
    }
    t.acc_n = t.bn;
}

// Launches `t`, whose maps, sizes, tiles and outputs are set, and joins the slices.
template <Epi E, typename T, int CG, bool AMN, bool BMN>
void launch(Handle& h, Args& t) {
    const int own = t.acc_n / CG;  // a CTA's columns of B
    t.b_bytes = BMN ? (own + 63) / 64 * CHUNK : own * 128;
    t.idesc = split(E) ? make_idesc(false, AMN, BMN, TM * CG, t.acc_n) : idesc_i8(TM * CG, t.acc_n);
    const int stage = (split(E) ? 2 : 1) * (A_BYTES + t.b_bytes);
    t.stages = std::min<int>(MAX_STAGES, stage_room<E, T>() / stage);
    t.err = h.d_err;
    const size_t smem = 1024 + (size_t)t.stages * stage + (SMEM_MAX - stage_room<E, T>()) + 512;
    const int64_t rest = tiles_of<E>(t) - t.whole;
    const int64_t work = t.whole + rest * t.splits;
    DevBuf<float4> ws((size_t)rest * t.splits * CG * (ACC_COLS / 4) * TM, h.stream);
    t.partial = ws.get();
    const bool any = t.out[0] && !t.tma[0];
    auto kern = tile_product_kernel<E, T, CG, AMN, BMN, false>;
    if constexpr (E == Epi::Int8 || E == Epi::Last)
        if (any) kern = tile_product_kernel<E, T, CG, AMN, BMN, true>;
    allow_smem(kern, 1024 + SMEM_MAX + 512);
    const unsigned grid = (unsigned)(std::min<int64_t>(work, sm_count(h.device) / CG) * CG);
    launch_dependent(h.stream, kern, grid, THREADS, smem, CG, t);
    after_launch(h, "tile_product");
    if (rest > 0) {
        const int64_t blocks = rest * CG * ((t.bn + 31) / 32) * (TM / 32);
        launch_dependent(h.stream, tile_join_kernel<E, T, CG>, (unsigned)blocks, 256, 0, 1, t);
        after_launch(h, "tile_join");
    }
}

}  // namespace product
}  // namespace xspmm_b200
