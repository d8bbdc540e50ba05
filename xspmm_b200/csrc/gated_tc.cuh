// gated_tc.cuh -- the matrix products of the gated feed-forward block on the 5th-generation tensor
// cores: one persistent kernel, three products.
//
//   Forward   y[m, f]  = act(sum_k x[m,k] wg[f,k]) * sum_k x[m,k] wu[f,k]
//   Dx        dx[m, k] = sum_f dg[m,f] wg[f,k] + du[m,f] wu[f,k]
//   Dw        dw[f, k] = sum_m d[m,f] x[m,k], d = dg, then du
//
// A CTA's part of an output tile is 128 rows by up to 256 accumulator columns; a summed slice is 64
// deep. Operands come by TMA in the SWIZZLE_128B layout, in whichever order memory has them: K-major
// where the summed index is contiguous (x, weights of Forward; dg, du of Dx), MN-major where the
// output index is (the others), so nothing is transposed. Edges need no code: TMA fills what lies
// outside with zeros.
//
// CG = 2: two CTAs form one MMA of 256 rows (cta_group::2). Each holds its own 128 rows of A and half
// of B's columns in its shared memory, and all columns of its rows in its TMEM. A CTA alone has to
// write and read 24 KB of shared memory per 16-deep MMA of 128 x 256, 192 clocks at 128 bytes a clock
// where the MMA takes 128; in a pair it is 16 KB. Measured on 2048 tokens of 4096 x 11008, forward:
// 354 us alone, 327 paired. CG = 1 is for at most 128 rows, where the second CTA would compute padding.
//   Forward: an MMA of N = 2 bf holds bf columns of both projections, so x is read once for both and the
//   epilogue finds g and u of an output bf columns apart; in a pair one CTA brings wg, the other wu.
//   Dw: the pair's first CTA computes rows of dwg, the second the same rows of dwu.
//
// Roles (384 threads, one CTA per SM): warp 0 of the pair's first CTA issues the MMAs (one lane), warp
// 1 of each the loads of its own operands (one lane; they report to the first CTA's barrier), warp 2
// allocates TMEM, warps 4..11 are the epilogue. TMEM holds two accumulators used in turn, so a tile's
// epilogue runs under the next tile's products. The epilogue converts 32 columns at a time and stores
// them by TMA from a warp's own pieces of shared memory (an output that TMA cannot address: by one or two
// elements a lane, in an instance of its own). Every wait is bounded; a timeout sets the error flag, and
// TMEM is freed only after the MMAs that were issued have completed.
//
// Tiles that would leave part of the GPU idle (the last wave's, or all where there are few) have their
// sum split: each slice's fp32 partial goes to scratch and a second kernel adds them in slice order (the
// same order every time) and finishes the tile.
#pragma once

#include "layers.cuh"
#include "tcgen05.cuh"

namespace xspmm_b200 {
namespace gated {

enum class Product { Forward, Dx, Dw };

constexpr int TM = 128;                 // tile rows (MMA M)
constexpr int TK = 64;                  // summed slice per stage: 128 bytes of 16-bit elements
constexpr int ACC_COLS = 256;           // TMEM columns per accumulator
constexpr int FIRST_EPI = 4, EPI_WARPS = 8;
constexpr int THREADS = 32 * (FIRST_EPI + EPI_WARPS);
constexpr int A_BYTES = TM * 128;       // one stage of A
constexpr int CHUNK = TK * 128;         // MN-major: 64 columns by TK summed rows
constexpr int TURN = 32 * 64;           // epilogue staging: 32 rows of 64 bytes, SWIZZLE_64B
constexpr int TURNS = 2;                // pieces of it per warp, used in turn
constexpr int TURN_BYTES = EPI_WARPS * TURNS * TURN;
constexpr int MAX_STAGES = 8;
constexpr int SMEM_MAX = 232448 - 1024 - 512;  // opt-in limit less alignment and barriers

struct TileArgs {
    CUtensorMap a[2], b[2];
    int64_t M, N;       // output rows and columns (Dw: rows of one weight)
    int mt, nt;         // tiles of CG CTAs
    int whole, splits;  // tiles [0, whole) are one work item each, the others `splits` items each
    int cols_first;     // tile order: columns fastest, or rows
    int bn;             // output columns per tile
    int acc_n;          // MMA N
    int ksteps, kseg;   // summed slices over all segments, and per segment
    int stages, b_bytes;
    uint32_t idesc;
    Activation act;
    void* out[3];       // Forward: y, gate, up; Dx: dx; Dw: dwg, dwu
    int64_t ld[3];
    int tma[3];         // stored by TMA (whole groups through omap) and in 16-byte words; else by store_rows,
    int even[3];        // two elements a store
    CUtensorMap omap[3];
    float4* partial;    // split tiles: [slice][tile][CTA][column / 4][row]
    unsigned* err;
};

__device__ __forceinline__ float exp2f_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The larger of two values and the smaller, NaN where one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// __fdividef(1, d) is 0 for d above 2^126, as the quotient nearly is.
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// Where silu and its slope have reached their limits in fp32. Gates further out, infinite ones among them,
// are taken from there: v * sigmoid(v) is 0 for v = -inf, as for every large negative v, instead of inf * 0.
constexpr float SILU_END = 100.0f;

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// gelu(v) = v Phi(v), Phi the normal distribution, from its upper tail Q(z) = erfc(z / sqrt 2) / 2 at z = |v|:
// v Phi(v) = max(v, 0) - z Q(z), which does not cancel for negative v as v (1 + erf(v / sqrt 2)) / 2 does (at
// v = -5.5 that sum is a rounding error). Q(z) = e^(-z^2 / 2) P(t), P a polynomial in t = 1 / (1 + p z) without a
// constant term: the form of Hastings, Approximations for Digital Computers (1955), with p and the coefficients
// fitted here for the least relative error on [0, GELU_END], 7e-7 (1.0e-6 with fp32's roundings). The slope,
// Phi(v) + v e^(-v^2 / 2) / sqrt(2 pi), has the same exponential. From GELU_END on Q is 0 in fp32.
constexpr float GELU_END = 16.0f, GELU_P = 0.2658f;
__device__ constexpr float GELU_Q[7] = {0.105937719f,   0.107884675f, 0.084771432f,  0.137925252f,
                                        -0.0588914752f, 0.189003125f, -0.0666310787f};
// Q(z) for z in [0, GELU_END], and e^(-z^2 / 2).
__device__ __forceinline__ float normal_tail(float z, float* bell) {
    const float t = rcp_approx(fmaf(GELU_P, z, 1.0f));
    float q = GELU_Q[6];
#pragma unroll
    for (int i = 5; i >= 0; --i) q = fmaf(q, t, GELU_Q[i]);
    *bell = exp2f_approx(z * z * -0.72134752044448170f);
    return q * t * *bell;
}
// gelu of two values in packed fp32, with one reciprocal for both: 1 / a0 = a1 / (a0 a1).
__device__ __forceinline__ float2 gelu2(float2 v) {
    const float2 z = make_float2(fminf(fabsf(v.x), GELU_END), fminf(fabsf(v.y), GELU_END));  // NaN: GELU_END
    const float2 a = fma2(z, make_float2(GELU_P, GELU_P), make_float2(1.0f, 1.0f));
    const float r = rcp_approx(a.x * a.y);
    const float2 t = mul2(make_float2(a.y, a.x), make_float2(r, r));
    float2 q = make_float2(GELU_Q[6], GELU_Q[6]);
#pragma unroll
    for (int i = 5; i >= 0; --i) q = fma2(q, t, make_float2(GELU_Q[i], GELU_Q[i]));
    const float2 x = mul2(mul2(z, z), make_float2(-0.72134752044448170f, -0.72134752044448170f));
    q = mul2(mul2(q, t), make_float2(exp2f_approx(x.x), exp2f_approx(x.y)));
    return fma2(make_float2(-z.x, -z.y), q, make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f)));
}

template <Activation ACT>
__device__ __forceinline__ float act_value(float v) {
    if constexpr (ACT == Activation::Silu) v = max_nan(v, -SILU_END);
    if constexpr (ACT == Activation::Silu) return __fdividef(v, 1.0f + __expf(-v));
    else if constexpr (ACT == Activation::Gelu) {
        const float z = min_nan(fabsf(v), GELU_END);
        float bell;
        return fmaf(-z, normal_tail(z, &bell), fmaxf(v, 0.0f));
    } else if constexpr (ACT == Activation::Relu) return v > 0.0f ? v : (v != v ? v : 0.0f);
    else return sigmoid(v);
}
// The sigmoids of two values, in packed fp32, and product = a0 a1. They share one reciprocal,
// 1 / a0 = a1 / (a0 a1): the special function unit (16 lanes a clock on an SM) weighs on the epilogue of
// short sums, and this takes three of its operations instead of four. They hold where the product is at most
// PAIR_MAX, so that its reciprocal is a normal number: for gates whose negative parts add up to -86 at least.
constexpr float PAIR_MAX = 4.2535296e37f;  // 2^125
__device__ __forceinline__ float2 sigmoid2(float2 v, float* product) {
    const float2 x = mul2(v, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    const float2 a = add2(make_float2(exp2f_approx(x.x), exp2f_approx(x.y)), make_float2(1.0f, 1.0f));
    *product = a.x * a.y;
    const float r = rcp_approx(*product);
    return mul2(make_float2(a.y, a.x), make_float2(r, r));
}
// y = act(g) * u of the first `cols` of a row's 32 columns as 16 packed words. silu takes them in pairs (2^20
// rows of 128 x 128, sustained: 216 us; one value at a time 229), and all of them again one at a time where a
// pair does not hold (a NaN among them). The choice is the row's own: neither other rows nor what lies past
// its columns enter it. The second form is a loop over copies in local memory, two pairs at a time:
// unrolled, its instructions cost the first one 6 us, by four 1 us. All gates below -43: 485 us (648 by one pair,
// 415 by four).
template <Activation ACT, typename T>
__device__ __forceinline__ void gate_words(uint32_t (&w)[16], const uint32_t (&g)[32], const uint32_t (&u)[32], int cols) {
    if constexpr (ACT == Activation::Silu) {
        bool holds = true;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float2 g2 = make_float2(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1]));
            const float2 u2 = make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1]));
            float product;
            const float2 y = mul2(mul2(g2, sigmoid2(g2, &product)), u2);
            holds = holds && product <= PAIR_MAX;
            w[e] = pack2(y.x, y.y, T());
        }
        if (__builtin_expect(holds, 1)) return;
        float2 gs[16], us[16];
        uint32_t ws[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            gs[e] = make_float2(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1]));
            us[e] = make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1]));
        }
        if (cols < 32) {
            holds = true;
#pragma unroll 1
            for (int e = 0; 2 * e < cols; ++e) {
                float product;
                sigmoid2(gs[e], &product);
                holds = holds && product <= PAIR_MAX;
            }
            if (holds) return;
        }
#pragma unroll 2
        for (int e = 0; e < 16; ++e)
            ws[e] = pack2(act_value<ACT>(gs[e].x) * us[e].x, act_value<ACT>(gs[e].y) * us[e].y, T());
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = ws[e];
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float2 g2 = make_float2(__uint_as_float(g[2 * e]), __uint_as_float(g[2 * e + 1]));
            float2 v;
            if constexpr (ACT == Activation::Gelu) v = gelu2(g2);
            else v = make_float2(act_value<ACT>(g2.x), act_value<ACT>(g2.y));
            const float2 y = mul2(v, make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1])));
            w[e] = pack2(y.x, y.y, T());
        }
    }
}
// act(v) and act'(v).
template <Activation ACT>
__device__ __forceinline__ void act_both(float v, float* value, float* slope) {
    if constexpr (ACT == Activation::Silu) {
        const float low = max_nan(v, -SILU_END), s = sigmoid(low);
        *value = low * s;
        *slope = s * (1.0f + min_nan(low, SILU_END) * (1.0f - s));
    } else if constexpr (ACT == Activation::Gelu) {
        const float z = min_nan(fabsf(v), GELU_END);
        float bell;
        const float tail = normal_tail(z, &bell);
        *value = fmaf(-z, tail, fmaxf(v, 0.0f));
        *slope = fmaf(copysignf(z, v) * 0.39894228040143268f, bell, v > 0.0f ? 1.0f - tail : tail);
    } else if constexpr (ACT == Activation::Relu) {
        *value = act_value<ACT>(v);
        *slope = v > 0.0f ? 1.0f : 0.0f;
    } else {
        // s(|v|) and s(-|v|) from one exponential: 1 - s would cancel for large positive v
        const float e = exp2f_approx(fabsf(v) * -1.4426950408889634f), high = rcp_approx(1.0f + e), low = e * high;
        *value = v < 0.0f ? low : high;
        *slope = high * low;
    }
}

// dg = dy * up * act'(gate) and du = dy * act(gate) of 8 packed values. silu's sigmoids share a reciprocal by
// twos as in sigmoid2, and all 8 are taken again one at a time where a pair does not hold. In its slope
// 1 - s = e^-v s, which does not cancel. The arithmetic is on single values: packed fp32 needs aligned
// register pairs, and the one-pass gradient, which has no register to spare, spills for them (2^20 rows of
// 128: 329 us here, 351 us packed).
template <Activation ACT, typename T>
__device__ __forceinline__ void slope_words(uint32_t (&dg)[4], uint32_t (&du)[4], const uint32_t (&dy)[4],
                                            const uint32_t (&gate)[4], const uint32_t (&up)[4]) {
    auto words = [&](auto both) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 d = unpack2(dy[e], T()), g = unpack2(gate[e], T()), u = unpack2(up[e], T());
            float2 v, s;
            both(g, &v, &s);
            dg[e] = pack2(d.x * u.x * s.x, d.y * u.y * s.y, T());
            du[e] = pack2(d.x * v.x, d.y * v.y, T());
        }
    };
    if constexpr (ACT == Activation::Silu) {
        bool holds = true;
        words([&](float2 g, float2* value, float2* slope) {
            const float e0 = exp2f_approx(g.x * -1.4426950408889634f), e1 = exp2f_approx(g.y * -1.4426950408889634f);
            const float a0 = 1.0f + e0, a1 = 1.0f + e1, product = a0 * a1;
            const float r = rcp_approx(product), s0 = a1 * r, s1 = a0 * r;
            holds = holds && product <= PAIR_MAX;
            *value = make_float2(g.x * s0, g.y * s1);
            *slope = make_float2(s0 * (1.0f + fminf(g.x, SILU_END) * (e0 * s0)),
                                 s1 * (1.0f + fminf(g.y, SILU_END) * (e1 * s1)));
        });
        if (holds) return;
    }
    words([](float2 g, float2* value, float2* slope) {
        act_both<ACT>(g.x, &value->x, &slope->x);
        act_both<ACT>(g.y, &value->y, &slope->y);
    });
}

// Work item t: a tile and the summed slices [k0, k1) of it; part < 0, or its place among the partials.
struct Item {
    int mi, ni, k0, k1, part;
};
__device__ __forceinline__ void tile_place(const TileArgs& p, int tile, int* mi, int* ni) {
    *mi = p.cols_first ? tile / p.nt : tile % p.mt;
    *ni = p.cols_first ? tile % p.nt : tile / p.mt;
}
__device__ __forceinline__ Item item_of(const TileArgs& p, int t) {
    Item it{0, 0, 0, p.ksteps, -1};
    int tile = t;
    if (t >= p.whole) {
        const int rest = p.mt * p.nt - p.whole, s = (t - p.whole) / rest;
        it.part = t - p.whole;
        tile = p.whole + it.part - s * rest;
        it.k0 = (int)((int64_t)p.ksteps * s / p.splits);
        it.k1 = (int)((int64_t)p.ksteps * (s + 1) / p.splits);
    }
    tile_place(p, tile, &it.mi, &it.ni);
    return it;
}

template <typename F>
__host__ __device__ __forceinline__ void with_activation(Activation a, F&& f) {
    switch (a) {
        case Activation::Silu: return f(std::integral_constant<Activation, Activation::Silu>{});
        case Activation::Gelu: return f(std::integral_constant<Activation, Activation::Gelu>{});
        case Activation::Relu: return f(std::integral_constant<Activation, Activation::Relu>{});
        case Activation::Sigmoid: return f(std::integral_constant<Activation, Activation::Sigmoid>{});
    }
}

// ---- device helpers -------------------------------------------------------------------------------
// 32 TMEM lanes (this warp's quarter) x 32 consecutive columns; the caller waits (tmem_wait).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
        "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// The forms of a pair of CTAs (CG = 2) and of a single one. Barrier addresses are shared::cluster ones.
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// `p`'s counterpart in the shared memory of the pair's first CTA.
__device__ __forceinline__ uint32_t first_cta_addr(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
    return a;
}
template <int CG>
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        tc_mma(d, a, b, idesc, accumulate);
}
// Arrives on the barrier at this place in every CTA of the pair once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
            " [%0], %1;" ::"r"(smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
    else
        tc_commit(bar);
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc_all(uint32_t* slot) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(slot)),
                     "r"(2 * ACC_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(slot)),
                     "r"(2 * ACC_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free_all(uint32_t tmem) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(2 * ACC_COLS)
                     : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(2 * ACC_COLS)
                     : "memory");
}

// Shared-memory descriptors, SWIZZLE_128B (layout 2, version 1). K-major: rows of 128 bytes, 8-row
// atoms 1 KB apart. MN-major: 8 summed rows 1 KB apart, 64-column chunks CHUNK apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(CHUNK >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// The first `rows` x `cols` of a staged piece to `out` without TMA, V elements a store (1, or 2 where cols, ld and
// the address of `out` are even). Eight reads are in flight before their stores, which the compiler would
// not move a later read over. One copy in the program: three inlined ones do not stay in the instruction cache
// (2^18 rows of 128 -> 127, projections kept: 120 us, inlined 199; -> 126: 104 and 131; -> 128 by TMA 58).
// Aligned words of 4 or 8 bytes of odd rows, with their first and last elements stored singly, were slower
// (140 us and more): a row's piece is 64 bytes in any case, and they add stores to its ends.
template <typename T, int V>
__device__ __noinline__ void store_rows(T* out, int64_t ld, const uint8_t* at, int rows, int cols) {
    using Word = Pack<T, V>;
    constexpr int PER = 32 / V;  // lanes a row
    const int lane = threadIdx.x & 31, first = lane / PER, c = lane % PER * V;
    if (c >= cols) return;
    out += first * ld + c;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 8 * V) {
        Word w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + i * V + first;
            w[i] = *reinterpret_cast<const Word*>(at + r * 64 + (((c >> 3) ^ ((r >> 1) & 3)) * 16) + (c & 7) * 2);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (r0 + i * V + first < rows) *reinterpret_cast<Word*>(out + (int64_t)(r0 + i * V) * ld) = w[i];
    }
}

// A warp's 32 rows x 32 columns (lane = row, 16 packed words each) to output `o` at (row0, col0), turned
// through one of the warp's staging pieces. `rows` x `cols` of them are
// valid. ANY: outputs that TMA cannot address may be among the product's.
// Every call commits one bulk group, an empty one where it stores without TMA: the wait counts groups, and
// the newest PIECES - 1 of them have to be those of the other pieces' last calls.
template <typename T, bool ANY, int PIECES = TURNS>
__device__ __forceinline__ void store_group(const TileArgs& p, int o, uint8_t* turn, int& piece,
                                            const uint32_t (&w)[16], int64_t row0, int64_t col0,
                                            int rows, int cols) {
    const int lane = threadIdx.x & 31;
    uint8_t* at = turn + piece * TURN;
    piece = piece == PIECES - 1 ? 0 : piece + 1;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PIECES - 1) : "memory");
    __syncwarp();  // the piece's last store has read it
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(at + lane * 64 + ((i ^ ((lane >> 1) & 3)) * 16)) =
            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    if ((!ANY || p.tma[o]) && cols == 32) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            if (rows > 0)
                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                                 reinterpret_cast<uint64_t>(&p.omap[o])),
                             "r"((int)col0), "r"((int)row0), "r"(smem_u32(at))
                             : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    } else {
        __syncwarp();
        T* out = static_cast<T*>(p.out[o]) + row0 * p.ld[o] + col0;
        if (!ANY || p.tma[o]) {  // a tile's last columns, a multiple of 8: 16-byte pieces
            const int per = cols >> 3;
            for (int i = lane; i < rows * per; i += 32) {
                const int r = i / per, c = i - r * per;
                *reinterpret_cast<uint4*>(out + r * p.ld[o] + c * 8) =
                    *reinterpret_cast<const uint4*>(at + r * 64 + ((c ^ ((r >> 1) & 3)) * 16));
            }
        } else if (p.even[o]) {
            store_rows<T, 2>(out, p.ld[o], at, rows, cols);
        } else {
            store_rows<T, 1>(out, p.ld[o], at, rows, cols);
        }
        __syncwarp();
        if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}

// 32 accumulator columns as 16 words of the output type.
template <typename T>
__device__ __forceinline__ void pack_words(uint32_t (&w)[16], const uint32_t (&v)[32]) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
        w[e] = pack2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]), T());
}

// The first `cols` (a multiple of 4) of 32 accumulator columns of a split tile's slice: lane = row, a
// warp's store covers 512 contiguous bytes.
__device__ __forceinline__ void store_partial(float4* dst, const uint32_t (&v)[32], int cols) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (4 * e < cols)
            dst[e * TM] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                      __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
}

// ---- the kernel -------------------------------------------------------------------------------------
template <typename T, Product P, int CG, bool ANY>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ TileArgs p) {
    static_assert(P != Product::Dw || CG == 2, "Dw: one weight a CTA");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stage_bytes = A_BYTES + p.b_bytes;
    uint8_t* turn = smem + p.stages * stage_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(turn + TURN_BYTES);
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

    const int work = p.whole + (p.mt * p.nt - p.whole) * p.splits;
    const int group = blockIdx.x / CG, groups = gridDim.x / CG;

    if (warp == 0) {
        if (lane == 0 && rank == 0) {
            int s = 0, turn = 0;  // the next stage, and whether its ring has come round an odd number of times
            bool ok = true;
            for (int t = group, i = 0; t < work && ok; t += groups, ++i) {
                const int b = i & 1;
                if (i >= 2 && !mbar_wait(&acc_empty[b], ((i >> 1) - 1) & 1, p.err)) break;
                tc_fence_after();
                const uint32_t acc = tmem + (uint32_t)(b * ACC_COLS);
                const Item it = item_of(p, t);
                for (int k = it.k0; k < it.k1; ++k) {
                    const uint32_t sa = smem_u32(smem + s * stage_bytes), sb = sa + A_BYTES;
                    const uint64_t da = P == Product::Dw ? desc_mn(sa) : desc_k(sa);
                    const uint64_t db = P == Product::Forward ? desc_k(sb) : desc_mn(sb);
                    if (!mbar_wait(&full[s], turn, p.err)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    // 16 summed elements: 32 bytes along a K-major row, 2 KB of MN-major rows, in units of 16
#pragma unroll
                    for (int q = 0; q < TK / 16; ++q)
                        pair_mma<CG>(acc, da + q * (P == Product::Dw ? 128 : 2), db + q * (P == Product::Forward ? 2 : 128),
                                     p.idesc, k > it.k0 || q > 0);
                    pair_commit<CG>(&empty[s]);
                    if (++s == p.stages) s = 0, turn ^= 1;
                }
                if (ok) pair_commit<CG>(&acc_full[b]);
            }
            pair_commit<CG>(done);  // arrives at once where nothing was issued
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int s = 0, turn = 0, held = 0;  // held: stages filled, at most all
            bool ok = true;
            for (int t = group; t < work && ok; t += groups) {
                const Item it = item_of(p, t);
                const int m0 = (P == Product::Dw ? it.mi : it.mi * CG + rank) * TM;
                const int n0 = it.ni * p.bn;
                for (int k = it.k0; k < it.k1; ++k) {
                    if (held == p.stages && !mbar_wait(&empty[s], turn ^ 1, p.err)) {
                        ok = false;
                        break;
                    }
                    if (held < p.stages) ++held;
                    uint8_t* sa = smem + s * stage_bytes;
                    uint8_t* sb = sa + A_BYTES;
                    if (rank == 0) mbar_expect_tx(&full[s], (uint32_t)(CG * stage_bytes));
                    const uint32_t bar = CG == 2 ? first_cta_addr(&full[s]) : smem_u32(&full[s]);
                    if constexpr (P == Product::Forward) {
                        pair_load<CG>(sa, &p.a[0], k * TK, m0, bar);
                        if constexpr (CG == 2) {
                            pair_load<CG>(sb, &p.b[rank], k * TK, n0, bar);
                        } else {
                            pair_load<CG>(sb, &p.b[0], k * TK, n0, bar);
                            pair_load<CG>(sb + p.bn * 128, &p.b[1], k * TK, n0, bar);
                        }
                    } else {
                        const int nb = n0 + rank * (p.acc_n / CG);  // this CTA's columns of B
                        if constexpr (P == Product::Dx) {
                            const int seg = k >= p.kseg, kk = (k - seg * p.kseg) * TK;
                            pair_load<CG>(sa, &p.a[seg], kk, m0, bar);
                            for (int c = 0; c * CHUNK < p.b_bytes; ++c)
                                pair_load<CG>(sb + c * CHUNK, &p.b[seg], nb + 64 * c, kk, bar);
                        } else {
                            for (int c = 0; c < TM / 64; ++c)
                                pair_load<CG>(sa + c * CHUNK, &p.a[rank], m0 + 64 * c, k * TK, bar);
                            for (int c = 0; c * CHUNK < p.b_bytes; ++c)
                                pair_load<CG>(sb + c * CHUNK, &p.b[0], nb + 64 * c, k * TK, bar);
                        }
                    }
                    if (++s == p.stages) s = 0, turn ^= 1;
                }
            }
            // No load may be in flight when the CTA ends. Each landed before its MMAs ran, and the commit
            // after those freed its stage (they have all done so unless a wait ran out).
            for (; held > 0; --held) {
                if (s-- == 0) s = p.stages - 1, turn ^= 1;
                mbar_wait(&empty[s], turn, p.err);
            }
        }
    } else if (warp >= FIRST_EPI) {
        const int quarter = warp & 3, half = (warp - FIRST_EPI) >> 2;
        uint8_t* my_turn = turn + (warp - FIRST_EPI) * TURNS * TURN;
        int piece = 0;
        for (int t = group, i = 0; t < work; t += groups, ++i) {
            const int b = i & 1;
            if (!mbar_wait(&acc_full[b], (i >> 1) & 1, p.err)) break;
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * ACC_COLS);
            const Item it = item_of(p, t);
            const int seg = P == Product::Dw ? rank : 0;
            const int64_t row0 = (int64_t)(P == Product::Dw ? it.mi : it.mi * CG + rank) * TM + quarter * 32;
            const int64_t n0 = (int64_t)it.ni * p.bn;
            float4* partial = p.partial + ((int64_t)it.part * CG + rank) * (ACC_COLS / 4) * TM + quarter * 32 + lane;
            const int rows = (int)max((int64_t)0, min((int64_t)32, p.M - row0));
            const int ncols = (int)min((int64_t)p.bn, p.N - n0);
            for (int c = half * 32; c < ncols; c += 64) {
                const int cols = min(32, ncols - c);
                uint32_t v[32], u[32], w[16];
                tmem_ld32(acc + (uint32_t)c, v);
                if constexpr (P == Product::Forward) tmem_ld32(acc + (uint32_t)(p.bn + c), u);
                tmem_wait();
                if (it.part >= 0) {
                    store_partial(partial + c / 4 * TM, v, p.bn - c);
                    if constexpr (P == Product::Forward) store_partial(partial + (p.bn + c) / 4 * TM, u, p.bn - c);
                } else if constexpr (P == Product::Forward) {
                    with_activation(p.act, [&](auto act) { gate_words<decltype(act)::value, T>(w, v, u, cols); });
                    store_group<T, ANY>(p, 0, my_turn, piece, w, row0, n0 + c, rows, cols);
                    if (p.out[1]) {
                        pack_words<T>(w, v);
                        store_group<T, ANY>(p, 1, my_turn, piece, w, row0, n0 + c, rows, cols);
                    }
                    if (p.out[2]) {
                        pack_words<T>(w, u);
                        store_group<T, ANY>(p, 2, my_turn, piece, w, row0, n0 + c, rows, cols);
                    }
                } else {
                    pack_words<T>(w, v);
                    store_group<T, ANY>(p, seg, my_turn, piece, w, row0, n0 + c, rows, cols);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) arrive_cluster(first_cta_addr(&acc_empty[b]));
                else mbar_arrive(&acc_empty[b]);
            }
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

// Adds the slices of the split tiles and finishes them. A CTA takes 4 rows x 32 columns; its eight warps
// add every eighth slice, and the eight sums are added in order: one fixed order for each size.
template <typename T, Product P, int CG>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TileArgs p) {
    __shared__ float4 red[2][8][32];
    cudaGridDependencySynchronize();
    const int rest = p.mt * p.nt - p.whole, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int groups = (p.bn + 31) / 32;  // per tile: 32 columns each, by 32 slabs of 4 rows
    const int64_t slice = (int64_t)rest * CG * (ACC_COLS / 4) * TM;  // float4s
    const int slab = (int)(blockIdx.x % (TM / 4)), grp = (int)(blockIdx.x / (TM / 4) % groups);
    const int part = (int)(blockIdx.x / (TM / 4) / groups), rank = part % CG;
    int mi, ni;
    tile_place(p, p.whole + part / CG, &mi, &ni);
    const int r = slab * 4 + (lane & 3), c4 = grp * 8 + (lane >> 2);
    const int64_t row = (int64_t)(P == Product::Dw ? mi : mi * CG + rank) * TM + r;
    const int64_t col = (int64_t)ni * p.bn + c4 * 4;
    const bool in = row < p.M && col < p.N && c4 * 4 < p.bn;
    const float4* src = p.partial + (int64_t)part * (ACC_COLS / 4) * TM + r;
    auto sum = [&](int column4) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (in)
#pragma unroll 4
            for (int i = warp; i < p.splits; i += 8) {
                const float4 v = src[(int64_t)column4 * TM + i * slice];
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
        return s;
    };
    red[0][warp][lane] = sum(c4);
    if (P == Product::Forward) red[1][warp][lane] = sum(p.bn / 4 + c4);
    __syncthreads();
    if (warp > 0 || !in) return;
    auto total = [&](int which) {
        float4 s = red[which][0][lane];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            const float4 v = red[which][i][lane];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        return s;
    };
    auto put = [&](int o, float4 s) {
        T* dst = static_cast<T*>(p.out[o]) + row * p.ld[o] + col;
        if (p.tma[o] && col + 4 <= p.N) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(s.x, s.y, T()), pack2(s.z, s.w, T()));
        } else {
            const float e[4] = {s.x, s.y, s.z, s.w};
            for (int i = 0; i < 4 && col + i < p.N; ++i) dst[i] = from_float<T>(e[i]);
        }
    };
    const float4 g = total(0);
    if constexpr (P == Product::Forward) {
        const float4 u = total(1);
        with_activation(p.act, [&](auto act) {
            constexpr Activation A = decltype(act)::value;
            put(0, make_float4(act_value<A>(g.x) * u.x, act_value<A>(g.y) * u.y, act_value<A>(g.z) * u.z,
                               act_value<A>(g.w) * u.w));
        });
        if (p.out[1]) put(1, g);
        if (p.out[2]) put(2, u);
    } else {
        put(P == Product::Dw ? rank : 0, g);
    }
}

// ---- host -----------------------------------------------------------------------------------------
// Instruction descriptor, kind::f16: fp32 accumulator, operand types and orders, N / 8, M / 16.
inline uint32_t make_idesc(bool bf16, bool a_mn, bool b_mn, int m, int n) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) |
           (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Whether TMA can address rows of a 16-bit matrix: 16-byte base and row stride (below 2^40 bytes).
inline bool tma_ok(const void* p, int64_t ld) {
    return aligned_to(p, 16) && ld % 8 == 0 && ld < (int64_t(1) << 39);
}

// Sets output `i`: an M x N matrix (or none) with row stride ld. A TMA store writes whole 16-byte pieces of
// a row, so its rows have to end on one.
inline void set_output(TileArgs& t, int i, void* out, int64_t ld) {
    if (out && t.M == 1) ld = t.N;  // the stride of a single row is never taken
    t.out[i] = out;
    t.ld[i] = ld;
    t.tma[i] = out && t.N % 8 == 0 && tma_ok(out, ld);
    t.even[i] = t.N % 2 == 0 && ld % 2 == 0 && aligned_to(out, 4);
    if (t.tma[i])
        t.omap[i] = make_map_2d(out, (uint64_t)t.N, (uint64_t)t.M, (uint64_t)ld * 2, 32, 32,
                                CU_TENSOR_MAP_SWIZZLE_64B);
}

// Accumulator columns (MMA N) of a tile of bn output columns: a multiple of 16, in a pair of 32.
template <Product P, int CG>
int acc_columns(int bn) {
    return P == Product::Forward ? 2 * bn : (bn + 16 * CG - 1) / (16 * CG) * 16 * CG;
}

// Fills in what follows from `t`'s maps, sizes, outputs and bn, launches, and joins the slices.
template <typename T, Product P, int CG>
void launch_product(Handle& h, TileArgs& t) {
    constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    t.acc_n = acc_columns<P, CG>(t.bn);
    const int own = t.acc_n / CG;  // a CTA's columns of B
    t.b_bytes = P == Product::Forward ? own * 128 : (own + 63) / 64 * CHUNK;
    t.idesc = make_idesc(bf16, P == Product::Dw, P != Product::Forward, TM * CG, t.acc_n);
    t.stages = std::min<int>(MAX_STAGES, (SMEM_MAX - TURN_BYTES) / (A_BYTES + t.b_bytes));
    t.err = h.d_err;
    const size_t smem = 1024 + (size_t)t.stages * (A_BYTES + t.b_bytes) + TURN_BYTES + 512;
    const int64_t rest = (int64_t)t.mt * t.nt - t.whole;  // split tiles
    const int64_t work = t.whole + rest * t.splits;
    XS_REQUIRE(work * CG < (int64_t(1) << 31), XSPMM_STATUS_UNSUPPORTED, "grid too large");
    DevBuf<float4> ws((size_t)rest * t.splits * CG * (ACC_COLS / 4) * TM, h.stream);
    t.partial = ws.get();
    bool any = false;
    for (int i = 0; i < 3; ++i) any = any || (t.out[i] && !t.tma[i]);
    auto kern = any ? tile_kernel<T, P, CG, true> : tile_kernel<T, P, CG, false>;
    allow_smem(kern, 1024 + SMEM_MAX + 512);
    const unsigned grid = (unsigned)(std::min<int64_t>(work, sm_count(h.device) / CG) * CG);
    launch_dependent(h.stream, kern, grid, THREADS, smem, CG, t);
    after_launch(h, "gated_product");
    if (rest > 0) {
        const int64_t blocks = rest * CG * ((t.bn + 31) / 32) * (TM / 4);
        launch_dependent(h.stream, join_kernel<T, P, CG>, (unsigned)blocks, 256, 0, 1, t);
        after_launch(h, "gated_join");
    }
}

}  // namespace gated
}  // namespace xspmm_b200
