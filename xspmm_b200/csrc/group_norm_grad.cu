// group_norm_grad.cu -- the gradient of the group norm with an activation.
//
// xh = (x - mean) * rstd, z = xh * w + b, dz = dy * act'(z). Per sample and channel, A = sum of dz and B = sum of
// dz * xh over the rows; dw = sum of B and db = sum of A over the samples. With t = dz * w the means over a group's n
// values are m1 = sum_c w A / n and m2 = sum_c w B / n, and dx = rstd * (t - m1 - xh * m2). So one pass over x and dy
// for A and B serves the weights and the groups, and a second one gives dx.
//
// Who takes which samples is decided as in the forward pass (group_norm.cu). The sums for the weights' gradients are
// kept for each thread over all samples that its CTA takes (at most TERMS) and leave as one row a CTA (or chunk), added in
// order and in 64 bits by the last kernel; a block of several tiles has no room for them and adds them to its CTA's row
// as it goes.
//
// 2^20 x 128 fp16, relu: 256 us (206 for both inputs read twice at the copy bandwidth), DRAM at 5.1 and 5.3 TB/s. 4096 samples
// of 2^18 x 256 bf16, silu: 223 to 228 us (62), bound by instructions: 44 for each value of a lane, issue in 46 % of the cycles,
// misses of the instruction cache the most frequent wait. The slope is computed in both passes: dz would take half as much
// shared memory again, and fewer samples would stay there.
#include "group_norm.cuh"

namespace xspmm_b200 {
namespace {

using namespace group;

constexpr int CTAS = 4;  // that an SM should hold: 128 registers a thread and
constexpr int SLOT_BYTES = 336;  // of shared memory a thread for rows of x and dy

template <typename TX, typename TY>
struct Backward {
    GroupNormArgs<TX> a;
    Tiling t;
    Chunks ch;
    int walkers;        // CTAs a block that walk over samples, 0 where all samples are long
    int each;           // neighbouring samples that one of them takes
    bool by_warp;       // short ones by a warp each
    const TY* dy;
    int64_t lddy;
    const float *mean, *rstd;
    TY* dx;  // or null
    int64_t lddx;
    float* weights;  // [walker, then chunk][2][channel]: sums of dz * xh and dz, or null
    float *dw, *db;  // not null: the only walker's, which leaves its sums there at once
    float2* part;    // Parts: sums of w A and w B
    int2* found;     // [chunk]: the long samples with rows in it
};

// A thread's view of its channels: the parameters, and a sample's statistics (minus the mean).
template <int P>
struct Channels {
    float2 w[P], b[P], m[P], rs[P];
};
template <int P>
struct Sums {
    float2 a[P] = {}, b[P] = {};
    __device__ void add(const Sums& o) {
#pragma unroll
        for (int e = 0; e < P; ++e) a[e] = pair_add(a[e], o.a[e]), b[e] = pair_add(b[e], o.b[e]);
    }
};
// A thread's sums over all samples that its CTA takes, in shared memory: touched once a sample.
template <int P>
struct Totals {
    float2 (*v)[THREADS];  // [2 P]
    __device__ void clear() const {
#pragma unroll
        for (int e = 0; e < 2 * P; ++e) v[e][threadIdx.x] = make_float2(0.0f, 0.0f);
    }
    __device__ void add(const Sums<P>& s) const {
#pragma unroll
        for (int e = 0; e < P; ++e) {
            v[e][threadIdx.x] = pair_add(v[e][threadIdx.x], s.a[e]);
            v[P + e][threadIdx.x] = pair_add(v[P + e][threadIdx.x], s.b[e]);
        }
    }
    __device__ Sums<P> get() const {
        Sums<P> s;
#pragma unroll
        for (int e = 0; e < P; ++e) s.a[e] = v[e][threadIdx.x], s.b[e] = v[P + e][threadIdx.x];
        return s;
    }
};

// A thread's slots for rows of both inputs.
template <typename TX, typename TY, int V, int U>
struct Pairs {
    static constexpr int BYTES = Slots<TX, V, U>::BYTES + Slots<TY, V, U>::BYTES, ROWS = SLOT_BYTES / BYTES, RING = ROWS / BATCH;
    Slots<TX, V, U> x;
    Slots<TY, V, U> g;
    __device__ Pairs(uint8_t* memory) : x{memory}, g{memory + ROWS * THREADS * Slots<TX, V, U>::BYTES} {}
};

enum class Rows { Fill, Kept, Pass };  // to the slots and stay there; there already; through a ring

// Calls f(dz, xh) for this thread's rows of [begin, end) in order, or with BACK from the last.
template <bool CTA, Rows HOW, bool BACK, typename TX, typename TY, int V, int U, typename F>
__device__ __forceinline__ void each_row(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm, const Pairs<TX, TY, V, U>& slots,
                                         const Tile& k, int begin, int end, const Channels<V * U / 2>& ch, F&& f) {
    constexpr int P = V * U / 2;
    const int rows = tm.rows(end - begin);
    auto fx = tm.template walk<BACK>(p.a.x + k.c0, begin, rows, p.a.ldx);
    auto fg = tm.template walk<BACK>(p.dy + k.c0, begin, rows, p.lddy);
    auto fill = [&](int slot) {
        slots.x.fill(slot, fx.next(), tm.at);
        slots.g.fill(slot, fg.next(), tm.at);
    };
    if constexpr (HOW == Rows::Fill) fill_all(rows, fill);
    with_act(p.a.act, [&](auto act) {
        constexpr Activation ACT = decltype(act)::value;
        auto use = [&](auto full, int slot) {
#pragma unroll
            for (int j = 0; j < (decltype(full)::value ? BATCH : 1); ++j) {
                Pack<TX, V> rx[U];
                Pack<TY, V> rg[U];
                slots.x.get(rx, slot + j);
                slots.g.get(rg, slot + j);
                float2 dz[P], xh[P];
                Place<V, U>::values(rx, xh);
                Place<V, U>::values(rg, dz);
#pragma unroll
                for (int e = 0; e < P; ++e) xh[e] = centred(xh[e], ch.m[e], ch.rs[e]);
                if constexpr (ACT != Activation::None) {
                    float2 z[P];
#pragma unroll
                    for (int e = 0; e < P; ++e) z[e] = affine(xh[e], ch.w[e], ch.b[e]);
                    act_row<true, sizeof(TY) == 4, ACT>(z);
#pragma unroll
                    for (int e = 0; e < P; ++e) dz[e] = pair_mul(dz[e], z[e]);
                }
                f(dz, xh);
            }
        };
        if constexpr (HOW == Rows::Pass) stream<Pairs<TX, TY, V, U>::RING>(rows, fill, use);
        else use_all(rows, use);
    });
}

// This thread's A and B over rows [begin, end), added to `total`, and the groups' sums of w A and w B, which one thread
// a group hands to f(group of the tile, sum, sum). channels(strips) is called between, once the tile's A and B are
// there by channel. The strips may be written again after a team_sync.
template <bool CTA, Rows HOW, typename TX, typename TY, int V, int U, typename F, typename C>
__device__ __forceinline__ void group_sums(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm,
                                           const Pairs<TX, TY, V, U>& slots, const Tile& k, int begin, int end,
                                           const Channels<V * U / 2>& ch, const Totals<V * U / 2>& total,
                                           Strips& sh, F&& f, C&& channels) {
    constexpr int P = V * U / 2;
    Sums<P> s;
    auto add = [&](int b, int e) {
        Sums<P> part;
        each_row<CTA, HOW, false>(p, tm, slots, k, b, e, ch, [&](const float2 (&dz)[P], const float2 (&xh)[P]) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                part.a[i] = pair_add(part.a[i], dz[i]);
                part.b[i] = pair_fma(dz[i], xh[i], part.b[i]);
            }
        });
        s.add(part);
    };
    if constexpr (HOW == Rows::Pass) {
        const int most = TERMS << tm.step_log;
#pragma unroll 1
        for (int b = begin; b < end; b += most) add(b, min(end, b + most));
    } else {
        add(begin, end);
    }
    total.add(s);
    sum_channels<CTA>(s.a, s.b, tm.at, sh);
    const int strip = CTA ? 0 : threadIdx.x >> 5;
    channels(sh.v[strip]);
    if (!p.dx) return;
    each_group<CTA>(k.ng, [&](int g, int j, int l, bool live) {
        float s1 = 0.0f, s2 = 0.0f;
        if (live)
            for (int c = j; c < k.lw; c += l) {
                const int at = g * k.lw + c;
                const float w = p.a.w ? __ldg(p.a.w + k.c0 + at) : 1.0f;
                s1 = fmaf(w, sh.v[strip][0][at], s1);
                s2 = fmaf(w, sh.v[strip][1][at], s2);
            }
        s1 = group_sum(s1, l);
        s2 = group_sum(s2, l);
        if (live && j == 0) f(g, s1, s2);
    });
}

// dx of rows [begin, end) from the groups' minus m1 and minus m2.
template <bool CTA, Rows HOW, bool BACK, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void apply(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm,
                                      const Pairs<TX, TY, V, U>& slots, const Tile& k, int begin, int end,
                                      const Channels<V * U / 2>& ch, const float* g1, const float* g2) {
    constexpr int P = V * U / 2;
    float2 m1[P], m2[P];
    tm.of_groups(m1, g1, k);
    tm.of_groups(m2, g2, k);
    auto to = tm.template walk<BACK>(p.dx + k.c0, begin, tm.rows(end - begin), p.lddx);
    each_row<CTA, HOW, BACK>(p, tm, slots, k, begin, end, ch, [&](const float2 (&dz)[P], const float2 (&xh)[P]) {
        float2 v[P];
#pragma unroll
        for (int e = 0; e < P; ++e)  // t rounded by itself: a group's only value has dx = 0, not a rounding times rstd
            v[e] = pair_mul(ch.rs[e], pair_fma(xh[e], m2[e], pair_add(pair_mul_alone(dz[e], ch.w[e]), m1[e])));
        tm.at.store(to.next(), v);
    });
}

template <bool CTA, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void parameters(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm, const Tile& k,
                                           Channels<V * U / 2>& ch) {
    tm.at.param(ch.w, p.a.w, k.c0, 1.0f);
    tm.at.param(ch.b, p.a.b, k.c0, 0.0f);
}
template <bool CTA, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void statistics(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm, const Tile& k, int s,
                                           Channels<V * U / 2>& ch) {
    tm.of_groups(ch.m, p.mean + (int64_t)s * p.t.groups + k.g0, k);
    tm.of_groups(ch.rs, p.rstd + (int64_t)s * p.t.groups + k.g0, k);
#pragma unroll
    for (int e = 0; e < V * U / 2; ++e) ch.m[e] = make_float2(-ch.m[e].x, -ch.m[e].y);
}

// The CTA's sums of a tile's channels to row `row` of the weights' parts, or to their place.
template <typename TX, typename TY, int V, int U>
__device__ __forceinline__ void leave_weights(const Backward<TX, TY>& p, int64_t row, const Tile& k, const Place<V, U>& at,
                                              const Totals<V * U / 2>& total, Strips& sh) {
    Sums<V * U / 2> s = total.get();
    sum_channels<true>(s.a, s.b, at, sh);
    if ((int)threadIdx.x >= k.cols) return;
    const int c = k.c0 + threadIdx.x;
    if (p.weights) {
        float* out = p.weights + row * 2 * p.a.C + c;
        out[0] = sh.v[0][1][threadIdx.x];
        out[p.a.C] = sh.v[0][0][threadIdx.x];
    } else {
        if (p.dw) p.dw[c] = sh.v[0][1][threadIdx.x];
        if (p.db) p.db[c] = sh.v[0][0][threadIdx.x];
    }
}

// A sample by a team. KEEP: it is one tile and fits the slots. `total` is the CTA's sums where a block is one tile; else
// they go to the CTA's row.
template <bool CTA, bool KEEP, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void whole_sample(const Backward<TX, TY>& p, const Pairs<TX, TY, V, U>& slots, int s, Span rows, int block,
                                             int64_t row,
                                             Channels<V * U / 2>& ch, const Totals<V * U / 2>& total, Strips& sh, float* g1,
                                             float* g2) {
    const int tpg = KEEP ? 1 : p.t.tpg, t0 = block * tpg;
    const bool one = tpg == 1;
    for (int j = 0; j < tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        if (!one) parameters(p, tm, k, ch);
        if (one || j == 0) statistics(p, tm, k, s, ch);
        const float per = -1.0f / ((float)(rows.end - rows.begin) * (float)p.t.width);
        group_sums<CTA, KEEP ? Rows::Fill : Rows::Pass>(p, tm, slots, k, rows.begin, rows.end, ch, total, sh,
                           [&](int g, float s1, float s2) {
                               if (j > 0) s1 += g1[g], s2 += g2[g];  // the same thread's sums of the tiles before
                               const bool last = j + 1 == tpg;
                               g1[g] = last ? s1 * per : s1;
                               g2[g] = last ? s2 * per : s2;
                           },
                           [&](const float (&v)[2][MAX_TILE]) {
                               if (CTA && !one && p.weights && (int)threadIdx.x < k.cols) {
                                   float* out = p.weights + row * 2 * p.a.C + k.c0 + threadIdx.x;
                                   out[0] += v[1][threadIdx.x];
                                   out[p.a.C] += v[0][threadIdx.x];
                               }
                           });
        team_sync<CTA>();
    }
    if (!p.dx) return;
    for (int j = 0; j < tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        if (!one) parameters(p, tm, k, ch);
        apply<CTA, KEEP ? Rows::Kept : Rows::Pass, false>(p, tm, slots, k, rows.begin, rows.end, ch, g1, g2);
    }
    team_sync<CTA>();
}

// CTAs [0, chunks x tiles): sums of the long samples' chunks. The others: short and middle samples.
template <typename TX, typename TY, int V, int U>
__global__ void __launch_bounds__(THREADS, CTAS) group_norm_grad_kernel(const __grid_constant__ Backward<TX, TY> p) {
    __shared__ Strips sh;
    __shared__ float g1[WARPS][MAX_TILE], g2[WARPS][MAX_TILE];
    __shared__ float2 totals[V * U][THREADS];
    extern __shared__ __align__(16) uint8_t slot_memory[];
    const Pairs<TX, TY, V, U> slots(slot_memory);
    constexpr int ROWS = Pairs<TX, TY, V, U>::ROWS;
    cudaGridDependencySynchronize();
    const int chunked = p.ch.count * p.t.tiles, warp = threadIdx.x >> 5;
    Channels<V * U / 2> ch;
    const Totals<V * U / 2> total{totals};
    total.clear();
    if ((int)blockIdx.x < chunked) {
        const int i = blockIdx.x / p.t.tiles, tile = blockIdx.x - i * p.t.tiles;
        const int2 found = long_samples(p.a.offsets, (int)p.a.samples, (int)p.a.rows, p.ch, i);
        if (tile == 0 && threadIdx.x == 0) p.found[i] = found;
        const Tile k = tile_of(p.t, tile);
        const Team<true, V, U> tm(p.t, k.cols);
        const int all = (int)p.a.rows, r0 = i * p.ch.rows, r1 = r0 + min(p.ch.rows, all - r0);
        const int64_t parts = p.t.tpg == 1 ? p.t.groups : p.t.tiles;
        parameters(p, tm, k, ch);
        for (int slot = 0; slot < 2; ++slot) {
            const int s = slot ? found.y : found.x;
            if (s < 0) continue;
            const Span sp = span_of(p.a.offsets, s, all);
            float2* out = p.part + (slot * parts + part_slot(p.t, tile, k)) * p.ch.count + i;
            statistics(p, tm, k, s, ch);
            group_sums<true, Rows::Pass>(p, tm, slots, k, max(r0, sp.begin), min(r1, sp.end), ch, total, sh,
                                [&](int g, float s1, float s2) { out[(int64_t)g * p.ch.count] = make_float2(s1, s2); },
                                [](const float (&)[2][MAX_TILE]) {});
            __syncthreads();
        }
        if (p.weights) leave_weights(p, p.walkers + i, k, tm.at, total, sh);
        return;
    }
    const int at = blockIdx.x - chunked, walker = p.t.blocks == 1 ? at : at / p.t.blocks, block = at - walker * p.t.blocks;
    const Tile k = tile_of(p.t, block * p.t.tpg);
    const Team<true, V, U> tm(p.t, k.cols);
    const bool one = p.t.tpg == 1;
    if (one) {
        parameters(p, tm, k, ch);
    } else if (p.weights) {
        float* out = p.weights + (int64_t)walker * 2 * p.a.C + k.c0;
        for (int c = threadIdx.x; c < p.t.width; c += THREADS) out[c] = out[p.a.C + c] = 0.0f;
        __syncthreads();
    }
    auto rows_of = [&](int s) { return span_of(p.a.offsets, s, (int)p.a.rows); };
    const int s0 = walker * p.each, s1 = s0 + min(p.each, (int)p.a.samples - s0);
    const int warp_rows = p.by_warp ? ROWS << (5 - p.t.lpr_log) : 0;  // most that a warp takes
    if (p.by_warp) {
        for (int s = s0 + warp; s < s1; s += WARPS) {
            const Span sp = rows_of(s);
            if (sp.end > sp.begin && sp.end - sp.begin <= warp_rows)
                whole_sample<false, true>(p, slots, s, sp, block, walker, ch, total, sh, g1[warp], g2[warp]);
        }
        __syncthreads();
    }
    for (int s = s0; s < s1; ++s) {
        const Span sp = rows_of(s);
        const int n = sp.end - sp.begin;
        if (n <= warp_rows || n > p.ch.longest) continue;
        if (one && n <= (ROWS << (5 + WARPS_LOG - p.t.lpr_log)))
            whole_sample<true, true>(p, slots, s, sp, block, walker, ch, total, sh, g1[0], g2[0]);
        else whole_sample<true, false>(p, slots, s, sp, block, walker, ch, total, sh, g1[0], g2[0]);
    }
    if (one && (p.weights || p.dw || p.db)) leave_weights(p, walker, k, tm.at, total, sh);
}

// dx of the long samples' chunks. Every CTA joins the sums of its tile's groups over all of the sample's chunks.
template <typename TX, typename TY, int V, int U>
__global__ void __launch_bounds__(THREADS, CTAS) group_norm_grad_apply_kernel(const __grid_constant__ Backward<TX, TY> p) {
    __shared__ float g1[MAX_TILE], g2[MAX_TILE];
    extern __shared__ __align__(16) uint8_t slot_memory[];
    const Pairs<TX, TY, V, U> slots(slot_memory);
    cudaGridDependencySynchronize();
    const int i = p.ch.count - 1 - blockIdx.x / p.t.tiles, tile = blockIdx.x % p.t.tiles;
    const int2 found = p.found[i];
    if (found.x < 0 && found.y < 0) return;
    const Tile k = tile_of(p.t, tile);
    const Team<true, V, U> tm(p.t, k.cols);
    const int all = (int)p.a.rows, r0 = i * p.ch.rows, r1 = r0 + min(p.ch.rows, all - r0);
    const int tpg = p.t.tpg, lane = threadIdx.x & 31;
    Channels<V * U / 2> ch;
    parameters(p, tm, k, ch);
    for (int slot = 1; slot >= 0; --slot) {
        const int s = slot ? found.y : found.x;
        if (s < 0) continue;
        const Span sp = span_of(p.a.offsets, s, all);
        const Parts parts(sp, p.ch, tpg == 1 ? p.t.groups : p.t.tiles);
        const bool lost = not_found(p.found, parts, s);
        const float per = lost ? __uint_as_float(0x7fc00000u) : -1.0f / ((float)(sp.end - sp.begin) * (float)p.t.width);
        for (int g = threadIdx.x >> 5; g < k.ng; g += WARPS) {
            float s1 = 0.0f, s2 = 0.0f;
            for (int part = 0; part < tpg; ++part)
#pragma unroll 8
                for (int c = lane; c < parts.count; c += 32) {
                    const float2 v = parts.get(p.part, (int64_t)(k.g0 + g) * tpg + part, c);
                    s1 += v.x;
                    s2 += v.y;
                }
            s1 = group_sum(s1, 32);
            s2 = group_sum(s2, 32);
            if (lane == 0) g1[g] = s1 * per, g2[g] = s2 * per;
        }
        __syncthreads();
        statistics(p, tm, k, s, ch);
        apply<true, Rows::Pass, true>(p, tm, slots, k, max(r0, sp.begin), min(r1, sp.end), ch, g1, g2);
    }
}

// dw and db: the rows of parts added in order, 32 channels a CTA; its warps take every 32nd. In 64 bits: there may be as
// many rows as samples.
__global__ void __launch_bounds__(1024) group_norm_weights_kernel(const float* part, int rows, int64_t C, float* dw, float* db) {
    __shared__ double red[32][33];
    cudaGridDependencySynchronize();
    float* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = blockIdx.x * 32ll + lane;
    double s = 0.0;
    if (c < C)
#pragma unroll 8
        for (int r = warp; r < rows; r += 32) s += (double)part[((int64_t)r * 2 + blockIdx.y) * C + c];
    red[warp][lane] = s;
    __syncthreads();
    s = red[lane][warp];  // of channel blockIdx.x * 32 + warp
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0 && blockIdx.x * 32ll + warp < C) out[blockIdx.x * 32ll + warp] = (float)s;
}

template <typename TX, typename TY, int V, int U>
void backward(Handle& h, Backward<TX, TY>& p, float* dw, float* db) {
    const int sms = sm_count(h.device);
    const Cut cut = make_cut(p.a, p.t, (int)(sizeof(TX) + sizeof(TY)), V > 1, sms, CTAS);
    p.ch = cut.ch;
    p.by_warp = cut.by_warp;
    // as many samples a CTA as make four waves of them, but no more than TERMS a thread
    const int64_t items = ceil_div(p.a.samples, cut.by_warp ? WARPS : 1);
    p.each = (int)std::clamp<int64_t>(items * p.t.blocks / (4 * CTAS * sms), 1, TERMS) * (cut.by_warp ? WARPS : 1);
    p.walkers = cut.only_long ? 0 : (int)std::max<int64_t>(1, ceil_div(p.a.samples, p.each));
    DevBuf<float2> part((size_t)p.ch.count * 2 * part_slots(p.t), h.stream);
    DevBuf<int2> found((size_t)p.ch.count, h.stream);
    const int rows = p.walkers + p.ch.count;
    const bool direct = p.walkers == 1 && p.ch.count == 0 && p.t.tpg == 1;  // nothing to add up
    DevBuf<float> weights((dw || db) && !direct ? (size_t)rows * 2 * p.a.C : 0, h.stream);
    if (direct) p.dw = dw, p.db = db;
    p.part = part.get();
    p.found = found.get();
    p.weights = weights.get();
    const int64_t chunked = (int64_t)p.ch.count * p.t.tiles, grid = chunked + (int64_t)p.walkers * p.t.blocks;
    XS_REQUIRE(grid < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "too many samples and groups");
    allow_smem(group_norm_grad_kernel<TX, TY, V, U>, SLOT_BYTES * THREADS);
    launch_dependent(h.stream, group_norm_grad_kernel<TX, TY, V, U>, (unsigned)grid, THREADS, SLOT_BYTES * THREADS, 1, p);
    after_launch(h, "group_norm_grad");
    if (p.ch.count > 0 && p.dx) {
        allow_smem(group_norm_grad_apply_kernel<TX, TY, V, U>, SLOT_BYTES * THREADS);
        launch_dependent(h.stream, group_norm_grad_apply_kernel<TX, TY, V, U>, (unsigned)chunked, THREADS, SLOT_BYTES * THREADS, 1, p);
        after_launch(h, "group_norm_grad_apply");
    }
    if (p.weights) {
        launch_dependent(h.stream, group_norm_weights_kernel, dim3((unsigned)ceil_div(p.a.C, 32), 2), 1024, 0, 1,
                         (const float*)p.weights, rows, p.a.C, dw, db);
        after_launch(h, "group_norm_weights");
    }
}

}  // namespace

template <typename TX, typename TY>
void group_norm_backward(Handle& h, const GroupNormArgs<TX>& a, const TY* dy, int64_t lddy, const float* mean,
                         const float* rstd, TY* dx, int64_t lddx, float* dw, float* db) {
    if (!dx && !dw && !db) return;
    Backward<TX, TY> p = {};
    p.a = a;
    p.dy = dy;
    p.lddy = lddy;
    p.mean = mean;
    p.rstd = rstd;
    p.dx = dx;
    p.lddx = lddx;
    const size_t bx = PER * sizeof(TX), by = PER * sizeof(TY);
    const bool wide = a.C % PER == 0 && (a.rows <= 1 || (a.ldx % PER == 0 && lddy % PER == 0 && (!dx || lddx % PER == 0))) &&
                      aligned_to(a.x, bx) && aligned_to(dy, by) && aligned_to(dx, by);
    if (wide && make_tiling(p.t, a, PER, 1, sm_count(h.device))) return backward<TX, TY, PER, 1>(h, p, dw, db);
    make_tiling(p.t, a, 1, PER, sm_count(h.device));
    backward<TX, TY, 1, PER>(h, p, dw, db);
}

#define XS_INST_GROUP_NORM_GRAD(TX, TY)                                                                          \
    template void group_norm_backward<TX, TY>(Handle&, const GroupNormArgs<TX>&, const TY*, int64_t, const float*, \
                                              const float*, TY*, int64_t, float*, float*);
XS_INST_GROUP_NORM_GRAD(__half, __half)
XS_INST_GROUP_NORM_GRAD(__nv_bfloat16, __nv_bfloat16)
XS_INST_GROUP_NORM_GRAD(float, float)
XS_INST_GROUP_NORM_GRAD(float, __half)
XS_INST_GROUP_NORM_GRAD(float, __nv_bfloat16)

}  // namespace xspmm_b200
