// group_norm_grad.cu -- the gradient of the group norm with an activation.
//
// xh = (x - mean) * rstd, z = xh * w + b, dz = dy * act'(z). Per sample and channel, A = sum of dz and B = sum of
// dz * xh over the rows; dw = sum of B and db = sum of A over the samples. With t = dz * w the means over a group's n
// values are m1 = sum_c w A / n and m2 = sum_c w B / n, and dx = rstd * (t - m1 - xh * m2). So one pass over x and dy
// for A and B serves the weights and the groups, and a second one gives dx.
//
// Who takes which samples is decided as in the forward pass (group_norm.cu). The sums for the weights' gradients stay
// in a thread's registers over all samples that its CTA takes and leave as one row a CTA (or chunk), added in order
// by the last kernel; a group wider than a tile has no registers for them and adds them to its CTA's row as it goes.
#include "group_norm.cuh"

namespace xspmm_b200 {
namespace {

using namespace group;

template <typename TX, typename TY>
struct Backward {
    GroupNormArgs<TX> a;
    Tiling t;
    Chunks ch;
    int each;           // samples of a work item: WARPS or 1
    int walkers;        // CTAs a block that walk the work items, 0 where all samples are long
    int64_t warp_rows;  // most rows that a warp takes
    const TY* dy;
    int64_t lddy;
    const float *mean, *rstd;
    TY* dx;  // or null
    int64_t lddx;
    float* weights;  // [walker, then chunk][2][channel]: sums of dz * xh and dz, or null
    float2* part;    // [slot][chunk][group or tile of it]: sums of w A and w B
    float2* fin;     // [chunk][group]: m1 and m2 of the long sample that begins in the chunk
    int2* found;     // [chunk]: the long samples with rows in it
};

// A thread's view of its channels: the parameters, and a sample's statistics.
template <int E>
struct Channels {
    float w[E], b[E], m[E], rs[E];
};

// dz and xh of a row's values.
template <typename TX, typename TY, int V, int U>
__device__ __forceinline__ void row_terms(const Pack<TX, V> (&rx)[U], const Pack<TY, V> (&rg)[U], const Channels<V * U>& ch,
                                          Activation act, float (&dz)[V * U], float (&xh)[V * U]) {
    constexpr int E = V * U;
    Place<V, U>::values(rx, xh);
    Place<V, U>::values(rg, dz);
#pragma unroll
    for (int e = 0; e < E; ++e) xh[e] = centred(xh[e], ch.m[e], ch.rs[e]);
    with_act(act, [&](auto a) {
        if constexpr (decltype(a)::value != Activation::None)
#pragma unroll
            for (int e = 0; e < E; ++e)
                dz[e] *= slope_one<sizeof(TY) == 4, decltype(a)::value>(affine(xh[e], ch.w[e], ch.b[e]));
    });
}

// Calls f(row, dz, xh) for this thread's rows of [begin, end).
template <bool CTA, int B, typename TX, typename TY, int V, int U, typename F>
__device__ __forceinline__ void each_row(const Team<CTA, V, U>& tm, const TX* x, int64_t ldx, const TY* dy, int64_t lddy,
                                         int64_t begin, int64_t end, const Channels<V * U>& ch, Activation act, F&& f) {
    for (int64_t r = begin + tm.rl; r < end; r += (int64_t)tm.step * B) {
        Pack<TX, V> rx[B][U];
        Pack<TY, V> rg[B][U];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int64_t row = r + (int64_t)i * tm.step;
            if (row < end) {
                tm.at.load(rx[i], x + row * ldx);
                tm.at.load(rg[i], dy + row * lddy);
            }
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int64_t row = r + (int64_t)i * tm.step;
            if (row >= end) break;
            float dz[V * U], xh[V * U];
            row_terms(rx[i], rg[i], ch, act, dz, xh);
            f(row, dz, xh);
        }
    }
}

template <int E>
struct Sums {
    float a[E] = {}, b[E] = {};
};

// This thread's A and B over rows [begin, end), added to `total`, and the groups' sums of w A and w B, which one thread
// a group hands to f(group of the tile, sum, sum). channels(strips) is called between, once the tile's A and B are
// there by channel. The strips may be written again after a team_sync.
template <bool CTA, int B, typename TX, typename TY, int V, int U, typename F, typename C>
__device__ __forceinline__ void group_sums(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm, const Tile& k, int64_t begin,
                                           int64_t end, const Channels<V * U>& ch, Sums<V * U>& total, Strips& sh, F&& f,
                                           C&& channels) {
    constexpr int E = V * U;
    Sums<E> s;
    each_row<CTA, B>(tm, p.a.x + k.c0, p.a.ldx, p.dy + k.c0, p.lddy, begin, end, ch, p.a.act,
                     [&](int64_t, const float (&dz)[E], const float (&xh)[E]) {
#pragma unroll
                         for (int e = 0; e < E; ++e) {
                             s.a[e] += dz[e];
                             s.b[e] = fmaf(dz[e], xh[e], s.b[e]);
                         }
                     });
#pragma unroll
    for (int e = 0; e < E; ++e) total.a[e] += s.a[e], total.b[e] += s.b[e];
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

// dx of rows [begin, end) from the groups' m1 and m2.
template <bool CTA, int B, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void apply(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm, const Tile& k, int64_t begin,
                                      int64_t end, const Channels<V * U>& ch, const float* g1, const float* g2) {
    constexpr int E = V * U;
    float m1[E], m2[E];
    tm.of_groups(m1, g1, k);
    tm.of_groups(m2, g2, k);
    each_row<CTA, B>(tm, p.a.x + k.c0, p.a.ldx, p.dy + k.c0, p.lddy, begin, end, ch, p.a.act,
                     [&](int64_t row, const float (&dz)[E], const float (&xh)[E]) {
                         float v[E];
#pragma unroll
                         for (int e = 0; e < E; ++e)
                             v[e] = ch.rs[e] * (fmaf(-xh[e], m2[e], fmaf(dz[e], ch.w[e], -m1[e])));
                         tm.at.store(p.dx + k.c0 + row * p.lddx, v);
                     });
}

template <bool CTA, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void parameters(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm, const Tile& k,
                                           Channels<V * U>& ch) {
    tm.at.param(ch.w, p.a.w, k.c0, 1.0f);
    tm.at.param(ch.b, p.a.b, k.c0, 0.0f);
}
template <bool CTA, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void statistics(const Backward<TX, TY>& p, const Team<CTA, V, U>& tm, const Tile& k, int64_t s,
                                           Channels<V * U>& ch) {
    tm.of_groups(ch.m, p.mean + s * p.t.groups + k.g0, k);
    tm.of_groups(ch.rs, p.rstd + s * p.t.groups + k.g0, k);
}

// The CTA's sums of a tile's channels to row `row` of the weights' parts.
template <typename TX, typename TY, int V, int U>
__device__ __forceinline__ void leave_weights(const Backward<TX, TY>& p, int64_t row, const Tile& k, const Place<V, U>& at,
                                              Sums<V * U>& total, Strips& sh) {
    sum_channels<true>(total.a, total.b, at, sh);
    if ((int)threadIdx.x < k.cols) {
        float* out = p.weights + row * 2 * p.a.C + k.c0 + threadIdx.x;
        out[0] = sh.v[0][1][threadIdx.x];
        out[p.a.C] = sh.v[0][0][threadIdx.x];
    }
}

// A sample by a team. `total` is the CTA's sums where a block is one tile; else they go to the CTA's row.
template <bool CTA, int B, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void whole_sample(const Backward<TX, TY>& p, int64_t s, Span rows, int block, int64_t row,
                                             Channels<V * U>& ch, Sums<V * U>& total, Strips& sh, float* g1, float* g2) {
    const int t0 = block * p.t.tpg;
    const bool one = p.t.tpg == 1;
    for (int j = 0; j < p.t.tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        if (!one) parameters(p, tm, k, ch);
        if (one || j == 0) statistics(p, tm, k, s, ch);
        const float per = 1.0f / ((float)(rows.end - rows.begin) * (float)p.t.width);
        group_sums<CTA, B>(p, tm, k, rows.begin, rows.end, ch, total, sh,
                           [&](int g, float s1, float s2) {
                               if (j > 0) s1 += g1[g], s2 += g2[g];  // the same thread's sums of the tiles before
                               const bool last = j + 1 == p.t.tpg;
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
    for (int j = 0; j < p.t.tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        if (!one) parameters(p, tm, k, ch);
        apply<CTA, B>(p, tm, k, rows.begin, rows.end, ch, g1, g2);
    }
    team_sync<CTA>();
}

// CTAs [0, chunks x tiles): sums of the long samples' chunks. The others: short and middle samples.
template <typename TX, typename TY, int V, int U, int B>
__global__ void __launch_bounds__(THREADS, 2) group_norm_grad_kernel(const __grid_constant__ Backward<TX, TY> p) {
    __shared__ Strips sh;
    __shared__ float g1[WARPS][MAX_TILE], g2[WARPS][MAX_TILE];
    cudaGridDependencySynchronize();
    const int chunked = p.ch.count * p.t.tiles, warp = threadIdx.x >> 5;
    Channels<V * U> ch;
    Sums<V * U> total;
    if ((int)blockIdx.x < chunked) {
        const int i = blockIdx.x / p.t.tiles, tile = blockIdx.x - i * p.t.tiles;
        const int2 found = long_samples(p.a.offsets, (int)p.a.samples, p.a.rows, p.ch, i);
        if (tile == 0 && threadIdx.x == 0) p.found[i] = found;
        const Tile k = tile_of(p.t, tile);
        const Team<true, V, U> tm(p.t, k.cols);
        const int64_t r0 = i * p.ch.rows, r1 = min(p.a.rows, r0 + p.ch.rows), slots = p.t.tpg == 1 ? p.t.groups : p.t.tiles;
        parameters(p, tm, k, ch);
        for (int slot = 0; slot < 2; ++slot) {
            const int s = slot ? found.y : found.x;
            if (s < 0) continue;
            const Span sp = span_of(p.a.offsets, s, p.a.rows);
            float2* out = p.part + ((int64_t)slot * p.ch.count + i) * slots + part_slot(p.t, tile, k);
            statistics(p, tm, k, s, ch);
            group_sums<true, B>(p, tm, k, max(r0, sp.begin), min(r1, sp.end), ch, total, sh,
                                [&](int g, float s1, float s2) { out[g] = make_float2(s1, s2); },
                                [](const float (&)[2][MAX_TILE]) {});
            __syncthreads();
        }
        if (p.weights) leave_weights(p, p.walkers + i, k, tm.at, total, sh);
        return;
    }
    const int at = blockIdx.x - chunked, block = at % p.t.blocks, walker = at / p.t.blocks;
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
    auto rows_of = [&](int64_t s) { return span_of(p.a.offsets, s, p.a.rows); };
    for (int64_t s0 = (int64_t)walker * p.each; s0 < p.a.samples; s0 += (int64_t)p.walkers * p.each) {
        if (p.each > 1) {
            const int64_t s = s0 + warp;
            if (s < p.a.samples) {
                const Span sp = rows_of(s);
                if (sp.end > sp.begin && sp.end - sp.begin <= p.warp_rows)
                    whole_sample<false, B, TX, TY, V, U>(p, s, sp, block, walker, ch, total, sh, g1[warp], g2[warp]);
            }
            __syncthreads();
        }
        for (int j = 0; j < p.each && s0 + j < p.a.samples; ++j) {
            const Span sp = rows_of(s0 + j);
            const int64_t n = sp.end - sp.begin;
            if (n > 0 && n <= p.ch.longest && (p.each == 1 || n > p.warp_rows))
                whole_sample<true, B, TX, TY, V, U>(p, s0 + j, sp, block, walker, ch, total, sh, g1[0], g2[0]);
        }
    }
    if (one && p.weights) leave_weights(p, walker, k, tm.at, total, sh);
}

// m1 and m2 of the long samples: a warp for each chunk and group. A sample belongs to the chunk it begins in.
template <typename TX, typename TY>
__global__ void __launch_bounds__(THREADS) group_norm_grad_join_kernel(const __grid_constant__ Backward<TX, TY> p) {
    cudaGridDependencySynchronize();
    const int i = blockIdx.x, s = p.found[i].y, g = blockIdx.y * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (s < 0 || g >= p.t.groups) return;
    const Span sp = span_of(p.a.offsets, s, p.a.rows);
    const int last = (int)((sp.end - 1) / p.ch.rows), tpg = p.t.tpg, parts = (last - i + 1) * tpg;
    const int64_t slots = tpg == 1 ? p.t.groups : p.t.tiles;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 4
    for (int q = lane; q < parts; q += 32) {
        const int c = i + q / tpg;
        const float2 v = p.part[((int64_t)(c == i) * p.ch.count + c) * slots + g * tpg + q % tpg];
        s1 += v.x;
        s2 += v.y;
    }
    s1 = group_sum(s1, 32);
    s2 = group_sum(s2, 32);
    const float per = 1.0f / ((float)(sp.end - sp.begin) * (float)p.t.width);
    if (lane == 0) p.fin[(int64_t)i * p.t.groups + g] = make_float2(s1 * per, s2 * per);
}

template <typename TX, typename TY, int V, int U, int B>
__global__ void __launch_bounds__(THREADS, 2) group_norm_grad_apply_kernel(const __grid_constant__ Backward<TX, TY> p) {
    __shared__ float g1[MAX_TILE], g2[MAX_TILE];
    cudaGridDependencySynchronize();
    const int i = p.ch.count - 1 - blockIdx.x / p.t.tiles, tile = blockIdx.x % p.t.tiles;
    const int2 found = p.found[i];
    if (found.x < 0 && found.y < 0) return;
    const Tile k = tile_of(p.t, tile);
    const Team<true, V, U> tm(p.t, k.cols);
    const int64_t r0 = i * p.ch.rows, r1 = min(p.a.rows, r0 + p.ch.rows);
    Channels<V * U> ch;
    parameters(p, tm, k, ch);
    for (int slot = 0; slot < 2; ++slot) {
        const int s = slot ? found.y : found.x;
        if (s < 0) continue;
        const Span sp = span_of(p.a.offsets, s, p.a.rows);
        __syncthreads();
        if ((int)threadIdx.x < k.ng) {
            const float2 v = p.fin[sp.begin / p.ch.rows * p.t.groups + k.g0 + threadIdx.x];
            g1[threadIdx.x] = v.x;
            g2[threadIdx.x] = v.y;
        }
        __syncthreads();
        statistics(p, tm, k, s, ch);
        apply<true, B>(p, tm, k, max(r0, sp.begin), min(r1, sp.end), ch, g1, g2);
    }
}

// dw and db: the rows of parts added in order, 32 channels a CTA; its warps take every 32nd row.
__global__ void __launch_bounds__(1024) group_norm_weights_kernel(const float* part, int rows, int64_t C, float* dw, float* db) {
    __shared__ float red[32][33];
    cudaGridDependencySynchronize();
    float* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = blockIdx.x * 32ll + lane;
    float s = 0.0f;
    if (c < C)
#pragma unroll 8
        for (int r = warp; r < rows; r += 32) s += part[((int64_t)r * 2 + blockIdx.y) * C + c];
    red[warp][lane] = s;
    __syncthreads();
    s = group_sum(red[lane][warp], 32);  // of channel blockIdx.x * 32 + warp
    if (lane == 0 && blockIdx.x * 32ll + warp < C) out[blockIdx.x * 32ll + warp] = s;
}

template <typename TX, typename TY, int V, int U, int B>
void backward(Handle& h, Backward<TX, TY>& p, float* dw, float* db) {
    const int sms = sm_count(h.device);
    const Cut cut = make_cut(p.a, p.t, (int)(sizeof(TX) + sizeof(TY)), sms);
    p.ch = cut.ch;
    p.each = cut.each;
    p.warp_rows = cut.warp_rows;
    const int64_t items = ceil_div(p.a.samples, p.each);
    p.walkers = cut.only_long ? 0 : (int)std::max<int64_t>(1, std::min(items, ceil_div(2 * sms, p.t.blocks)));
    DevBuf<float2> ws((size_t)p.ch.count * (2 * part_slots(p.t) + p.t.groups), h.stream);
    DevBuf<int2> found((size_t)p.ch.count, h.stream);
    const int parts = p.walkers + p.ch.count;
    DevBuf<float> weights(dw || db ? (size_t)parts * 2 * p.a.C : 0, h.stream);
    p.part = ws.get();
    p.fin = ws.get() + (int64_t)p.ch.count * 2 * part_slots(p.t);
    p.found = found.get();
    p.weights = weights.get();
    const int64_t chunked = (int64_t)p.ch.count * p.t.tiles, grid = chunked + (int64_t)p.walkers * p.t.blocks;
    XS_REQUIRE(grid < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "too many samples and groups");
    launch_dependent(h.stream, group_norm_grad_kernel<TX, TY, V, U, B>, (unsigned)grid, THREADS, 0, 1, p);
    after_launch(h, "group_norm_grad");
    if (p.ch.count > 0 && p.dx) {
        launch_dependent(h.stream, group_norm_grad_join_kernel<TX, TY>,
                         dim3((unsigned)p.ch.count, (unsigned)ceil_div(p.t.groups, WARPS)), THREADS, 0, 1, p);
        after_launch(h, "group_norm_grad_join");
        launch_dependent(h.stream, group_norm_grad_apply_kernel<TX, TY, V, U, B>, (unsigned)chunked, THREADS, 0, 1, p);
        after_launch(h, "group_norm_grad_apply");
    }
    if (p.weights) {
        launch_dependent(h.stream, group_norm_weights_kernel, dim3((unsigned)ceil_div(p.a.C, 32), 2), 1024, 0, 1,
                         (const float*)p.weights, parts, p.a.C, dw, db);
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
    constexpr int V = 16 / sizeof(TX);
    constexpr size_t other = std::min<size_t>(16, V * sizeof(TY));
    const bool wide = a.C % V == 0 && (a.rows <= 1 || (a.ldx % V == 0 && lddy % V == 0 && (!dx || lddx % V == 0))) &&
                      aligned_to(a.x, 16) && aligned_to(dy, other) && aligned_to(dx, other);
    if (wide && make_tiling(p.t, a.C, a.groups, V, 1, 32 * V)) return backward<TX, TY, V, 1, 4>(h, p, dw, db);
    if (a.C <= 32) {
        make_tiling(p.t, a.C, a.groups, 1, 1, 32);
        backward<TX, TY, 1, 1, 8>(h, p, dw, db);
    } else {
        make_tiling(p.t, a.C, a.groups, 1, 8, MAX_TILE);
        backward<TX, TY, 1, 8, 2>(h, p, dw, db);
    }
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
