// group_norm.cu -- group norm with an activation over the samples of a packed batch.
//
// Over the n values of a sample's rows and a group's channels, mean = sum(x) / n, var = sum((x - mean)^2) / n,
// rstd = 1 / sqrt(var + eps); z = ((x - mean) * rstd) * w + b, y = act(z).
//
// The pass is bound by memory: x has to be read and y written once, and where a sample does not fit on chip x is read
// a second time, from L2 as far as it is still there. The host does not know the samples' lengths, so each launch
// decides on the device who takes what:
//   * short samples (a few tens of KB of a column tile) by a warp each, eight to a CTA; where there are too few to
//     fill the GPU with warps, by a CTA each;
//   * samples of up to Chunks::longest rows by a CTA, which reads them twice;
//   * longer ones in chunks of rows by all CTAs: moments of each chunk, a second kernel that joins them, a third that
//     applies them, from the last chunk to the first, since the last ones read are still in L2. These two are not
//     launched where no sample can be long.
// Moments are joined from those of batches of rows that a thread holds in registers, each taken about its own mean, so
// neither a large mean nor rows far from the others cost accuracy; all orders are fixed by the sizes and offsets.
#include "group_norm.cuh"

namespace xspmm_b200 {
namespace {

using namespace group;

template <typename TX, typename TY>
struct Forward {
    GroupNormArgs<TX> a;
    Tiling t;
    Chunks ch;
    int each;         // samples that a CTA of short samples takes: WARPS or 1
    int64_t warp_rows;  // most rows that a warp takes
    float eps;
    TY* y;
    int64_t ldy;
    float *mean, *rstd;  // or null
    float2* part;        // [slot][chunk][group or tile of it]: mean and sum of squares about it
    float2* fin;         // [chunk][group]: mean and rstd of the long sample that begins in the chunk
    int2* found;         // [chunk]: the long samples with rows in it
};

template <int E>
struct Moments {
    float n = 0.0f, mean[E] = {}, m2[E] = {};
};

// Adds the first `count` rows of a batch.
template <int B, typename TX, int V, int U>
__device__ __forceinline__ void add_rows(Moments<V * U>& m, const Pack<TX, V> (&raw)[B][U], int count) {
    constexpr int E = V * U;
    float s[E], q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = q[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < B; ++i) {  // rows past the last are zeros
        float v[E];
        Place<V, U>::values(raw[i], v);
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += v[e];
    }
    const float n = (float)count, per = count == B ? 1.0f / B : 1.0f / n;
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] *= per;
#pragma unroll
    for (int i = 0; i < B; ++i) {
        if (i >= count) break;
        float v[E];
        Place<V, U>::values(raw[i], v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = v[e] - s[e];
            q[e] = fmaf(d, d, q[e]);
        }
    }
    const float total = m.n + n, fb = n / total, f = m.n * fb;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float d = s[e] - m.mean[e];
        m.mean[e] = fmaf(d, fb, m.mean[e]);
        m.m2[e] += fmaf(d * d, f, q[e]);
    }
    m.n = total;
}

// Moments of the tile's groups over rows [begin, end) of x (its first channel): f(group of the tile, mean, sum of
// squares), called by one thread a group. The strips may be written again after a team_sync.
template <bool CTA, int B, typename TX, int V, int U, typename F>
__device__ __forceinline__ void group_moments(const Team<CTA, V, U>& tm, const TX* x, int64_t ldx, int64_t begin,
                                              int64_t end, const Tile& k, Strips& sh, F&& f) {
    constexpr int E = V * U;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Moments<E> m;
    for (int64_t r = begin + tm.rl; r < end; r += (int64_t)tm.step * B) {
        Pack<TX, V> raw[B][U];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int64_t row = r + (int64_t)i * tm.step;
            if (row < end) tm.at.load(raw[i], x + row * ldx);
            else
#pragma unroll
                for (int u = 0; u < U; ++u) raw[i][u] = Pack<TX, V>{};
        }
        add_rows(m, raw, (int)min((int64_t)B, (end - r + tm.step - 1) / tm.step));
    }
    auto weights = [](float na, float nb, float* fb, float* f) {
        const float n = na + nb;
        *fb = n > 0.0f ? nb / n : 0.0f;
        *f = na * *fb;
        return n;
    };
    for (int o = 16; o >= tm.at.lpr; o >>= 1) {
        // both of a pair take the lower lane's moments first, so that they end with the same numbers
        const bool low = (lane & o) == 0;
        const float other = __shfl_xor_sync(0xffffffffu, m.n, o);
        float fb, g;
        const float n = weights(low ? m.n : other, low ? other : m.n, &fb, &g);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float mo = __shfl_xor_sync(0xffffffffu, m.mean[e], o), so = __shfl_xor_sync(0xffffffffu, m.m2[e], o);
            float ma = low ? m.mean[e] : mo, sa = low ? m.m2[e] : so;
            join_moments(ma, sa, low ? mo : m.mean[e], low ? so : m.m2[e], fb, g);
            m.mean[e] = ma;
            m.m2[e] = sa;
        }
        m.n = n;
    }
    team_sync<CTA>();
    if (lane < tm.at.lpr)
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (tm.at.in(u))
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sh.v[warp][0][tm.at.col(u) + e] = m.mean[u * V + e];
                    sh.v[warp][1][tm.at.col(u) + e] = m.m2[u * V + e];
                }
    if (lane == 0) sh.n[warp] = m.n;
    team_sync<CTA>();
    if constexpr (CTA) {
        const int c = threadIdx.x;
        if (c < k.cols) {
            float n = sh.n[0], ma = sh.v[0][0][c], sa = sh.v[0][1][c];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) {
                float fb, g;
                n = weights(n, sh.n[w], &fb, &g);
                join_moments(ma, sa, sh.v[w][0][c], sh.v[w][1][c], fb, g);
            }
            sh.v[0][0][c] = ma;
            sh.v[0][1][c] = sa;
        }
        __syncthreads();
    }
    // every channel has the same number of values
    const float* cm = sh.v[CTA ? 0 : warp][0];
    const float* cs = sh.v[CTA ? 0 : warp][1];
    const float n = (float)(end - begin);
    each_group<CTA>(k.ng, [&](int g, int j, int l, bool live) {
        float s = 0.0f;
        if (live)
            for (int c = j; c < k.lw; c += l) s += cm[g * k.lw + c];
        const float mean = group_sum(s, l) / (float)k.lw;
        s = 0.0f;
        if (live)
            for (int c = j; c < k.lw; c += l) {
                const float d = cm[g * k.lw + c] - mean;
                s += fmaf(n * d, d, cs[g * k.lw + c]);
            }
        s = group_sum(s, l);
        if (live && j == 0) f(g, mean, s);
    });
}

// y of rows [begin, end) from the groups' mean and rstd at st[group of the tile].
template <bool CTA, int B, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void apply(const Team<CTA, V, U>& tm, const TX* x, int64_t ldx, TY* y, int64_t ldy,
                                      int64_t begin, int64_t end, const Tile& k, const float* gm, const float* gr,
                                      const float (&w)[V * U], const float (&b)[V * U], Activation act) {
    constexpr int E = V * U;
    float m[E], rs[E];
    tm.of_groups(m, gm, k);
    tm.of_groups(rs, gr, k);
    for (int64_t r = begin + tm.rl; r < end; r += (int64_t)tm.step * B) {
        Pack<TX, V> raw[B][U];
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (r + (int64_t)i * tm.step < end) tm.at.load(raw[i], x + (r + (int64_t)i * tm.step) * ldx);
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int64_t row = r + (int64_t)i * tm.step;
            if (row >= end) break;
            float v[E];
            Place<V, U>::values(raw[i], v);
            with_act(act, [&](auto a) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    v[e] = act_one<sizeof(TY) == 4, decltype(a)::value>(affine(centred(v[e], m[e], rs[e]), w[e], b[e]));
            });
            tm.at.store(y + row * ldy, v);
        }
    }
}

// A sample by a team: all tiles of the block twice.
template <bool CTA, int B, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void whole_sample(const Forward<TX, TY>& p, int s, Span rows, int block, Strips& sh,
                                             float* gm, float* gr) {
    const int t0 = block * p.t.tpg;
    const float n = (float)(rows.end - rows.begin);
    for (int j = 0; j < p.t.tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        group_moments<CTA, B>(tm, p.a.x + k.c0, p.a.ldx, rows.begin, rows.end, k, sh, [&](int g, float mean, float m2) {
            if (j > 0) {  // the same thread's sums of the tiles before
                const float na = n * (float)(j * p.t.max_cols), nb = n * (float)k.lw, fb = nb / (na + nb);
                float ma = gm[g], sa = gr[g];
                join_moments(ma, sa, mean, m2, fb, na * fb);
                mean = ma;
                m2 = sa;
            }
            if (j + 1 == p.t.tpg) {
                const float count = n * (float)p.t.width;
                m2 = 1.0f / sqrtf(m2 / count + p.eps);
                const int64_t at = (int64_t)s * p.t.groups + k.g0 + g;
                if (p.mean) p.mean[at] = mean;
                if (p.rstd) p.rstd[at] = m2;
            }
            gm[g] = mean;
            gr[g] = m2;
        });
        team_sync<CTA>();
    }
    for (int j = 0; j < p.t.tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        float w[V * U], b[V * U];
        tm.at.param(w, p.a.w, k.c0, 1.0f);
        tm.at.param(b, p.a.b, k.c0, 0.0f);
        apply<CTA, B>(tm, p.a.x + k.c0, p.a.ldx, p.y + k.c0, p.ldy, rows.begin, rows.end, k, gm, gr, w, b, p.a.act);
    }
    team_sync<CTA>();
}

// CTAs [0, chunks x tiles): moments of the long samples' chunks. The others: short and middle samples.
template <typename TX, typename TY, int V, int U, int B>
__global__ void __launch_bounds__(THREADS) group_norm_kernel(const __grid_constant__ Forward<TX, TY> p) {
    __shared__ Strips sh;
    __shared__ float gm[WARPS][MAX_TILE], gr[WARPS][MAX_TILE];
    cudaGridDependencySynchronize();
    const int chunked = p.ch.count * p.t.tiles;
    if ((int)blockIdx.x < chunked) {
        const int i = blockIdx.x / p.t.tiles, tile = blockIdx.x - i * p.t.tiles;
        const int2 found = long_samples(p.a.offsets, (int)p.a.samples, p.a.rows, p.ch, i);
        if (tile == 0 && threadIdx.x == 0) p.found[i] = found;
        const Tile k = tile_of(p.t, tile);
        const Team<true, V, U> tm(p.t, k.cols);
        const int64_t r0 = i * p.ch.rows, r1 = min(p.a.rows, r0 + p.ch.rows), slots = p.t.tpg == 1 ? p.t.groups : p.t.tiles;
        for (int slot = 0; slot < 2; ++slot) {
            const int s = slot ? found.y : found.x;
            if (s < 0) continue;
            const Span sp = span_of(p.a.offsets, s, p.a.rows);
            float2* out = p.part + ((int64_t)slot * p.ch.count + i) * slots + part_slot(p.t, tile, k);
            group_moments<true, B>(tm, p.a.x + k.c0, p.a.ldx, max(r0, sp.begin), min(r1, sp.end), k, sh,
                                   [&](int g, float mean, float m2) { out[g] = make_float2(mean, m2); });
            __syncthreads();
        }
        return;
    }
    const int warp = threadIdx.x >> 5;
    const int64_t at = blockIdx.x - chunked;
    const int block = (int)(at % p.t.blocks);
    const int64_t s0 = at / p.t.blocks * p.each;
    auto rows_of = [&](int64_t s) { return span_of(p.a.offsets, s, p.a.rows); };
    // a sample without rows has statistics all the same
    auto empty = [&](int64_t s) {
        const Tile first = tile_of(p.t, block * p.t.tpg);
        const float rs = 1.0f / sqrtf(p.eps);
        for (int g = threadIdx.x & 31; g < first.ng; g += 32) {
            const int64_t o = s * p.t.groups + first.g0 + g;
            if (p.mean) p.mean[o] = 0.0f;
            if (p.rstd) p.rstd[o] = rs;
        }
    };
    if (p.each > 1) {
        const int64_t s = s0 + warp;
        if (s < p.a.samples) {
            const Span sp = rows_of(s);
            const int64_t n = sp.end - sp.begin;
            if (n == 0) empty(s);
            else if (n <= p.warp_rows) whole_sample<false, B, TX, TY, V, U>(p, (int)s, sp, block, sh, gm[warp], gr[warp]);
        }
        __syncthreads();
    }
    for (int j = 0; j < p.each; ++j) {
        const int64_t s = s0 + j;
        if (s >= p.a.samples) break;
        const Span sp = rows_of(s);
        const int64_t n = sp.end - sp.begin;
        if (n == 0 && p.each == 1 && warp == 0) empty(s);
        if (n > 0 && n <= p.ch.longest && (p.each == 1 || n > p.warp_rows))
            whole_sample<true, B, TX, TY, V, U>(p, (int)s, sp, block, sh, gm[0], gr[0]);
    }
}

// Mean and rstd of the long samples: a warp for each chunk and group, whose lanes take every 32nd of the parts. A sample
// belongs to the chunk it begins in.
template <typename TX, typename TY>
__global__ void __launch_bounds__(THREADS) group_norm_join_kernel(const __grid_constant__ Forward<TX, TY> p) {
    cudaGridDependencySynchronize();
    const int i = blockIdx.x, s = p.found[i].y, g = blockIdx.y * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (s < 0 || g >= p.t.groups) return;
    const Span sp = span_of(p.a.offsets, s, p.a.rows);
    const int last = (int)((sp.end - 1) / p.ch.rows), tpg = p.t.tpg, parts = (last - i + 1) * tpg;
    const int64_t slots = tpg == 1 ? p.t.groups : p.t.tiles;
    float n = 0.0f, mean = 0.0f, m2 = 0.0f;
    auto join = [&](float nb, float mb, float sb) {
        const float total = n + nb, fb = total > 0.0f ? nb / total : 0.0f;
        join_moments(mean, m2, mb, sb, fb, n * fb);
        n = total;
    };
#pragma unroll 4
    for (int q = lane; q < parts; q += 32) {
        const int c = i + q / tpg, part = q % tpg;
        const int64_t rows = min(sp.end, (c + 1) * p.ch.rows) - max(sp.begin, c * p.ch.rows);
        const int lw = tpg == 1 ? p.t.width : min(p.t.max_cols, p.t.width - part * p.t.max_cols);
        const float2 v = p.part[((int64_t)(c == i) * p.ch.count + c) * slots + g * tpg + part];
        join((float)rows * (float)lw, v.x, v.y);
    }
    for (int o = 16; o > 0; o >>= 1) {
        const bool low = (lane & o) == 0;
        float nb = __shfl_xor_sync(0xffffffffu, n, o), mb = __shfl_xor_sync(0xffffffffu, mean, o);
        float sb = __shfl_xor_sync(0xffffffffu, m2, o);
        if (!low) {
            float x;
            x = n, n = nb, nb = x;
            x = mean, mean = mb, mb = x;
            x = m2, m2 = sb, sb = x;
        }
        join(nb, mb, sb);
    }
    if (lane == 0) {
        const float rs = 1.0f / sqrtf(m2 / n + p.eps);
        p.fin[(int64_t)i * p.t.groups + g] = make_float2(mean, rs);
        if (p.mean) p.mean[(int64_t)s * p.t.groups + g] = mean;
        if (p.rstd) p.rstd[(int64_t)s * p.t.groups + g] = rs;
    }
}

template <typename TX, typename TY, int V, int U, int B>
__global__ void __launch_bounds__(THREADS) group_norm_apply_kernel(const __grid_constant__ Forward<TX, TY> p) {
    __shared__ float gm[MAX_TILE], gr[MAX_TILE];
    cudaGridDependencySynchronize();
    const int i = p.ch.count - 1 - blockIdx.x / p.t.tiles, tile = blockIdx.x % p.t.tiles;
    const int2 found = p.found[i];
    if (found.x < 0 && found.y < 0) return;
    const Tile k = tile_of(p.t, tile);
    const Team<true, V, U> tm(p.t, k.cols);
    const int64_t r0 = i * p.ch.rows, r1 = min(p.a.rows, r0 + p.ch.rows);
    float w[V * U], b[V * U];
    tm.at.param(w, p.a.w, k.c0, 1.0f);
    tm.at.param(b, p.a.b, k.c0, 0.0f);
    for (int slot = 0; slot < 2; ++slot) {
        const int s = slot ? found.y : found.x;
        if (s < 0) continue;
        const Span sp = span_of(p.a.offsets, s, p.a.rows);
        __syncthreads();
        if ((int)threadIdx.x < k.ng) {
            const float2 v = p.fin[sp.begin / p.ch.rows * p.t.groups + k.g0 + threadIdx.x];
            gm[threadIdx.x] = v.x;
            gr[threadIdx.x] = v.y;
        }
        __syncthreads();
        apply<true, B>(tm, p.a.x + k.c0, p.a.ldx, p.y + k.c0, p.ldy, max(r0, sp.begin), min(r1, sp.end), k, gm, gr, w, b, p.a.act);
    }
}

template <typename TX, typename TY, int V, int U, int B>
void forward(Handle& h, Forward<TX, TY>& p) {
    const int sms = sm_count(h.device);
    const Cut cut = make_cut(p.a, p.t, (int)sizeof(TX), sms);
    p.ch = cut.ch;
    p.each = cut.each;
    p.warp_rows = cut.warp_rows;
    DevBuf<float2> ws((size_t)p.ch.count * (2 * part_slots(p.t) + p.t.groups), h.stream);
    DevBuf<int2> found((size_t)p.ch.count, h.stream);
    p.part = ws.get();
    p.fin = ws.get() + (int64_t)p.ch.count * 2 * part_slots(p.t);
    p.found = found.get();
    const int64_t chunked = (int64_t)p.ch.count * p.t.tiles;
    const int64_t grid = chunked + (cut.only_long ? 0 : ceil_div(p.a.samples, p.each) * p.t.blocks);
    XS_REQUIRE(grid < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "too many samples and groups");
    launch_dependent(h.stream, group_norm_kernel<TX, TY, V, U, B>, (unsigned)grid, THREADS, 0, 1, p);
    after_launch(h, "group_norm");
    if (p.ch.count == 0) return;
    launch_dependent(h.stream, group_norm_join_kernel<TX, TY>, dim3((unsigned)p.ch.count, (unsigned)ceil_div(p.t.groups, WARPS)),
                     THREADS, 0, 1, p);
    after_launch(h, "group_norm_join");
    launch_dependent(h.stream, group_norm_apply_kernel<TX, TY, V, U, B>, (unsigned)chunked, THREADS, 0, 1, p);
    after_launch(h, "group_norm_apply");
}

}  // namespace

template <typename TX, typename TY>
void group_norm(Handle& h, const GroupNormArgs<TX>& a, float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    if (a.samples == 0) return;
    Forward<TX, TY> p = {};
    p.a = a;
    p.eps = eps;
    p.y = y;
    p.ldy = ldy;
    p.mean = mean;
    p.rstd = rstd;
    constexpr int V = 16 / sizeof(TX);
    const bool wide = a.C % V == 0 && (a.rows <= 1 || (a.ldx % V == 0 && ldy % V == 0)) && aligned_to(a.x, 16) &&
                      aligned_to(y, std::min<size_t>(16, V * sizeof(TY)));
    if (wide && make_tiling(p.t, a.C, a.groups, V, 1, 32 * V)) return forward<TX, TY, V, 1, 8>(h, p);
    if (a.C <= 32) {
        make_tiling(p.t, a.C, a.groups, 1, 1, 32);
        forward<TX, TY, 1, 1, 8>(h, p);
    } else {
        make_tiling(p.t, a.C, a.groups, 1, 8, MAX_TILE);
        forward<TX, TY, 1, 8, 2>(h, p);
    }
}

#define XS_INST_GROUP_NORM(TX, TY) \
    template void group_norm<TX, TY>(Handle&, const GroupNormArgs<TX>&, float, TY*, int64_t, float*, float*);
XS_INST_GROUP_NORM(__half, __half)
XS_INST_GROUP_NORM(__nv_bfloat16, __nv_bfloat16)
XS_INST_GROUP_NORM(float, float)
XS_INST_GROUP_NORM(float, __half)
XS_INST_GROUP_NORM(float, __nv_bfloat16)

}  // namespace xspmm_b200
