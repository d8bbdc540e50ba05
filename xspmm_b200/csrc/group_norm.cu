// group_norm.cu -- group norm with an activation over the samples of a packed batch.
//
// Over the n values of a sample's rows and a group's channels, mean = sum(x) / n, var = sum((x - mean)^2) / n,
// rstd = 1 / sqrt(var + eps); z = ((x - mean) * rstd) * w + b, y = act(z).
//
// x has to be read and y written once; where a sample does not fit on chip x is read a second time, from L2 as far as it
// is still there. The host does not know the samples' lengths, so each launch decides on the device who takes what:
//   * samples by a CTA each, or where they have a row or two for each of its threads by a warp each: up to what the
//     threads' slots in shared memory hold they are read once, else twice;
//   * samples of more than Chunks::longest rows in chunks of rows by all CTAs: moments of each chunk, and a second kernel
//     that joins them and writes y, from the last chunk and row to the first, since the last ones read are still in L2. It
//     is not launched where no sample can be long.
// Long samples are bound by DRAM in the first pass (2^20 x 128 fp32: 88 us, 6.1 TB/s) and by the activation's instructions
// and their latency in the second (silu, to fp16: 165 us for 786 MB; issue in 43 % of the cycles). Short ones are bound by
// instructions (4096 samples of 2^18 x 256 bf16, gelu: 117 us, 41 at the copy bandwidth; 33 warp instructions for each value
// of a lane, issue in 63 % of the cycles). More CTAs of fewer registers an SM, or fewer of more slots, were not faster.
// Moments are joined from those of batches of rows that a thread holds in registers, each taken about its own mean, so
// neither a large mean nor rows far from the others cost accuracy; means are joined about one of them, so equal values have
// that mean exactly, of any size. All orders are fixed by the sizes and offsets.
#include "group_norm.cuh"

namespace xspmm_b200 {
namespace {

using namespace group;

constexpr int CTAS = 6;  // that an SM should hold: 80 registers a thread and
constexpr int SLOT_BYTES = 224;  // of shared memory a thread for rows
constexpr int RING_BYTES = 192;  // of them for rows that only pass

template <typename TX, typename TY>
struct Forward {
    GroupNormArgs<TX> a;
    Tiling t;
    Chunks ch;
    int each;  // samples that a CTA takes: WARPS, one a warp where it can, or 1
    float eps;
    TY* y;
    int64_t ldy;
    float *mean, *rstd;  // or null
    float2* part;        // Parts: mean and sum of squares about it
    int2* found;         // [chunk]: the long samples with rows in it
};

template <int P>  // pairs of channels
struct Moments {
    float n = 0.0f;
    float2 mean[P] = {}, m2[P] = {};
};

// Adds B rows. Their mean is the sum of parts of them, and a weight is multiplied to one deviation before the other: no sum
// of values leaves fp32's range, and where no rows were before (weight 0) no infinite square becomes NaN.
template <int B, typename TX, int V, int U>
__device__ __forceinline__ void add_rows(Moments<V * U / 2>& m, const Pack<TX, V> (&raw)[B][U]) {
    constexpr int P = V * U / 2;
    float2 s[P] = {}, q[P] = {}, v[P];  // s: minus the mean
#pragma unroll
    for (int i = 0; i < B; ++i) {
        Place<V, U>::values(raw[i], v);
#pragma unroll
        for (int e = 0; e < P; ++e) s[e] = pair_fma(v[e], both(-1.0f / B), s[e]);
    }
    if constexpr (B > 1)
#pragma unroll
        for (int i = 0; i < B; ++i) {
            Place<V, U>::values(raw[i], v);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float2 d = pair_add(v[e], s[e]);
                q[e] = pair_fma(d, d, q[e]);
            }
        }
    const float total = m.n + (float)B, fb = __fdividef((float)B, total), f = -m.n * fb;
#pragma unroll
    for (int e = 0; e < P; ++e) {
        const float2 d = pair_add(s[e], m.mean[e]);  // the batch's mean and the rows' before it, apart; minus that
        m.mean[e] = pair_fma(d, both(-fb), m.mean[e]);
        m.m2[e] = pair_add(m.m2[e], pair_fma(pair_mul(d, both(-f)), d, q[e]));
    }
    m.n = total;
}

// Weights of the second of two sets of moments of na and nb values, and their number.
__device__ __forceinline__ float join_weights(float na, float nb, float* fb, float* f) {
    const float n = na + nb;
    *fb = n > 0.0f ? nb / n : 0.0f;
    *f = na * *fb;
    return n;
}

// Moments of the tile's groups over rows [begin, end) of x (its first channel): f(group of the tile, mean, sum of
// squares), called by one thread a group. KEEP: the rows fit the slots and stay there. The strips may be written again
// after a team_sync.
template <bool CTA, bool KEEP, typename TX, int V, int U, typename F>
__device__ __forceinline__ void group_moments(const Team<CTA, V, U>& tm, const Slots<TX, V, U>& slots, const TX* x, int64_t ldx,
                                              int begin, int end, const Tile& k, Strips& sh, F&& f) {
    constexpr int P = V * U / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Moments<P> m;
    auto add = [&](Moments<P>& to, int b, int e) {
        const int rows = tm.rows(e - b);
        auto from = tm.template walk<false>(x, b, rows, ldx);
        auto fill = [&](int slot) { slots.fill(slot, from.next(), tm.at); };
        auto use = [&](auto full, int slot) {
            constexpr int B = decltype(full)::value ? BATCH : 1;
            Pack<TX, V> raw[B][U];
#pragma unroll
            for (int j = 0; j < B; ++j) slots.get(raw[j], slot + j);
            add_rows<B>(to, raw);
        };
        if constexpr (KEEP) {
            fill_all(rows, fill);
            use_all(rows, use);
        } else {
            stream<RING_BYTES / Slots<TX, V, U>::BYTES / BATCH>(rows, fill, use);
        }
    };
    if constexpr (KEEP) {
        add(m, begin, end);
    } else {
        const int most = TERMS * BATCH << tm.step_log;
#pragma unroll 1
        for (int b = begin; b < end; b += most) {
            Moments<P> part;
            add(part, b, min(end, b + most));
            float fb, f;
            m.n = join_weights(m.n, part.n, &fb, &f);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                join_moments(m.mean[e].x, m.m2[e].x, part.mean[e].x, part.m2[e].x, fb, f);
                join_moments(m.mean[e].y, m.m2[e].y, part.mean[e].y, part.m2[e].y, fb, f);
            }
        }
    }
    for (int o = 16; o >= tm.at.lpr; o >>= 1) {
        // both of a pair take the lower lane's moments first, so that they end with the same numbers
        const bool low = (lane & o) == 0;
        const float other = __shfl_xor_sync(0xffffffffu, m.n, o);
        float fb, g;
        const float n = join_weights(low ? m.n : other, low ? other : m.n, &fb, &g);
        auto join = [&](float& mean, float& m2) {
            const float mo = __shfl_xor_sync(0xffffffffu, mean, o), so = __shfl_xor_sync(0xffffffffu, m2, o);
            float ma = low ? mean : mo, sa = low ? m2 : so;
            join_moments(ma, sa, low ? mo : mean, low ? so : m2, fb, g);
            mean = ma;
            m2 = sa;
        };
#pragma unroll
        for (int e = 0; e < P; ++e) {
            join(m.mean[e].x, m.m2[e].x);
            join(m.mean[e].y, m.m2[e].y);
        }
        m.n = n;
    }
    team_sync<CTA>();
    if (lane < tm.at.lpr) put_channels(m.mean, m.m2, tm.at, sh.v[warp]);
    if (lane == 0) sh.n[warp] = m.n;
    team_sync<CTA>();
    if constexpr (CTA) {
        const int c = threadIdx.x;
        if (c < k.cols) {
            // means about one of them: equal ones give that value, and no sum of them leaves the range
            const float per = 1.0f / (float)(end - begin), base = sh.v[0][0][c];
            float mean = 0.0f, m2 = 0.0f;
#pragma unroll
            for (int w = 1; w < WARPS; ++w) mean = fmaf(sh.n[w] * per, sh.v[w][0][c] - base, mean);
            mean += base;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float d = sh.v[w][0][c] - mean;
                m2 += fmaf(sh.n[w] * d, d, sh.v[w][1][c]);
            }
            sh.v[0][0][c] = mean;
            sh.v[0][1][c] = m2;
        }
        __syncthreads();
    }
    // every channel has the same number of values
    const float* cm = sh.v[CTA ? 0 : warp][0];
    const float* cs = sh.v[CTA ? 0 : warp][1];
    const float n = (float)(end - begin), per = 1.0f / (float)k.lw;
    each_group<CTA>(k.ng, [&](int g, int j, int l, bool live) {
        float s = 0.0f;
        const float base = live ? cm[g * k.lw] : 0.0f;
        if (live)
            for (int c = j; c < k.lw; c += l) s = fmaf(cm[g * k.lw + c] - base, per, s);
        const float mean = base + group_sum(s, l);
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

// y of rows [begin, end) from the groups' minus mean and rstd at gm and gr[group of the tile]. KEPT: the rows are in the
// slots. BACK: the last rows first.
template <bool CTA, bool KEPT, bool BACK, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void apply(const Forward<TX, TY>& p, const Team<CTA, V, U>& tm, const Slots<TX, V, U>& slots,
                                      int begin, int end, const Tile& k, const float* gm, const float* gr) {
    constexpr int P = V * U / 2;
    float2 w[P], b[P], m[P], rs[P];
    tm.at.param(w, p.a.w, k.c0, 1.0f);
    tm.at.param(b, p.a.b, k.c0, 0.0f);
    tm.of_groups(m, gm, k);
    tm.of_groups(rs, gr, k);
    const int rows = tm.rows(end - begin);
    auto from = tm.template walk<BACK>(p.a.x + k.c0, begin, rows, p.a.ldx);
    auto to = tm.template walk<BACK>(p.y + k.c0, begin, rows, p.ldy);
    with_act(p.a.act, [&](auto act) {
        auto use = [&](auto full, int slot) {
#pragma unroll
            for (int j = 0; j < (decltype(full)::value ? BATCH : 1); ++j) {
                Pack<TX, V> raw[U];
                slots.get(raw, slot + j);
                float2 v[P];
                Place<V, U>::values(raw, v);
#pragma unroll
                for (int e = 0; e < P; ++e) v[e] = affine(centred(v[e], m[e], rs[e]), w[e], b[e]);
                act_row<false, sizeof(TY) == 4, decltype(act)::value>(v);
                tm.at.store(to.next(), v);
            }
        };
        if constexpr (KEPT) use_all(rows, use);
        else stream<RING_BYTES / Slots<TX, V, U>::BYTES / BATCH>(rows, [&](int slot) { slots.fill(slot, from.next(), tm.at); }, use);
    });
}

// A group's statistics: gm and gr take minus the mean and rstd, the caller's arrays the mean and rstd.
template <typename TX, typename TY>
__device__ __forceinline__ void finish(const Forward<TX, TY>& p, int s, int group, float mean, float m2, float count,
                                       bool out, float* gm, float* gr) {
    const float rs = 1.0f / sqrtf(m2 / count + p.eps);
    const int64_t at = (int64_t)s * p.t.groups + group;
    if (out && p.mean) p.mean[at] = mean;
    if (out && p.rstd) p.rstd[at] = rs;
    *gm = -mean;
    *gr = rs;
}

// A sample by a team. KEEP: it is one tile and fits the slots; else all tiles of the block are read twice.
template <bool CTA, bool KEEP, typename TX, typename TY, int V, int U>
__device__ __forceinline__ void whole_sample(const Forward<TX, TY>& p, const Slots<TX, V, U>& slots, int s, Span rows, int block,
                                             Strips& sh, float* gm, float* gr) {
    const int tpg = KEEP ? 1 : p.t.tpg, t0 = block * tpg;
    const float n = (float)(rows.end - rows.begin);
    for (int j = 0; j < tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        group_moments<CTA, KEEP>(tm, slots, p.a.x + k.c0, p.a.ldx, rows.begin, rows.end, k, sh, [&](int g, float mean, float m2) {
            if (j > 0) {  // the same thread's moments of the tiles before
                float ma = gm[g], sa = gr[g], fb, f;
                join_weights(n * (float)(j * p.t.max_cols), n * (float)k.lw, &fb, &f);
                join_moments(ma, sa, mean, m2, fb, f);
                mean = ma;
                m2 = sa;
            }
            gm[g] = mean;
            gr[g] = m2;
            if (j + 1 == tpg) finish(p, s, k.g0 + g, mean, m2, n * (float)p.t.width, true, gm + g, gr + g);
        });
        team_sync<CTA>();
    }
    for (int j = 0; j < tpg; ++j) {
        const Tile k = tile_of(p.t, t0 + j);
        const Team<CTA, V, U> tm(p.t, k.cols);
        apply<CTA, KEEP, false>(p, tm, slots, rows.begin, rows.end, k, gm, gr);
    }
    team_sync<CTA>();
}

// CTAs [0, chunks x tiles): moments of the long samples' chunks. The others: short and middle samples.
template <typename TX, typename TY, int V, int U>
__global__ void __launch_bounds__(THREADS, CTAS) group_norm_kernel(const __grid_constant__ Forward<TX, TY> p) {
    __shared__ Strips sh;
    __shared__ float gm[WARPS][MAX_TILE], gr[WARPS][MAX_TILE];
    extern __shared__ __align__(16) uint8_t slot_memory[];
    const Slots<TX, V, U> slots{slot_memory};
    constexpr int ROWS = SLOT_BYTES / Slots<TX, V, U>::BYTES;  // of a thread in the slots
    cudaGridDependencySynchronize();
    const int chunked = p.ch.count * p.t.tiles;
    if ((int)blockIdx.x < chunked) {
        const int i = blockIdx.x / p.t.tiles, tile = blockIdx.x - i * p.t.tiles;
        const int2 found = long_samples(p.a.offsets, (int)p.a.samples, (int)p.a.rows, p.ch, i);
        if (tile == 0 && threadIdx.x == 0) p.found[i] = found;
        const Tile k = tile_of(p.t, tile);
        const Team<true, V, U> tm(p.t, k.cols);
        const int total = (int)p.a.rows, r0 = i * p.ch.rows, r1 = r0 + min(p.ch.rows, total - r0);
        const int64_t parts = p.t.tpg == 1 ? p.t.groups : p.t.tiles;
        for (int slot = 0; slot < 2; ++slot) {
            const int s = slot ? found.y : found.x;
            if (s < 0) continue;
            const Span sp = span_of(p.a.offsets, s, total);
            float2* out = p.part + (slot * parts + part_slot(p.t, tile, k)) * p.ch.count + i;
            group_moments<true, false>(tm, slots, p.a.x + k.c0, p.a.ldx, max(r0, sp.begin), min(r1, sp.end), k, sh,
                                   [&](int g, float mean, float m2) { out[(int64_t)g * p.ch.count] = make_float2(mean, m2); });
            __syncthreads();
        }
        return;
    }
    const int warp = threadIdx.x >> 5;
    const int at = blockIdx.x - chunked, samples = (int)p.a.samples;
    const int item = p.t.blocks == 1 ? at : at / p.t.blocks, block = at - item * p.t.blocks, s0 = item * p.each;
    auto rows_of = [&](int s) { return span_of(p.a.offsets, s, (int)p.a.rows); };
    // a sample without rows has statistics all the same
    auto empty = [&](int s) {
        const Tile first = tile_of(p.t, block * p.t.tpg);
        float unused[2];
        for (int g = threadIdx.x & 31; g < first.ng; g += 32)
            finish(p, s, first.g0 + g, 0.0f, 0.0f, 1.0f, true, &unused[0], &unused[1]);
    };
    if (p.each > 1) {
        const int s = s0 + warp;
        if (s < samples) {
            const Span sp = rows_of(s);
            const int n = sp.end - sp.begin;
            if (n == 0) empty(s);
            else if (n <= (ROWS << (5 - p.t.lpr_log))) whole_sample<false, true>(p, slots, s, sp, block, sh, gm[warp], gr[warp]);
        }
        __syncthreads();
    }
    for (int j = 0; j < p.each; ++j) {
        const int s = s0 + j;
        if (s >= samples) break;
        const Span sp = rows_of(s);
        const int n = sp.end - sp.begin;
        if (n == 0 && p.each == 1 && warp == 0) empty(s);
        if (n == 0 || n > p.ch.longest || (p.each > 1 && n <= (ROWS << (5 - p.t.lpr_log)))) continue;
        if (p.t.tpg == 1 && n <= (ROWS << (5 + WARPS_LOG - p.t.lpr_log)))
            whole_sample<true, true>(p, slots, s, sp, block, sh, gm[0], gr[0]);
        else whole_sample<true, false>(p, slots, s, sp, block, sh, gm[0], gr[0]);
    }
}

// y of the long samples' chunks. Every CTA joins the moments of its tile's groups over all of the sample's chunks, a
// warp for a group, whose lanes take every 32nd.
template <typename TX, typename TY, int V, int U>
__global__ void __launch_bounds__(THREADS, CTAS) group_norm_apply_kernel(const __grid_constant__ Forward<TX, TY> p) {
    __shared__ float gm[MAX_TILE], gr[MAX_TILE];
    extern __shared__ __align__(16) uint8_t slot_memory[];
    const Slots<TX, V, U> slots{slot_memory};
    cudaGridDependencySynchronize();
    const int i = p.ch.count - 1 - blockIdx.x / p.t.tiles, tile = blockIdx.x % p.t.tiles;
    const int2 found = p.found[i];
    if (found.x < 0 && found.y < 0) return;
    const Tile k = tile_of(p.t, tile);
    const Team<true, V, U> tm(p.t, k.cols);
    const int total = (int)p.a.rows, r0 = i * p.ch.rows, r1 = r0 + min(p.ch.rows, total - r0);
    const int tpg = p.t.tpg, lane = threadIdx.x & 31;
    for (int slot = 1; slot >= 0; --slot) {
        const int s = slot ? found.y : found.x;
        if (s < 0) continue;
        const Span sp = span_of(p.a.offsets, s, total);
        const Parts parts(sp, p.ch, tpg == 1 ? p.t.groups : p.t.tiles);
        const bool lost = not_found(p.found, parts, s);
        for (int g = threadIdx.x >> 5; g < k.ng; g += WARPS) {
            // the mean of the parts' means, then the squares about it
            const int n_rows = sp.end - sp.begin;
            const float n = (float)n_rows * (float)p.t.width;
            const int lead = min(n_rows, (parts.first + 1) * p.ch.rows - sp.begin), trail = n_rows - lead - (parts.count - 2) * p.ch.rows;
            auto each_part = [&](auto&& f) {
                for (int part = 0; part < tpg; ++part) {
                    const int lw = tpg == 1 ? p.t.width : min(p.t.max_cols, p.t.width - part * p.t.max_cols);
#pragma unroll 8
                    for (int c = lane; c < parts.count; c += 32) {
                        const int in = c == 0 ? lead : c == parts.count - 1 ? trail : p.ch.rows;
                        f((float)in * (float)lw, parts.get(p.part, (int64_t)(k.g0 + g) * tpg + part, c));
                    }
                }
            };
            const float base = parts.get(p.part, (int64_t)(k.g0 + g) * tpg, 0).x, per = 1.0f / n;
            float mean = 0.0f, m2 = 0.0f;
            each_part([&](float count, float2 v) { mean = fmaf(count * per, v.x - base, mean); });
            mean = base + group_sum(mean, 32);
            each_part([&](float count, float2 v) {
                const float d = v.x - mean;
                m2 += fmaf(count * d, d, v.y);
            });
            m2 = group_sum(m2, 32);
            if (lost) mean = m2 = __uint_as_float(0x7fc00000u);
            if (lane == 0) finish(p, s, k.g0 + g, mean, m2, n, slot == 1 && (tpg == 1 || tile % tpg == 0), gm + g, gr + g);
        }
        __syncthreads();
        apply<true, false, true>(p, tm, slots, max(r0, sp.begin), min(r1, sp.end), k, gm, gr);
    }
}

template <typename TX, typename TY, int V, int U>
void forward(Handle& h, Forward<TX, TY>& p) {
    const Cut cut = make_cut(p.a, p.t, (int)sizeof(TX), V > 1, sm_count(h.device), CTAS);
    p.ch = cut.ch;
    p.each = cut.by_warp ? WARPS : 1;
    DevBuf<float2> part((size_t)p.ch.count * 2 * part_slots(p.t), h.stream);
    DevBuf<int2> found((size_t)p.ch.count, h.stream);
    p.part = part.get();
    p.found = found.get();
    const int64_t chunked = (int64_t)p.ch.count * p.t.tiles;
    const int64_t grid = chunked + (cut.only_long ? 0 : ceil_div(p.a.samples, p.each) * p.t.blocks);
    XS_REQUIRE(grid < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "too many samples and groups");
    allow_smem(group_norm_kernel<TX, TY, V, U>, SLOT_BYTES * THREADS);
    launch_dependent(h.stream, group_norm_kernel<TX, TY, V, U>, (unsigned)grid, THREADS, SLOT_BYTES * THREADS, 1, p);
    after_launch(h, "group_norm");
    if (p.ch.count == 0) return;
    launch_dependent(h.stream, group_norm_apply_kernel<TX, TY, V, U>, (unsigned)chunked, THREADS, RING_BYTES * THREADS, 1, p);
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
    const size_t bx = PER * sizeof(TX), by = PER * sizeof(TY);
    const bool wide = a.C % PER == 0 && (a.rows <= 1 || (a.ldx % PER == 0 && ldy % PER == 0)) && aligned_to(a.x, bx) &&
                      aligned_to(y, by);
    if (wide && make_tiling(p.t, a, PER, 1, sm_count(h.device))) return forward<TX, TY, PER, 1>(h, p);
    make_tiling(p.t, a, 1, PER, sm_count(h.device));
    forward<TX, TY, 1, PER>(h, p);
}

#define XS_INST_GROUP_NORM(TX, TY) \
    template void group_norm<TX, TY>(Handle&, const GroupNormArgs<TX>&, float, TY*, int64_t, float*, float*);
XS_INST_GROUP_NORM(__half, __half)
XS_INST_GROUP_NORM(__nv_bfloat16, __nv_bfloat16)
XS_INST_GROUP_NORM(float, float)
XS_INST_GROUP_NORM(float, __half)
XS_INST_GROUP_NORM(float, __nv_bfloat16)

}  // namespace xspmm_b200
