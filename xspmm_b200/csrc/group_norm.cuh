// group_norm.cuh -- what the group norm and its gradient share: how channels and rows are cut, sums over a team of
// threads, the activation and its slope. group_norm.cu explains the whole.
#pragma once

#include "gated_tc.cuh"

namespace xspmm_b200 {
namespace group {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_TILE = 256;  // channels of a column tile

// Channels are cut into column tiles: whole groups side by side (gpt of them), or, where a group is wider than a
// tile, tpg tiles to a group. A block is a tile, or all tiles of a wide group: what shares statistics.
struct Tiling {
    int groups, width;  // width: channels of a group
    int gpt, tpg, tiles, blocks;
    int max_cols;       // channels of the widest tile
    int lpr;            // threads side by side in a row, a power of two up to 32
};
struct Tile {
    int c0, cols;  // channels [c0, c0 + cols)
    int g0, ng;    // groups [g0, g0 + ng)
    int lw;        // channels of each of them in the tile
};
__device__ __forceinline__ Tile tile_of(const Tiling& t, int i) {
    Tile k;
    if (t.tpg == 1) {
        k.g0 = i * t.gpt;
        k.ng = min(t.gpt, t.groups - k.g0);
        k.c0 = k.g0 * t.width;
        k.cols = k.ng * t.width;
        k.lw = t.width;
    } else {
        k.g0 = i / t.tpg;
        k.ng = 1;
        const int off = (i - k.g0 * t.tpg) * t.max_cols;
        k.c0 = k.g0 * t.width + off;
        k.lw = k.cols = min(t.max_cols, t.width - off);
    }
    return k;
}
// Slot of a tile's first group among the partial sums of a chunk of rows: one a group, or one a tile of it.
__device__ __forceinline__ int part_slot(const Tiling& t, int tile, const Tile& k) { return t.tpg == 1 ? k.g0 : tile; }
inline int part_slots(const Tiling& t) { return t.tpg == 1 ? t.groups : t.tiles; }

// Rows are cut into chunks for samples too long for one CTA. `longest` rows are the most that a CTA takes by
// itself; a chunk is no longer, so at most two long samples have rows in one: one that began before it (slot 0)
// and one that begins in it (slot 1).
struct Chunks {
    int64_t rows;     // of a chunk
    int64_t longest;
    int count;        // 0: no sample can be long
};

struct Span {
    int64_t begin, end;
};
// Sample s's rows, within the matrix whatever the offsets hold.
__device__ __forceinline__ Span span_of(const int64_t* offsets, int64_t s, int64_t rows) {
    if (!offsets) return {0, rows};
    const int64_t b = max((int64_t)0, min(rows, offsets[s]));
    return {b, max(b, min(rows, offsets[s + 1]))};
}
// The last sample that begins at or before row r, -1 if none does. A warp's threads call it together and probe 32
// offsets at a time.
__device__ __forceinline__ int last_begun(const int64_t* offsets, int samples, int64_t r) {
    if (!offsets) return 0;
    int lo = 0, n = samples;  // the answer is lo - 1 + (how many of the next n begin by r)
    while (n > 0) {
        const int step = (n + 31) / 32, at = min((int)(threadIdx.x & 31) * step + step, n) - 1;  // the last of a part
        const int hits = __popc(__ballot_sync(0xffffffffu, offsets[lo + at] <= r));
        // whole parts that begin by r; the next one's last does not, so it is not looked at again
        const int done = min(hits * step, n);
        if (done == n) return lo + n - 1;
        lo += done;
        n = min(step, n - done) - 1;
    }
    return lo - 1;
}
// The long samples with rows in chunk i, -1 where there is none; the same in all threads.
__device__ __forceinline__ int2 long_samples(const int64_t* offsets, int samples, int64_t rows, const Chunks& ch, int i) {
    __shared__ int found[2];
    const int64_t r0 = i * ch.rows, r1 = min(rows, r0 + ch.rows);
    const int warp = threadIdx.x >> 5;
    if (warp < 2) {
        int s = last_begun(offsets, samples, warp == 0 ? r0 : r1 - 1);
        if (s >= 0) {
            const Span sp = span_of(offsets, s, rows);
            if (sp.end - sp.begin <= ch.longest || (warp == 0 ? sp.begin >= r0 : sp.begin < r0)) s = -1;
        }
        if ((threadIdx.x & 31) == 0) found[warp] = s;
    }
    __syncthreads();
    return make_int2(found[0], found[1]);
}

// A thread's channels of a tile: V consecutive ones at each of U places, lpr * V apart.
template <int V, int U>
struct Place {
    int lane, lpr, cols;
    __device__ int col(int u) const { return (u * lpr + lane) * V; }
    __device__ bool in(int u) const { return col(u) < cols; }
    template <typename T>
    __device__ void load(Pack<T, V> (&raw)[U], const T* row) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u] = Pack<T, V>{};
            if (in(u)) raw[u] = *reinterpret_cast<const Pack<T, V>*>(row + col(u));
        }
    }
    template <typename T>
    static __device__ void values(const Pack<T, V> (&raw)[U], float (&v)[V * U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V];
            unpack<T, V>(raw[u], f);
#pragma unroll
            for (int e = 0; e < V; ++e) v[u * V + e] = f[e];
        }
    }
    template <typename T>
    __device__ void store(T* row, const float (&v)[V * U]) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = v[u * V + e];
            if (in(u)) store_pack<T, V>(row + col(u), f);
        }
    }
    // A parameter vector's values at the tile's channels, `none` where it is absent.
    __device__ void param(float (&v)[V * U], const float* p, int c0, float none) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) v[u * V + e] = p && in(u) ? __ldg(p + c0 + col(u) + e) : none;
    }
};

// A team is a warp or the CTA.
template <bool CTA>
__device__ __forceinline__ void team_sync() {
    if constexpr (CTA) __syncthreads();
    else __syncwarp();
}

// A team's threads on a tile: thread t takes channels by t mod lpr and rows t / lpr, t / lpr + step, ...
template <bool CTA, int V, int U>
struct Team {
    Place<V, U> at;
    int rl, step;
    __device__ Team(const Tiling& t, int cols) {
        const int id = CTA ? threadIdx.x : threadIdx.x & 31;
        at.lpr = t.lpr;
        at.cols = cols;
        at.lane = id & (t.lpr - 1);
        rl = id / t.lpr;
        step = (CTA ? THREADS : 32) / t.lpr;
    }
    // The values of the tile's groups at this thread's channels.
    __device__ void of_groups(float (&v)[V * U], const float* g, const Tile& k) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) v[u * V + e] = g[at.in(u) ? (at.col(u) + e) / k.lw : 0];
    }
};

// Shared memory of a team's sums over rows: two values a channel, for each warp.
struct Strips {
    float v[WARPS][2][MAX_TILE];
    float n[WARPS];
};

// Joins (nb, mb, sb) into (na, ma, sa): counts, means and sums of squares about the mean (Chan, Golub and LeVeque,
// 1979). fb = nb / (na + nb) and f = na nb / (na + nb) are the same for all channels of a row.
__device__ __forceinline__ void join_moments(float& ma, float& sa, float mb, float sb, float fb, float f) {
    const float d = mb - ma;
    ma = fmaf(d, fb, ma);
    sa += fmaf(d * d, f, sb);
}

// The sums over a team's threads of two values a channel, at `out` (strips of this warp, or of the CTA's first) by
// channel of the tile. Every thread of the team has the result on return and may not write the strips before its next
// team_sync.
template <bool CTA, int V, int U>
__device__ __forceinline__ void sum_channels(float (&a)[V * U], float (&b)[V * U], const Place<V, U>& at, Strips& sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int o = 16; o >= at.lpr; o >>= 1)
#pragma unroll
        for (int e = 0; e < V * U; ++e) {
            a[e] += __shfl_xor_sync(0xffffffffu, a[e], o);
            b[e] += __shfl_xor_sync(0xffffffffu, b[e], o);
        }
    team_sync<CTA>();
    if (lane < at.lpr)
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at.in(u))
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sh.v[warp][0][at.col(u) + e] = a[u * V + e];
                    sh.v[warp][1][at.col(u) + e] = b[u * V + e];
                }
    team_sync<CTA>();
    if constexpr (CTA) {
        if ((int)threadIdx.x < at.cols) {
            float s = sh.v[0][0][threadIdx.x], t = sh.v[0][1][threadIdx.x];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) s += sh.v[w][0][threadIdx.x], t += sh.v[w][1][threadIdx.x];
            sh.v[0][0][threadIdx.x] = s;
            sh.v[0][1][threadIdx.x] = t;
        }
        __syncthreads();
    }
}

// Threads of a team that sum one of ng groups: a power of two up to 32.
template <bool CTA>
__device__ __forceinline__ int threads_a_group(int ng) {
    int l = 32;
    while (l > 1 && l * ng > (CTA ? THREADS : 32)) l >>= 1;
    return l;
}
// f(group of the tile, thread of the group, threads a group) for every group, all the group's threads together in a
// warp; groups past the last are called with live = false.
template <bool CTA, typename F>
__device__ __forceinline__ void each_group(int ng, F&& f) {
    const int l = threads_a_group<CTA>(ng), t = CTA ? threadIdx.x : threadIdx.x & 31, step = (CTA ? THREADS : 32) / l;
    for (int base = 0; base < ng; base += step) {
        const int i = base + t / l;
        f(i, t % l, l, i < ng);
    }
}
__device__ __forceinline__ float group_sum(float v, int l) {
    for (int o = l >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// z, each operation rounded by itself: the sign of z, which decides relu's slope, is then the same in the forward
// and the backward pass and however the compiler orders the code around it.
__device__ __forceinline__ float centred(float x, float mean, float rstd) { return __fmul_rn(__fsub_rn(x, mean), rstd); }
__device__ __forceinline__ float affine(float xh, float w, float b) { return __fadd_rn(__fmul_rn(xh, w), b); }

// act(z) of a row's values and its slope. 16-bit outputs take the gated block's approximate forms (errors far below
// their rounding), fp32 ones CUDA's accurate functions.
template <bool FINE, Activation ACT>
__device__ __forceinline__ float act_one(float z) {
    if constexpr (ACT == Activation::None) return z;
    else if constexpr (!FINE) return gated::act_value<ACT>(z);
    else if constexpr (ACT == Activation::Silu) return z > -gated::SILU_END ? z / (1.0f + expf(-z)) : (z != z ? z : 0.0f);
    else if constexpr (ACT == Activation::Gelu) return z > -gated::GELU_END ? z * normcdff(z) : (z != z ? z : 0.0f);
    else if constexpr (ACT == Activation::Sigmoid) return 1.0f / (1.0f + expf(-z));
    else return z > 0.0f ? z : (z != z ? z : 0.0f);
}
template <bool FINE, Activation ACT>
__device__ __forceinline__ float slope_one(float z) {
    if constexpr (ACT == Activation::None) return 1.0f;
    else if constexpr (ACT == Activation::Relu) return z > 0.0f ? 1.0f : 0.0f;
    else if constexpr (!FINE) {
        float value, slope;
        gated::act_both<ACT>(z, &value, &slope);
        return slope;
    } else if constexpr (ACT == Activation::Silu) {
        const float low = gated::max_nan(gated::min_nan(z, gated::SILU_END), -gated::SILU_END);
        // the smaller tail from the exponential itself: 1 - s would cancel
        const float e = expf(-fabsf(low)), high = 1.0f / (1.0f + e), tail = e * high;
        const float s = low < 0.0f ? tail : high, r = low < 0.0f ? high : tail;
        return s * (1.0f + low * r);
    } else if constexpr (ACT == Activation::Gelu) {
        const float low = gated::max_nan(gated::min_nan(z, gated::GELU_END), -gated::GELU_END);
        return normcdff(low) + low * 0.39894228040143268f * expf(-0.5f * low * low);
    } else {
        const float e = expf(-fabsf(z)), high = 1.0f / (1.0f + e);
        return high * (e * high);
    }
}
// One branch for a row's values.
template <typename F>
__device__ __forceinline__ void with_act(Activation act, F&& f) {
    if (act == Activation::None) f(std::integral_constant<Activation, Activation::None>{});
    else gated::with_activation(act, f);
}

// ---- host ---------------------------------------------------------------------------------------------
// Column tiles of `vec` elements a thread and at most `most` channels a tile. A tile that starts within a 16-byte
// word cannot take wide loads: false where the groups' width allows none that does not.
inline bool make_tiling(Tiling& t, int64_t C, int64_t groups, int vec, int places, int most) {
    t.groups = (int)groups;
    t.width = (int)(C / groups);
    if (t.width > most) {
        if (t.width % vec != 0) return false;
        t.gpt = 1;
        t.tpg = (int)ceil_div(t.width, most);
        t.max_cols = most;
        t.tiles = t.groups * t.tpg;
        t.blocks = t.groups;
    } else {
        int unit = 1;  // groups that make whole words
        while (unit * t.width % vec != 0) unit *= 2;
        if (unit * t.width > most && unit < groups) return false;
        t.gpt = (int)std::min<int64_t>(groups, std::max(1, most / t.width / unit) * unit);
        t.tpg = 1;
        t.max_cols = t.gpt * t.width;
        if (t.max_cols > most) return false;
        t.tiles = t.blocks = (int)ceil_div(groups, t.gpt);
    }
    t.lpr = 1;
    while (t.lpr < 32 && t.lpr * vec * places < t.max_cols) t.lpr *= 2;
    return true;
}

// Who takes which samples. `longest`: 256 KB of a tile's columns, which the CTAs of a wave hold in L2 between their
// two reads. Chunks: about four a wave's CTA, at least 64 rows. Short samples go to warps where that leaves every
// SM 16 of them at least; a warp takes up to 64 KB.
struct Cut {
    Chunks ch;
    int each;
    int64_t warp_rows;
    bool only_long;  // all rows are one sample, and it is long
};
template <typename TX>
Cut make_cut(const GroupNormArgs<TX>& a, const Tiling& t, int bytes, int sms) {
    const int64_t rows = a.rows, samples = a.samples;
    Cut c = {};
    const int64_t row = (int64_t)t.max_cols * bytes;
    c.ch.longest = std::max<int64_t>(256, (256 << 10) / row);
    if (rows > c.ch.longest) {
        c.ch.rows = std::min(c.ch.longest, std::max<int64_t>(64, ceil_div(rows * t.tiles, 16 * sms)));
        c.ch.count = (int)ceil_div(rows, c.ch.rows);
    }
    c.each = samples * t.blocks >= 16 * sms && t.tpg == 1 ? WARPS : 1;
    c.warp_rows = std::max<int64_t>(1, (64 << 10) / row);
    c.only_long = !a.offsets && rows > c.ch.longest;
    return c;
}

}  // namespace group
}  // namespace xspmm_b200
