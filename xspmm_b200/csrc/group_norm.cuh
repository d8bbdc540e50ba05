// group_norm.cuh -- what the group norm and its gradient share: how channels and rows are cut, sums over a team of
// threads, the activation and its slope. group_norm.cu explains the whole.
#pragma once

#include "gated_tc.cuh"

namespace xspmm_b200 {
namespace group {

constexpr int WARPS_LOG = 2, WARPS = 1 << WARPS_LOG, THREADS = 32 * WARPS;
constexpr int PER = 4;         // channels a thread holds of a row
constexpr int MAX_TILE = 32 * PER;  // channels of a column tile

// Two fp32 operations in one instruction. The compiler's own, not layers.cuh's inline assembly: it then keeps pairs in
// aligned registers through a whole loop (2^20 x 128 fp32 to fp16 with silu, second pass: 27 instructions a value with
// the assembly).
__device__ __forceinline__ float2 pair_add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 pair_mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 pair_fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
// A product that is rounded by itself whatever is added to it: a packed one and an addition are joined to one operation,
// as the results show, .rn or not.
__device__ __forceinline__ float2 pair_mul_alone(float2 a, float2 b) {
    return make_float2(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y));
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Channels are cut into column tiles: whole groups side by side (gpt of them), or, where a group is wider than a
// tile, tpg tiles to a group. A block is a tile, or all tiles of a wide group: what shares statistics.
struct Tiling {
    int groups, width;  // width: channels of a group
    int gpt, tpg, tiles, blocks;
    int max_cols;       // channels of the widest tile
    int lpr, lpr_log;   // threads side by side in a row, a power of two up to 32
    uint32_t inv;       // 2^16 / width rounded up (groups within a tile)
};
struct Tile {
    int c0, cols;  // channels [c0, c0 + cols)
    int g0, ng;    // groups [g0, g0 + ng)
    int lw;        // channels of each of them in the tile
    uint32_t inv;  // 2^16 / lw rounded up: exact for the channels of a tile
    __device__ int group(int c) const { return (int)(c * inv >> 16); }
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
    k.inv = t.tpg == 1 ? t.inv : 0;
    return k;
}
// Slot of a tile's first group among the partial sums of a chunk of rows: one a group, or one a tile of it.
__device__ __forceinline__ int part_slot(const Tiling& t, int tile, const Tile& k) { return t.tpg == 1 ? k.g0 : tile; }
inline int part_slots(const Tiling& t) { return t.tpg == 1 ? t.groups : t.tiles; }

// Rows are cut into chunks for samples too long for one CTA. `longest` rows are the most that a CTA takes by
// itself; a chunk is no longer, so at most two long samples have rows in one: one that began before it (slot 0)
// and one that begins in it (slot 1).
struct Chunks {
    int rows;     // of a chunk
    int longest;
    int count;    // 0: no sample can be long
};

struct Span {
    int begin, end;
};
// Sample s's rows, within the matrix whatever the offsets hold.
__device__ __forceinline__ Span span_of(const int64_t* offsets, int s, int rows) {
    if (!offsets) return {0, rows};
    const int b = (int)max((int64_t)0, min((int64_t)rows, offsets[s]));
    return {b, max(b, (int)max((int64_t)0, min((int64_t)rows, offsets[s + 1])))};
}
// The last sample that begins at or before row r, -1 if none does. A warp's threads call it together and probe 32
// offsets at a time. Offsets that decrease give some sample or -1.
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
// A long sample's chunks: it belongs to the one it begins in, where its part is in slot 1; in the others it is in slot 0.
struct Parts {
    int first, count;       // chunks first ... first + count - 1
    int64_t slots, chunks;  // parts[slot][part of the tile's groups][chunk]
    __device__ Parts(const Span& sp, const Chunks& ch, int64_t slots_) : slots(slots_), chunks(ch.count) {
        first = sp.begin / ch.rows;
        count = (sp.end - 1) / ch.rows - first + 1;
    }
    __device__ float2 get(const float2* part, int64_t slot, int i) const {
        return part[((int64_t)(i == 0) * slots + slot) * chunks + first + i];
    }
};

// The long samples with rows in chunk i, -1 where there is none; the same in all threads.
__device__ __forceinline__ int2 long_samples(const int64_t* offsets, int samples, int rows, const Chunks& ch, int i) {
    __shared__ int found[2];
    const int r0 = i * ch.rows, r1 = r0 + min(ch.rows, rows - r0);
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

// Whether a chunk of long sample s, its parts being `parts`, does not have it: the offsets decrease, and what parts[] holds
// for it is in part not of this call. Called by the whole CTA; the same in all threads.
__device__ __forceinline__ bool not_found(const int2* found, const Parts& parts, int s) {
    bool lost = false;
    for (int i = threadIdx.x; i < parts.count; i += THREADS) {
        const int2 f = found[parts.first + i];
        lost = lost || (i == 0 ? f.y : f.x) != s;
    }
    return __syncthreads_or(lost);
}

// A thread's channels of a tile: V consecutive ones at each of U places, lpr * V apart. Pointers to rows are at the
// thread's first channel.
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
            if (U == 1 || in(u)) raw[u] = *reinterpret_cast<const Pack<T, V>*>(row + u * lpr * V);
        }
    }
    template <typename T>
    static __device__ void values(const Pack<T, V> (&raw)[U], float2 (&v)[V * U / 2]) {
        if constexpr (V == 1) {
#pragma unroll
            for (int u = 0; u < U; u += 2) v[u / 2] = make_float2(to_float(raw[u].v[0]), to_float(raw[u + 1].v[0]));
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[V];
                unpack<T, V>(raw[u], f);
#pragma unroll
                for (int e = 0; e < V; e += 2) v[(u * V + e) / 2] = make_float2(f[e], f[e + 1]);
            }
        }
    }
    template <typename T>
    __device__ void store(T* row, const float2 (&v)[V * U / 2]) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = (u * V + e) % 2 ? v[(u * V + e) / 2].y : v[(u * V + e) / 2].x;
            if (U == 1 || in(u)) store_pack<T, V>(row + u * lpr * V, f);
        }
    }
    // f(channel of the tile, whether it is one of its) for each of the thread's channels, as pairs.
    template <typename F>
    __device__ void each(float2 (&v)[V * U / 2], F&& f) const {
#pragma unroll
        for (int i = 0; i < V * U; i += 2) {
            v[i / 2].x = f(col(i / V) + i % V, in(i / V));
            v[i / 2].y = f(col((i + 1) / V) + (i + 1) % V, in((i + 1) / V));
        }
    }
    // A parameter vector's values at the tile's channels, `none` where it is absent.
    __device__ void param(float2 (&v)[V * U / 2], const float* p, int c0, float none) const {
        each(v, [&](int c, bool mine) { return p && mine ? __ldg(p + c0 + c) : none; });
    }
};

// A team is a warp or the CTA.
template <bool CTA>
__device__ __forceinline__ void team_sync() {
    if constexpr (CTA) __syncthreads();
    else __syncwarp();
}

// A thread's rows in a matrix, walked in order: the next one's first channel and the step to the one after.
template <typename T>
struct Walk {
    T* p;
    int64_t step;
    __device__ T* next() {
        T* r = p;
        p += step;
        return r;
    }
};

// A team's threads on a tile: thread t takes channels by t mod lpr and rows t / lpr, t / lpr + step, ...
template <bool CTA, int V, int U>
struct Team {
    Place<V, U> at;
    int rl, step, step_log;
    __device__ Team(const Tiling& t, int cols) {
        const int id = CTA ? threadIdx.x : threadIdx.x & 31;
        at.lpr = t.lpr;
        at.cols = cols;
        at.lane = id & (t.lpr - 1);
        rl = id >> t.lpr_log;
        step_log = (CTA ? 5 + WARPS_LOG : 5) - t.lpr_log;
        step = 1 << step_log;
    }
    // This thread's number of rows among n; none where it has no channels.
    __device__ int rows(int n) const { return at.in(0) && rl < n ? (n - rl + step - 1) >> step_log : 0; }
    // Its `rows` rows of a matrix whose tile is at `p` and whose rows count from `begin`; BACK: the last ones first.
    template <bool BACK, typename T>
    __device__ Walk<T> walk(T* p, int begin, int rows, int64_t ld) const {
        const int64_t first = begin + rl + (BACK ? max(rows - 1, 0) * (int64_t)step : 0);
        return {p + first * ld + at.lane * V, (BACK ? -step : step) * ld};
    }
    // The values of the tile's groups at this thread's channels.
    __device__ void of_groups(float2 (&v)[V * U / 2], const float* g, const Tile& k) const {
        at.each(v, [&](int c, bool mine) { return g[mine ? k.group(c) : 0]; });
    }
};

// ---- a thread's rows through shared memory -----------------------------------------------------------
// Every thread copies the values that it will itself use, asynchronously where the size of its piece of a row allows, to
// slots of its own: no registers are held and no barrier is needed, and all rows of a short sample are in flight at
// once. With registers for two batches instead, 2^18 x 256 bf16 in 4096 samples took 165 us.
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
constexpr int BATCH = 4;  // rows that are worked on together
// Terms that a thread adds up one after the other: sums of more are joined from such ones, so that the rounding of a sum
// does not grow with its length (7000 of 1 + 2^-13 in a row lose 2^-13.5 of it).
constexpr int TERMS = 1024;

// One thread's slots for rows of T.
template <typename T, int V, int U>
struct Slots {
    static constexpr int BYTES = V * U * (int)sizeof(T), PIECE = V * (int)sizeof(T);
    uint8_t* base;  // shared memory; slot i of a thread is at (i * THREADS + thread) * BYTES
    __device__ uint8_t* at(int slot) const { return base + (slot * THREADS + (int)threadIdx.x) * BYTES; }
    __device__ void fill(int slot, const T* row, const Place<V, U>& p) const {
        uint8_t* to = at(slot);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (U == 1 || p.in(u)) {
                const T* from = row + u * p.lpr * V;
                if constexpr (PIECE >= 4) copy_async<PIECE>(to + u * PIECE, from);
                else *reinterpret_cast<T*>(to + u * PIECE) = *from;
            } else {
                *reinterpret_cast<T*>(to + u * PIECE) = T();
            }
    }
    __device__ void get(Pack<T, V> (&raw)[U], int slot) const {
        if constexpr (U == 1) {
            raw[0] = *reinterpret_cast<const Pack<T, V>*>(at(slot));
        } else {
            const Pack<T, V * U> all = *reinterpret_cast<const Pack<T, V * U>*>(at(slot));
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int v = 0; v < V; ++v) raw[u].v[v] = all.v[u * V + v];
        }
    }
};

// All n rows to slots 0, 1, ...; fill(slot) takes the next row.
template <typename F>
__device__ __forceinline__ void fill_all(int n, F&& fill) {
#pragma unroll 4
    for (int i = 0; i < n; ++i) fill(i);
    copies_commit();
    copies_wait<0>();
}
// use(full, slot) for rows already in slots 0, 1, ...: with full (a constant) BATCH of them, one run of instructions without
// branches; else one. Warps at different places of the code have to share the instruction cache, where misses are what
// they wait for most: what is done once a sample is not unrolled.
template <typename F>
__device__ __forceinline__ void use_all(int n, F&& use) {
    int i = 0;
#pragma unroll 1
    for (; i + BATCH <= n; i += BATCH) use(std::true_type{}, i);
#pragma unroll 1
    for (; i < n; ++i) use(std::false_type{}, i);
}
// The same of rows that pass through a ring of RING batches.
template <int RING, typename F, typename G>
__device__ __forceinline__ void stream(int n, F&& fill, G&& use) {
    auto batch = [&](int slot, int left) {
        if (left >= BATCH)
#pragma unroll
            for (int j = 0; j < BATCH; ++j) fill(slot + j);
        else
#pragma unroll 1
            for (int j = 0; j < left; ++j) fill(slot + j);
        copies_commit();  // a group a batch, empty past the last
    };
#pragma unroll 1
    for (int k = 0; k < RING; ++k) batch(k * BATCH, n - k * BATCH);
    int slot = 0;
#pragma unroll 1
    for (int left = n; left > 0; left -= BATCH) {
        copies_wait<RING - 1>();
        if (left >= BATCH) use(std::true_type{}, slot);
        else
#pragma unroll 1
            for (int j = 0; j < left; ++j) use(std::false_type{}, slot + j);
        batch(slot, left - RING * BATCH);
        slot = slot == (RING - 1) * BATCH ? 0 : slot + BATCH;
    }
    copies_wait<0>();
}

// Shared memory of a team's sums over rows: two values a channel, for each warp.
struct Strips {
    float v[WARPS][2][MAX_TILE];
    float n[WARPS];  // rows
};

// Joins (nb, mb, sb) into (na, ma, sa): counts, means and sums of squares about the mean (Chan, Golub and LeVeque,
// 1979). fb = nb / (na + nb) and f = na nb / (na + nb) are the same for all channels of a row. f, 0 where one side has no
// values, comes before the second d: 0 times an infinite square would be NaN.
__device__ __forceinline__ void join_moments(float& ma, float& sa, float mb, float sb, float fb, float f) {
    const float d = mb - ma;
    ma = fmaf(d, fb, ma);
    sa += fmaf(d * f, d, sb);
}

// A thread's two values a channel to a warp's strips.
template <int V, int U>
__device__ __forceinline__ void put_channels(const float2 (&a)[V * U / 2], const float2 (&b)[V * U / 2], const Place<V, U>& at,
                                             float (&strips)[2][MAX_TILE]) {
#pragma unroll
    for (int i = 0; i < V * U; ++i)
        if (at.in(i / V)) {
            const int c = at.col(i / V) + i % V;
            strips[0][c] = i % 2 ? a[i / 2].y : a[i / 2].x;
            strips[1][c] = i % 2 ? b[i / 2].y : b[i / 2].x;
        }
}

// The sums over a team's threads of two values a channel, at `out` (strips of this warp, or of the CTA's first) by
// channel of the tile. Every thread of the team has the result on return and may not write the strips before its next
// team_sync.
template <bool CTA, int V, int U>
__device__ __forceinline__ void sum_channels(float2 (&a)[V * U / 2], float2 (&b)[V * U / 2], const Place<V, U>& at, Strips& sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto from = [](float2 v, int o) {
        return make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o));
    };
    for (int o = 16; o >= at.lpr; o >>= 1)
#pragma unroll
        for (int i = 0; i < V * U / 2; ++i) {
            a[i] = pair_add(a[i], from(a[i], o));
            b[i] = pair_add(b[i], from(b[i], o));
        }
    team_sync<CTA>();
    if (lane < at.lpr) put_channels(a, b, at, sh.v[warp]);
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

// f(group of the tile, thread of the group, threads a group) for every group, all the group's threads together in a
// warp: a power of two up to 32. Groups past the last are called with live = false.
template <bool CTA, typename F>
__device__ __forceinline__ void each_group(int ng, F&& f) {
    constexpr int TEAM_LOG = CTA ? 5 + WARPS_LOG : 5;
    const int log = max(0, min(5, TEAM_LOG - (ng > 1 ? 32 - __clz(ng - 1) : 0))), l = 1 << log;
    const int t = CTA ? threadIdx.x : threadIdx.x & 31;
    for (int base = 0; base < ng; base += 1 << (TEAM_LOG - log)) {
        const int i = base + (t >> log);
        f(i, t & (l - 1), l, i < ng);
    }
}
__device__ __forceinline__ float group_sum(float v, int l) {
    for (int o = l >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// z, each operation rounded by itself: the sign of z, which decides relu's slope, is then the same in the forward
// and the backward pass and however the compiler orders the code around it.
__device__ __forceinline__ float2 centred(float2 x, float2 neg_mean, float2 rstd) { return pair_mul(pair_add(x, neg_mean), rstd); }
__device__ __forceinline__ float2 affine(float2 xh, float2 w, float2 b) { return pair_add(pair_mul_alone(xh, w), b); }

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
// A row's four values one at a time: where a pair's shared reciprocal does not hold.
template <bool SLOPE, Activation ACT>
__device__ __noinline__ float4 singly(float4 z) {
    auto one = [](float v) { return SLOPE ? slope_one<false, ACT>(v) : act_one<false, ACT>(v); };
    return make_float4(one(z.x), one(z.y), one(z.z), one(z.w));
}
// act of a row's values, or its slope, in place of them. 16-bit silu and sigmoid take one reciprocal for two values
// where its product holds (gated_tc.cuh), 16-bit gelu its packed form.
template <bool SLOPE, bool FINE, Activation ACT>
__device__ __forceinline__ void act_row(float2 (&z)[PER / 2]) {
    constexpr int P = PER / 2;
    if constexpr (ACT == Activation::None) {
        if (SLOPE)
#pragma unroll
            for (int i = 0; i < P; ++i) z[i] = both(1.0f);
    } else if constexpr (!FINE && (ACT == Activation::Silu || ACT == Activation::Sigmoid)) {
        bool holds = true;
        float2 v[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float2 x = pair_mul(z[i], both(-1.4426950408889634f));
            const float2 e = make_float2(gated::exp2f_approx(x.x), gated::exp2f_approx(x.y)), a = pair_add(e, both(1.0f));
            const float product = a.x * a.y;
            holds = holds && product <= gated::PAIR_MAX;
            const float2 s = pair_mul(make_float2(a.y, a.x), both(gated::rcp_approx(product)));
            if constexpr (!SLOPE) {
                v[i] = ACT == Activation::Silu ? pair_mul(z[i], s) : s;
            } else {
                const float2 tail = pair_mul(e, s);  // 1 - s without cancelling
                if constexpr (ACT == Activation::Sigmoid) v[i] = pair_mul(s, tail);
                else v[i] = pair_mul(s, pair_fma(make_float2(fminf(z[i].x, gated::SILU_END), fminf(z[i].y, gated::SILU_END)), tail, both(1.0f)));
            }
        }
        if (__builtin_expect(!holds, 0)) {
            const float4 t = singly<SLOPE, ACT>(make_float4(z[0].x, z[0].y, z[1].x, z[1].y));
            v[0] = make_float2(t.x, t.y);
            v[1] = make_float2(t.z, t.w);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) z[i] = v[i];
    } else if constexpr (!FINE && ACT == Activation::Gelu) {
#pragma unroll
        for (int i = 0; i < P; ++i) {  // gated::gelu2 and act_both's slope, packed
            const float2 t = make_float2(fminf(fabsf(z[i].x), gated::GELU_END), fminf(fabsf(z[i].y), gated::GELU_END));
            const float2 a = pair_fma(t, both(gated::GELU_P), both(1.0f));
            const float2 r = pair_mul(make_float2(a.y, a.x), both(gated::rcp_approx(a.x * a.y)));
            float2 q = both(gated::GELU_Q[6]);
#pragma unroll
            for (int j = 5; j >= 0; --j) q = pair_fma(q, r, both(gated::GELU_Q[j]));
            const float2 x = pair_mul(pair_mul(t, t), both(-0.72134752044448170f));
            const float2 bell = make_float2(gated::exp2f_approx(x.x), gated::exp2f_approx(x.y));
            q = pair_mul(pair_mul(q, r), bell);
            if constexpr (!SLOPE) {
                z[i] = pair_fma(make_float2(-t.x, -t.y), q, make_float2(gated::max_nan(z[i].x, 0.0f), gated::max_nan(z[i].y, 0.0f)));
            } else {
                const float2 side = pair_mul(make_float2(copysignf(t.x, z[i].x), copysignf(t.y, z[i].y)), both(0.39894228040143268f));
                const float2 low = make_float2(z[i].x > 0.0f ? 1.0f - q.x : q.x, z[i].y > 0.0f ? 1.0f - q.y : q.y);
                const float2 s = pair_fma(side, bell, low);
                z[i] = make_float2(z[i].x != z[i].x ? z[i].x : s.x, z[i].y != z[i].y ? z[i].y : s.y);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i)
            z[i] = SLOPE ? make_float2(slope_one<FINE, ACT>(z[i].x), slope_one<FINE, ACT>(z[i].y))
                         : make_float2(act_one<FINE, ACT>(z[i].x), act_one<FINE, ACT>(z[i].y));
    }
}
// One branch for a row's values.
template <typename F>
__device__ __forceinline__ void with_act(Activation act, F&& f) {
    if (act == Activation::None) f(std::integral_constant<Activation, Activation::None>{});
    else gated::with_activation(act, f);
}

// Elements of a small call: 8 samples of 200 x 128 bf16 take 11.3 us in narrow tiles, 15.4 in wide ones. Narrow ones are
// still the faster above it (8 samples of 800 rows 11.2 us, in wide ones 34).
constexpr int64_t SMALL = 1 << 18;

// ---- host ---------------------------------------------------------------------------------------------
// Column tiles of `places` times `vec` channels a thread: as wide as may be; in a small call, where there would be fewer
// tiles of samples than two for every SM, narrower, down to 32 bytes of a row. A tile that starts within a word of `vec`
// elements cannot take wide loads: false where the groups' width allows none that does not.
template <typename TX>
bool make_tiling(Tiling& t, const GroupNormArgs<TX>& a, int vec, int places, int sms) {
    t.groups = (int)a.groups;
    t.width = (int)(a.C / a.groups);
    int unit = 1;  // groups that make whole words
    while (unit < t.groups && unit * t.width % vec != 0) unit *= 2;
    unit = std::min(unit, t.groups);
    if (t.width > MAX_TILE) {
        if (t.width % vec != 0) return false;
        t.gpt = 1;
        t.tpg = (int)ceil_div(t.width, MAX_TILE);
        t.max_cols = MAX_TILE;
        t.tiles = t.groups * t.tpg;
        t.blocks = t.groups;
    } else {
        if (unit * t.width > MAX_TILE) return false;
        int most = MAX_TILE;
        const int64_t least = std::max<int64_t>(1, std::min(a.samples, a.rows));
        while (a.rows * a.C <= SMALL && most * sizeof(TX) > 32 && least * ceil_div(a.C, most) < 2 * sms) most /= 2;
        t.gpt = std::min(t.groups, std::max(1, most / t.width / unit) * unit);
        t.tpg = 1;
        t.max_cols = t.gpt * t.width;
        t.tiles = t.blocks = (int)ceil_div(t.groups, t.gpt);
    }
    t.inv = (uint32_t)ceil_div(65536, t.width);
    t.lpr = 1;
    t.lpr_log = 0;
    while (t.lpr < 32 && t.lpr * vec * places < t.max_cols) t.lpr *= 2, ++t.lpr_log;
    return true;
}

// Who takes which samples. Chunks: one for each CTA of a wave (per_sm an SM), at least 64 rows. `longest`: 512 KB of a
// tile's columns but no more rows than a thread can take one after the other in about 20 us (256; fewer in single
// elements), which is less where a channel has under four bytes; or a chunk. One sample of 2000 rows of 128 bf16 takes 14.0 us in
// chunks, 14.2 by a CTA, one of 4000 18.1 and 23.0; of 800 10.4 by a CTA, 15.5 in chunks (the gradient 12.5 and 19.5).
// Samples of less than 4 KB of a tile on the average go to warps, each as far as the warp's slots hold it, since a CTA's
// threads would have a row or two: 2^18 x 128 bf16 in samples of 8 rows 60 us (by CTAs 134), of 4 rows 166 in the gradient
// (414). Up to 8 KB warps are still the faster (16 rows 46 us, by CTAs 77; gradient of 8 rows 120 and 239).
struct Cut {
    Chunks ch;
    bool by_warp;
    bool only_long;  // all rows are one sample, and it is long
};
template <typename TX>
Cut make_cut(const GroupNormArgs<TX>& a, const Tiling& t, int bytes, bool vector, int sms, int per_sm) {
    Cut c = {};
    const int64_t row = (int64_t)t.max_cols * bytes, share = std::max<int64_t>(64, ceil_div(a.rows * t.tiles, per_sm * sms));
    const int64_t step = THREADS / t.lpr;  // rows that a CTA takes at a time
    c.ch.longest = (int)std::max(share, std::min((512 << 10) / row, step * (vector ? 256 : 48)));
    if (a.rows > c.ch.longest) {
        c.ch.rows = (int)share;
        c.ch.count = (int)ceil_div(a.rows, share);
    }
    c.by_warp = a.samples >= WARPS && a.rows * row < a.samples * (4 << 10) && t.tpg == 1;
    c.only_long = !a.offsets && a.rows > c.ch.longest;
    return c;
}

}  // namespace group
}  // namespace xspmm_b200
