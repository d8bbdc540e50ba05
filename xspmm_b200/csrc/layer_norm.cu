// layer_norm.cu -- layer norm over the features of each row, forward and backward.
//
// Forward: mean = sum(x) / D, var = sum((x - mean)^2) / D, rstd = 1 / sqrt(var + eps),
// y = (x - mean) * rstd * w + b. Backward, with xh = (x - mean) * rstd and t = dy * w:
// dx = rstd * (t - mean(t) - xh * mean(t * xh)), dw = sum over rows of dy * xh, db = sum of dy.
// Every sum is held in fp32 in an order fixed by the sizes alone; the variance is summed about the
// mean (x stays in registers, so its second pass costs no memory traffic).
//
// Each input is read once and each output written once, which bounds aligned rows (2^20 x 128 fp32 to fp16:
// 144 us, 126 at the copy bandwidth). What bounds the others: rows of an odd width, the instructions of single
// elements (65537 x 1021 fp16: 110 us for 41; an instruction issues in 64 % of the cycles with 15 warps an SM); the
// gradient of long rows, a row's chain of wait, sums over the CTA and barriers with two CTAs an SM (4096 x 4096
// bf16: 29 us for 15.6; issue in 49 %). A row is held in registers by `tpr` threads (a power of two within a warp, or a whole CTA), E elements a
// thread as loads of V. With that few rows in registers, loads alone would not keep the memory
// busy, so a CTA's next tiles of rows come through a ring in shared memory filled by bulk copies
// (RING), and parameters stay in registers. A tile whose rows do not start on 16 bytes (an odd D) is copied
// with the bytes before it that complete its first 16, and read element by element; rows that the
// copies cannot take (odd strides or addresses) are loaded directly. The weights' gradients are
// kept per thread over all rows a CTA takes (in registers, or for rows above 8192 elements in shared
// memory), written as one partial per CTA and added in CTA order by a second kernel. Rows above
// 16384 elements do not fit a CTA's registers and are read again for each pass.
#include "layers.cuh"
#include "tcgen05.cuh"

#include <climits>

namespace xspmm_b200 {
namespace {

constexpr int LN_MAX_D = 16384;      // longest row held in registers
constexpr int LN_MAX_ACC = 8192;     // longest row whose weight gradients stay in registers
constexpr int LN_RED = 64;           // row_sum: two areas of one value per warp of a CTA
constexpr int LN_SMALL_BLOCK = 128;  // CTA size where a row takes at most a warp

// Sums of N values over the tpr threads of a row. All threads of the CTA call it together; `red`
// alternates between two areas so that one barrier per call is enough.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int tpr, float (*red)[N], int& phase) {
    for (int o = (tpr < 32 ? tpr : 32) >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (tpr <= 32) return;
    float(*area)[N] = red + LN_RED / 2 * phase;
    phase ^= 1;
    const int warps = tpr >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) area[threadIdx.x >> 5][i] = v[i];
    __syncthreads();
    const int width = 1 << (32 - __clz(warps - 1)), at = lane & (width - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = at < warps ? area[at][i] : 0.0f;
    for (int o = width >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

// One CTA's ring of tiles: tile i of the CTA is rows [(blockIdx + i * gridDim) * rpb, + rpb).
constexpr int LN_RING = 8;  // most tiles in flight

// A tile's bytes in memory from the 16-byte boundary at or before its first element. Contiguous rows are
// one copy; the last tile's bytes after its last 16-byte boundary are left to plain loads.
template <typename T>
struct TileSource {
    const T* p;
    int64_t ld;
    int D, rpb;
    int64_t rows;
    bool dense;  // ld == D
    uint32_t bytes;  // of a tile's slot in shared memory

    __device__ int shift(int64_t row) const {  // elements between the slot's start and the tile's
        return dense ? (int)((uint64_t)(row * D) % (16 / sizeof(T))) : 0;
    }
    __device__ uint32_t issue(uint8_t* slot, int64_t row, uint64_t* bar, bool send) const {
        const int n = (int)min((int64_t)rpb, rows - row);
        if (dense) {
            const uint64_t per = 16 / sizeof(T);
            const uint64_t lo = row * D - shift(row), hi = (row + n) * D;
            // up to the next boundary, which the next rows reach, but not past the last row
            const uint64_t top = min((hi + per - 1) / per * per, rows * (uint64_t)D / per * per);
            const uint32_t size = (uint32_t)((top - lo) * sizeof(T));
            if (send && size) bulk_load(slot, p + lo, size, bar);
            return size;
        }
        if (send)
            for (int i = 0; i < n; ++i)
                bulk_load(slot + (size_t)i * D * sizeof(T), p + (row + i) * ld, (uint32_t)(D * sizeof(T)), bar);
        return (uint32_t)(n * D * sizeof(T));
    }
    // Elements of the tile at or past this index (from the slot's start) were not copied.
    __device__ int copied(int64_t row) const {
        if (!dense) return INT_MAX;
        const uint64_t per = 16 / sizeof(T), lo = row * D - shift(row);
        return (int)min((uint64_t)INT_MAX, rows * (uint64_t)D / per * per - lo);
    }
};

// After a wait that ran out: gives the copies still in flight (bounded) time to land.
__device__ __noinline__ void drain(uint64_t* full, int stages, unsigned* err) {
    for (int i = 0; i < stages; ++i) mbar_wait(&full[i], 0, err) && mbar_wait(&full[i], 1, err);
}

// The columns of one thread: load j holds V of them from (tid + j * tpr) * V - off on. Element pair i is
// (2i, 2i + 1) of the thread's elements taken load after load. TAIL1: every load but the last lies
// within the row. OFF: the row does not start on a load's boundary but `off` elements past one (the
// same for every row the thread takes); its first and last loads hold elements of its neighbours too.
template <int V, int CH, bool TAIL1, bool OFF>
struct Columns {
    static constexpr int PAIRS = V * CH / 2;
    int tid, tpr, D, off;
    bool idle;
    __device__ Columns(int tid_, int tpr_, int D_, int64_t row)
        : tid(tid_), tpr(tpr_), D(D_), off(OFF ? (int)((uint64_t)(row * D_) % V) : 0), idle(tid_ >= tpr_) {}
    __device__ int place(int j) const { return (tid + j * tpr) * V; }  // from the boundary
    __device__ int col(int j) const { return place(j) - off; }
    __device__ bool in(int j) const { return (TAIL1 && j < CH - 1) || col(j) < D; }
    __device__ bool whole(int j) const {
        if (!OFF) return in(j);
        return (j > 0 || col(0) >= 0) && ((TAIL1 && j < CH - 1) || col(j) + V <= D);
    }

    // `row`: the row's first element, here aligned at its boundary. Zeros outside the row.
    template <typename T>
    __device__ void load(Pack<T, V> (&raw)[CH], const T* row, bool live) const {
#pragma unroll
        for (int j = 0; j < CH; ++j) raw[j] = Pack<T, V>{};
        if (live && !idle)
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (in(j)) raw[j] = *reinterpret_cast<const Pack<T, V>*>(row + col(j));
    }
    // OFF: the same from `image`, a copy of the row's elements before column `copied` amid its neighbours'.
    template <typename T>
    __device__ void load_off(Pack<T, V> (&raw)[CH], const T* image, const T* row, int copied, bool live) const {
#pragma unroll
        for (int j = 0; j < CH; ++j) raw[j] = Pack<T, V>{};
        if (live && !idle)
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                if (!in(j)) continue;
                raw[j] = *reinterpret_cast<const Pack<T, V>*>(image + col(j));
                if (!whole(j) || col(j) + V > copied)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int c = col(j) + e;
                        if (c < 0 || c >= D) raw[j].v[e] = Pack<T, V>{}.v[0];
                        else if (c >= copied) raw[j].v[e] = row[c];
                    }
            }
    }
    template <typename T>
    static __device__ void pairs(const Pack<T, V> (&raw)[CH], float2 (&v)[PAIRS]) {
        if constexpr (V == 1) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i)
                v[i] = make_float2(to_float(raw[2 * i].v[0]), to_float(raw[2 * i + 1].v[0]));
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                float f[V];
                unpack<T, V>(raw[j], f);
#pragma unroll
                for (int e = 0; e < V; e += 2) v[(j * V + e) / 2] = make_float2(f[e], f[e + 1]);
            }
        }
    }
    // Element pair i of the loads as they came.
    template <typename T>
    static __device__ float2 pair(const Pack<T, V> (&raw)[CH], int i) {
        if constexpr (V == 1) return make_float2(to_float(raw[2 * i].v[0]), to_float(raw[2 * i + 1].v[0]));
        else if constexpr (sizeof(T) == 2) return unpack2(reinterpret_cast<const uint32_t*>(&raw[2 * i / V])[i % (V / 2)], T());
        else return make_float2(raw[2 * i / V].v[2 * i % V], raw[2 * i / V].v[2 * i % V + 1]);
    }
    // (x + neg) * scale * w + b for load j.
    template <typename T>
    static __device__ void affine(float (&o)[V], const Pack<T, V> (&raw)[CH], int j, float2 neg,
                                  float2 scale, const float2 (&w)[PAIRS], const float2 (&b)[PAIRS]) {
        if constexpr (V == 1) {
            o[0] = (to_float(raw[j].v[0]) + neg.x) * scale.x * (j % 2 ? w[j / 2].y : w[j / 2].x) +
                   (j % 2 ? b[j / 2].y : b[j / 2].x);
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const int i = (j * V + e) / 2;
                const float2 t = fma2(mul2(add2(pair(raw, i), neg), scale), w[i], b[i]);
                o[e] = t.x;
                o[e + 1] = t.y;
            }
        }
    }
    // Whether element 2i (second: 2i + 1) lies within the row.
    __device__ bool in_pair(int i, int second) const {
        const int j = V == 1 ? 2 * i + second : 2 * i / V, c = col(j) + (V == 1 ? 0 : 2 * i % V + second);
        if (!OFF) return in(j);
        return (j > 0 || c >= 0) && ((TAIL1 && j < CH - 1) || c < D);
    }
    static __device__ float element(const float2 (&v)[PAIRS], int i) { return i % 2 ? v[i / 2].y : v[i / 2].x; }
    // `p` is the row's first element, aligned at its boundary as the loads are.
    template <typename T>
    __device__ void store(T* p, const float2 (&v)[PAIRS], bool live) const {
        if (!live || idle) return;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = element(v, j * V + e);
            store_load<T>(p, j, f);
        }
    }
    template <typename T>
    __device__ void store_load(T* p, int j, const float (&f)[V]) const {
        if (whole(j)) {
            store_pack<T, V>(p + col(j), f);
        } else if (OFF && in(j)) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (col(j) + e >= 0 && col(j) + e < D) p[col(j) + e] = from_float<T>(f[e]);
        }
    }
    // A vector over the columns, aligned at column 0.
    __device__ void load_vector(float2 (&v)[PAIRS], const float* p) const {
        if constexpr (!OFF) {
            Pack<float, V> raw[CH];
            load<float>(raw, p, true);
            pairs<float>(raw, v);
        } else {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int c = col(2 * i / V) + 2 * i % V;
                v[i].x = !idle && in_pair(i, 0) ? p[c] : 0.0f;
                v[i].y = !idle && in_pair(i, 1) ? p[c + 1] : 0.0f;
            }
        }
    }
    __device__ void store_vector(float* p, const float2 (&v)[PAIRS]) const {
        if constexpr (!OFF) {
            store<float>(p, v, true);
        } else if (!idle) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int c = col(2 * i / V) + 2 * i % V;
                if (in_pair(i, 0)) p[c] = v[i].x;
                if (in_pair(i, 1)) p[c + 1] = v[i].y;
            }
        }
    }
    // A parameter vector, `none` where it is absent.
    __device__ void param(float2 (&v)[PAIRS], const float* p, float none) const {
        if (p) load_vector(v, p);
        else
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) v[i] = make_float2(none, none);
    }
};

// A row from the ring or from memory.
template <bool RING, bool OFF, typename T, typename C, int V, int CH>
__device__ __forceinline__ void take_row(Pack<T, V> (&raw)[CH], const C& cols, const TileSource<T>& src,
                                         const uint8_t* slot, int64_t base, int group, bool live) {
    const T* row = src.p + (base + group) * src.ld;
    if constexpr (!RING) {
        cols.load(raw, row, live);
    } else {
        const int at = (V == 1 || OFF ? src.shift(base) : 0) + group * src.D;
        const T* image = reinterpret_cast<const T*>(slot) + at;
        if constexpr (OFF) {
            cols.load_off(raw, image, row, src.copied(base) - at, live);
        } else {
            cols.load(raw, image, live);
            if constexpr (V == 1) {
                const int most = src.copied(base) - at;
                if (most < src.D && live && !cols.idle)
#pragma unroll
                    for (int j = 0; j < CH; ++j)
                        if (cols.col(j) >= most && cols.in(j)) raw[j].v[0] = row[cols.col(j)];
            }
        }
    }
}

template <typename TX, typename TY, int V, int CH, bool RING, bool TAIL1, bool OFF>
__global__ void __launch_bounds__(512)
layer_norm_kernel(const TileSource<TX> x, const float* __restrict__ w, const float* __restrict__ b,
                  float eps, TY* y, int64_t ldy, float* mean, float* rstd, int tpr, int stages,
                  unsigned* err) {
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float red[LN_RED][1];
    __shared__ uint64_t full[LN_RING];
    using Cols = Columns<V, CH, TAIL1, OFF>;
    constexpr int PAIRS = Cols::PAIRS;
    int phase = 0;
    cudaGridDependencySynchronize();
    const int D = x.D, rpb = x.rpb, group = rpb == 1 ? 0 : threadIdx.x / tpr;
    const Cols cols(threadIdx.x - group * tpr, tpr, D, (int64_t)blockIdx.x * rpb + group);
    const int width = rpb == 1 ? blockDim.x : tpr;  // threads that sum a row
    const int64_t rows = x.rows, step = (int64_t)gridDim.x * rpb;
    int64_t base = (int64_t)blockIdx.x * rpb;
    auto fill = [&](int slot, int64_t row) {
        mbar_expect_tx(&full[slot], x.issue(nullptr, row, nullptr, false));
        x.issue(ring + (size_t)slot * x.bytes, row, &full[slot], true);
    };
    if constexpr (RING) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            for (int i = 0; i < stages && base + i * step < rows; ++i) fill(i, base + i * step);
        }
        __syncthreads();
    }
    float2 wr[PAIRS], br[PAIRS];
    cols.param(wr, w, 1.0f);
    cols.param(br, b, 0.0f);
    const float per = 1.0f / (float)D;
    bool ok = true;
    for (int slot = 0, turn = 0; base < rows; base += step) {
        const int64_t r = base + group;
        Pack<TX, V> raw[CH];
        if constexpr (RING) ok = ok && mbar_wait(&full[slot], turn, err);
        take_row<RING, OFF>(raw, cols, x, ring + (size_t)slot * x.bytes, base, group, r < rows);
        float2 q0 = make_float2(0.0f, 0.0f), q1 = q0;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) (i % 2 ? q1 : q0) = add2(i % 2 ? q1 : q0, Cols::pair(raw, i));
        float s[1] = {(q0.x + q0.y) + (q1.x + q1.y)};
        row_sum<1>(s, width, red, phase);
        if constexpr (RING) {
            if (width <= 32) __syncthreads();  // else row_sum's barrier: every thread has its part of the tile
            if (threadIdx.x == 0 && ok && base + stages * step < rows) fill(slot, base + stages * step);
            if (++slot == stages) slot = 0, turn ^= 1;
        }
        const float m = s[0] / (float)D;
        const float2 neg = make_float2(-m, -m);
        q0 = q1 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            float2 d = add2(Cols::pair(raw, i), neg);
            if (!cols.in_pair(i, 0)) d.x = 0.0f;
            if (!cols.in_pair(i, 1)) d.y = 0.0f;
            (i % 2 ? q1 : q0) = fma2(d, d, i % 2 ? q1 : q0);
        }
        s[0] = cols.idle ? 0.0f : (q0.x + q0.y) + (q1.x + q1.y);
        row_sum<1>(s, width, red, phase);
        const float rs = rsqrtf(s[0] * per + eps);
        const float2 scale = make_float2(rs, rs);
        if (r < rows && !cols.idle)
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                if (!cols.in(j)) continue;
                float o[V];
                Cols::affine(o, raw, j, neg, scale, wr, br);
                cols.template store_load<TY>(y + r * ldy, j, o);
            }
        if (cols.tid == 0 && r < rows) {
            if (mean) mean[r] = m;
            if (rstd) rstd[r] = rs;
        }
    }
    if constexpr (RING)
        if (!ok) drain(full, stages, err);
}

// dx, and one partial of dw and db per CTA at part[0 | 1][CTA][column]. SM: the sums over rows are
// kept in shared memory instead of registers, and the weight is read from memory.
template <typename TX, typename TY, int V, int CH, bool RING, bool SM, bool TAIL1>
__global__ void __launch_bounds__(512)
layer_norm_grad_kernel(const TileSource<TY> dy, const TileSource<TX> x, const float* __restrict__ w,
                       const float* __restrict__ mean, const float* __restrict__ rstd, TY* dx,
                       int64_t lddx, float* __restrict__ part, int tpr, int stages, unsigned* err) {
    extern __shared__ __align__(16) uint8_t ring[];  // ring or SM's sums; at the end the CTA's sums
    __shared__ float red[LN_RED][2];                 // [2][rpb][D] in the ring's place
    __shared__ uint64_t full[LN_RING];
    using Cols = Columns<V, CH, TAIL1, false>;
    constexpr int PAIRS = Cols::PAIRS, HELD = SM ? 1 : PAIRS;
    int phase = 0;
    cudaGridDependencySynchronize();
    const int D = x.D, rpb = x.rpb, group = rpb == 1 ? 0 : threadIdx.x / tpr;
    const Cols cols(threadIdx.x - group * tpr, tpr, D, 0);
    const int width = rpb == 1 ? blockDim.x : tpr;
    const int64_t rows = x.rows, step = (int64_t)gridDim.x * rpb;
    int64_t base = (int64_t)blockIdx.x * rpb;
    const uint32_t slot_bytes = x.bytes + dy.bytes;
    float* sums = reinterpret_cast<float*>(ring);
    auto fill = [&](int slot, int64_t row) {
        mbar_expect_tx(&full[slot], x.issue(nullptr, row, nullptr, false) + dy.issue(nullptr, row, nullptr, false));
        uint8_t* at = ring + (size_t)slot * slot_bytes;
        x.issue(at, row, &full[slot], true);
        dy.issue(at + x.bytes, row, &full[slot], true);
    };
    if constexpr (RING) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            for (int i = 0; i < stages && base + i * step < rows; ++i) fill(i, base + i * step);
        }
        __syncthreads();
    }
    float2 wr[PAIRS], aw[HELD], ab[HELD];
    if constexpr (!SM) cols.param(wr, w, 1.0f);
#pragma unroll
    for (int i = 0; i < HELD; ++i) aw[i] = ab[i] = make_float2(0.0f, 0.0f);
    if constexpr (SM) {  // every thread touches its own columns only
        const float2 zero[PAIRS] = {};
        cols.store_vector(sums, zero);
        cols.store_vector(sums + D, zero);
    }
    const float per = 1.0f / (float)D;
    bool ok = true;
    float m = 0.0f, rs = 0.0f;
    if (base + group < rows) m = mean[base + group], rs = rstd[base + group];
    for (int slot = 0, turn = 0; base < rows; base += step) {
        const int64_t r = base + group;
        Pack<TX, V> rx[CH];
        Pack<TY, V> rg[CH];
        const uint8_t* at = ring + (size_t)slot * slot_bytes;
        if constexpr (RING) ok = ok && mbar_wait(&full[slot], turn, err);
        take_row<RING, false>(rx, cols, x, at, base, group, r < rows);
        take_row<RING, false>(rg, cols, dy, at + x.bytes, base, group, r < rows);
        float next_m = 0.0f, next_rs = 0.0f;
        if (r + step < rows) next_m = mean[r + step], next_rs = rstd[r + step];
        const float2 neg = make_float2(-m, -m), scale = make_float2(rs, rs);
        float2 xh[PAIRS], g[PAIRS], s0 = make_float2(0.0f, 0.0f), s1 = s0;
        Cols::pairs(rx, xh);
        Cols::pairs(rg, g);
        if constexpr (SM) cols.param(wr, w, 1.0f);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {  // dy = 0 past the row's end, so nothing is added there
            xh[i] = mul2(add2(xh[i], neg), scale);
            const float2 t = mul2(g[i], wr[i]);
            s0 = add2(s0, t);
            s1 = fma2(t, xh[i], s1);
            if constexpr (!SM) {
                aw[i] = fma2(g[i], xh[i], aw[i]);
                ab[i] = add2(ab[i], g[i]);
            }
        }
        if constexpr (SM) {
            float2 q[PAIRS];
            cols.load_vector(q, sums);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) q[i] = fma2(g[i], xh[i], q[i]);
            cols.store_vector(sums, q);
            cols.load_vector(q, sums + D);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) q[i] = add2(g[i], q[i]);
            cols.store_vector(sums + D, q);
        }
        float s[2] = {s0.x + s0.y, s1.x + s1.y};
        row_sum<2>(s, width, red, phase);
        if constexpr (RING) {
            if (width <= 32) __syncthreads();  // else row_sum's barrier: every thread has its part of the tile
            if (threadIdx.x == 0 && ok && base + stages * step < rows) fill(slot, base + stages * step);
            if (++slot == stages) slot = 0, turn ^= 1;
        }
        if (dx) {
            const float c1 = -rs * (s[0] * per), c2 = -rs * (s[1] * per);
            if constexpr (SM) cols.param(wr, w, 1.0f);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i)
                g[i] = fma2(xh[i], make_float2(c2, c2), fma2(mul2(g[i], wr[i]), scale, make_float2(c1, c1)));
            cols.store(dx + r * lddx, g, r < rows);
        }
        m = next_m;
        rs = next_rs;
    }
    if constexpr (RING)
        if (!ok) drain(full, stages, err);
    if (!part) return;
    float* pw = part + (int64_t)blockIdx.x * D;
    float* pb = pw + (int64_t)gridDim.x * D;
    if constexpr (SM) {
        float2 q[PAIRS];
        cols.load_vector(q, sums);
        cols.store_vector(pw, q);
        cols.load_vector(q, sums + D);
        cols.store_vector(pb, q);
    } else if (rpb == 1) {
        cols.store_vector(pw, aw);
        cols.store_vector(pb, ab);
    } else {  // add the CTA's rows: group after group, column by column
        const int n = rpb * D;
        __syncthreads();  // the ring's last tile has been read
        cols.store_vector(sums + group * D, aw);
        cols.store_vector(sums + n + group * D, ab);
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += blockDim.x) {
            float sw = 0.0f, sb = 0.0f;
            for (int q = 0; q < rpb; ++q) {
                sw += sums[q * D + c];
                sb += sums[n + q * D + c];
            }
            pw[c] = sw;
            pb[c] = sb;
        }
    }
}

// out[0 | 1][column] = sum of the partials in a fixed order: 32 columns (16 bytes a lane, or with an odd D
// one element), 32 strided slices of the CTAs.
template <bool VEC>
__global__ void __launch_bounds__(VEC ? 256 : 1024)
layer_norm_join_kernel(const float* __restrict__ part, int parts, int D, float* dw, float* db) {
    constexpr int V = VEC ? 4 : 1, LANES = 32 / V;
    __shared__ float red[32][33];
    const int lane = threadIdx.x % LANES, slice = threadIdx.x / LANES;
    const int c = blockIdx.x * 32 + lane * V;
    float s[V] = {};
    cudaGridDependencySynchronize();
    if (c < D) {
        const float* src = part + (int64_t)blockIdx.y * parts * D + c;
#pragma unroll 4
        for (int i = slice; i < parts; i += 32) {
            float v[V];
            load_pack<float, V>(src + (int64_t)i * D, v);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red[slice][lane * V + e] = s[e];
    __syncthreads();
    const int col = blockIdx.x * 32 + threadIdx.x;
    if (threadIdx.x < 32 && col < D) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += red[i][threadIdx.x];
        float* out = blockIdx.y == 0 ? dw : db;
        if (out) out[col] = t;
    }
}

// ---- rows above LN_MAX_D elements: a CTA per row, read again for each pass -------------------------
constexpr int LN_WIDE = 512;

template <typename TX, typename TY>
__global__ void __launch_bounds__(LN_WIDE)
layer_norm_wide_kernel(int64_t rows, int64_t D, const TX* x, int64_t ldx, const float* w,
                       const float* b, float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    __shared__ float red[LN_RED][1];
    int phase = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const TX* xr = x + r * ldx;
        float s[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < D; c += LN_WIDE) s[0] += to_float(xr[c]);
        row_sum<1>(s, LN_WIDE, red, phase);
        const float m = s[0] / (float)D;
        s[0] = 0.0f;
        for (int64_t c = threadIdx.x; c < D; c += LN_WIDE) {
            const float d = to_float(xr[c]) - m;
            s[0] += d * d;
        }
        row_sum<1>(s, LN_WIDE, red, phase);
        const float rs = 1.0f / sqrtf(s[0] / (float)D + eps);
        for (int64_t c = threadIdx.x; c < D; c += LN_WIDE) {
            const float xh = (to_float(xr[c]) - m) * rs;
            y[r * ldy + c] = from_float<TY>(xh * (w ? w[c] : 1.0f) + (b ? b[c] : 0.0f));
        }
        if (threadIdx.x == 0) {
            if (mean) mean[r] = m;
            if (rstd) rstd[r] = rs;
        }
    }
}

// dx may be dy: the two statistics of a row are complete (row_sum's barrier) before it is written, and
// the weights' gradients are taken by a kernel of their own, launched before this one.
template <typename TX, typename TY>
__global__ void __launch_bounds__(LN_WIDE)
layer_norm_wide_dx_kernel(int64_t rows, int64_t D, const TY* dy, int64_t lddy, const TX* x,
                          int64_t ldx, const float* w, const float* mean, const float* rstd,
                          TY* dx, int64_t lddx) {
    __shared__ float red[LN_RED][2];
    int phase = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float m = mean[r], rs = rstd[r];
        float s[2] = {0.0f, 0.0f};
        for (int64_t c = threadIdx.x; c < D; c += LN_WIDE) {
            const float t = to_float(dy[r * lddy + c]) * (w ? w[c] : 1.0f);
            s[0] += t;
            s[1] += t * ((to_float(x[r * ldx + c]) - m) * rs);
        }
        row_sum<2>(s, LN_WIDE, red, phase);
        const float c1 = s[0] / (float)D, c2 = s[1] / (float)D;
        for (int64_t c = threadIdx.x; c < D; c += LN_WIDE) {
            const float t = to_float(dy[r * lddy + c]) * (w ? w[c] : 1.0f);
            const float xh = (to_float(x[r * ldx + c]) - m) * rs;
            dx[r * lddx + c] = from_float<TY>(rs * (t - c1 - xh * c2));
        }
    }
}

// 32 columns a CTA, 16 strided slices of the rows.
template <typename TX, typename TY>
__global__ void __launch_bounds__(LN_WIDE)
layer_norm_wide_dw_kernel(int64_t rows, int64_t D, const TY* dy, int64_t lddy, const TX* x,
                          int64_t ldx, const float* mean, const float* rstd, float* dw, float* db) {
    __shared__ float red[2][LN_WIDE / 32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float sw = 0.0f, sb = 0.0f;
    if (c < D)
        for (int64_t r = slice; r < rows; r += LN_WIDE / 32) {
            const float g = to_float(dy[r * lddy + c]);
            sw += g * ((to_float(x[r * ldx + c]) - mean[r]) * rstd[r]);
            sb += g;
        }
    red[0][slice][lane] = sw;
    red[1][slice][lane] = sb;
    __syncthreads();
    if (slice < 2 && c < D) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < LN_WIDE / 32; ++i) t += red[slice][i][lane];
        float* out = slice == 0 ? dw : db;
        if (out) out[c] = t;
    }
}

// ---- host -----------------------------------------------------------------------------------------
int pow2_ceil(int64_t v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

// How the rows of an operand are taken: through the ring in aligned loads; the same with rows that start
// anywhere (one run of memory); through the ring by element; without the ring by element.
enum class Access { Wide, Offset, Element, Direct };
template <typename T>
Access access_of(const T* p, int64_t ld, int64_t rows, int64_t D) {
    constexpr int per = 16 / sizeof(T);
    if (!aligned_to(p, 16)) return Access::Direct;
    if (D % per == 0 && (ld % per == 0 || rows == 1)) return Access::Wide;
    return ld == D || rows == 1 ? Access::Offset : Access::Direct;
}
inline Access worst(Access a, Access b) { return a > b ? a : b; }

// Threads per row for E elements a thread, and the CTA size. Within a warp a power of two, else as
// many as there are columns for (the CTA's last ones idle): then only the last load can pass the row.
void row_threads(int64_t D, int E, int V, bool off, int* tpr, int* block) {
    const int64_t n = ceil_div(ceil_div(off ? D + V - 1 : D, V), E / V);
    *tpr = n <= 32 ? pow2_ceil(n) : (int)n;
    *block = *tpr <= 32 ? LN_SMALL_BLOCK : (int)ceil_div(n, 32) * 32;
}

template <typename T>
TileSource<T> tile_source(const T* p, int64_t ld, int64_t rows, int64_t D, int rpb) {
    TileSource<T> s;
    s.p = p;
    s.ld = ld;
    s.D = (int)D;
    s.rpb = rpb;
    s.rows = rows;
    s.dense = ld == D || rows == 1;
    s.bytes = (uint32_t)((rpb * D * sizeof(T) + 47) / 16 * 16);  // 16-byte pieces at both ends
    return s;
}

// Tiles in flight: about 32 KB a CTA, two at least.
int ring_stages(uint32_t tile_bytes) {
    return (int)std::max<uint32_t>(2, std::min<uint32_t>(LN_RING, 32768 / tile_bytes));
}

// Grid of a persistent kernel: a CTA per tile while they fit the GPU at once, else a multiple of `multiple`
// CTAs (which keeps the offset of the rows a CTA takes).
template <typename K>
unsigned tile_grid(Handle& h, K kern, int block, size_t smem, int64_t tiles, int multiple) {
    const int sms = sm_count(h.device);
    // a launch may take 48 KB unasked, the kernel's static shared memory (below 2 KB here) among them
    if (smem > 46 * 1024) allow_smem(kern);
    if (tiles <= sms) return (unsigned)tiles;  // each has its own
    int per_sm = 0;
    XS_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, block, smem));
    const int64_t fit = (int64_t)sms * std::max(1, per_sm) / multiple * multiple;
    return (unsigned)std::min(tiles, fit);  // fewer tiles than fit: a CTA takes one
}

template <typename TX, typename TY, int V, int E, bool RING, bool OFF>
void norm_launch(Handle& h, int64_t rows, int64_t D, const TX* x, int64_t ldx, const float* w,
                 const float* b, float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    int tpr, block;
    row_threads(D, E, V, OFF, &tpr, &block);
    const TileSource<TX> src = tile_source(x, ldx, rows, D, tpr <= 32 ? block / tpr : 1);
    const int stages = ring_stages(src.bytes);
    const size_t smem = RING ? (size_t)stages * src.bytes : 0;
    const bool tail1 = ceil_div(D, V) > (int64_t)tpr * (E / V - 1);
    auto kern = tail1 ? layer_norm_kernel<TX, TY, V, E / V, RING, true, OFF>
                      : layer_norm_kernel<TX, TY, V, E / V, RING, false, OFF>;
    const unsigned grid = tile_grid(h, kern, block, smem, ceil_div(rows, src.rpb), OFF ? V : 1);
    launch_dependent(h.stream, kern, grid, block, smem, 1, src, w, b, eps, y, ldy, mean, rstd, tpr, stages,
                     h.d_err);
    after_launch(h, "layer_norm");
}

template <typename TX, typename TY, int V, int E, bool RING, bool SM>
void norm_grad_launch(Handle& h, int64_t rows, int64_t D, const TY* dy, int64_t lddy, const TX* x,
                      int64_t ldx, const float* w, const float* mean, const float* rstd, TY* dx,
                      int64_t lddx, float* dw, float* db) {
    int tpr, block;
    row_threads(D, E, V, false, &tpr, &block);
    const TileSource<TX> sx = tile_source(x, ldx, rows, D, tpr <= 32 ? block / tpr : 1);
    const TileSource<TY> sg = tile_source(dy, lddy, rows, D, tpr <= 32 ? block / tpr : 1);
    const int stages = ring_stages(sx.bytes + sg.bytes);
    const size_t ring = RING ? (size_t)stages * (sx.bytes + sg.bytes) : 0;
    const size_t smem = SM ? (size_t)D * 8 : std::max(ring, sx.rpb > 1 ? (size_t)block * E * 8 : (size_t)0);
    const bool tail1 = ceil_div(D, V) > (int64_t)tpr * (E / V - 1);
    auto kern = tail1 ? layer_norm_grad_kernel<TX, TY, V, E / V, RING, SM, true>
                      : layer_norm_grad_kernel<TX, TY, V, E / V, RING, SM, false>;
    const unsigned grid = tile_grid(h, kern, block, smem, ceil_div(rows, sx.rpb), 1);
    const bool sums = dw || db;
    DevBuf<float> part(sums ? (size_t)2 * grid * D : 0, h.stream);
    launch_dependent(h.stream, kern, grid, block, smem, 1, sg, sx, w, mean, rstd, dx, lddx, part.get(), tpr,
                     stages, h.d_err);
    after_launch(h, "layer_norm_grad");
    if (sums) {
        const bool vec = D % 4 == 0;
        launch_dependent(h.stream, vec ? layer_norm_join_kernel<true> : layer_norm_join_kernel<false>,
                         dim3((unsigned)ceil_div(D, 32), 2), vec ? 256 : 1024, 0, 1,
                         (const float*)part.get(), (int)grid, (int)D, dw, db);
        after_launch(h, "layer_norm_join");
    }
}

}  // namespace

template <typename TX, typename TY>
void layer_norm(Handle& h, int64_t rows, int64_t D, const TX* x, int64_t ldx, const float* w,
                const float* b, float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    if (rows == 0) return;
    constexpr int V = 16 / sizeof(TX);
    // 32 elements a thread halve the reductions' share of a long 16-bit row (4096 columns, 16384 rows:
    // 54 us against 69), and fit the longest rows to 512 threads. Short rows take 16: more of them are
    // in flight; there loads of 4 let a warp read the fp32 parameters in whole lines (16-bit, 128
    // columns: 99 us against 112 with loads of 8).
    const bool more = D > (sizeof(TX) == 2 ? 512 : 8192);
    const int need_v = more ? V : 4;
    Access how = access_of(x, ldx, rows, D);
    const bool dense = (ldx == D && ldy == D) || rows == 1;
    if (how == Access::Wide && !(aligned_to(y, sizeof(TY) * need_v) && (ldy % need_v == 0 || rows == 1) &&
                                 aligned_to(w, 16) && aligned_to(b, 16)))
        how = ldx == D || rows == 1 ? Access::Offset : Access::Direct;
    // Rows that start anywhere: long ones keep 16-byte loads (4821 columns, bf16: 70 us against 126 by
    // element); in short ones every warp would have edges (1021 columns, fp16: 199 against 112).
    if (how == Access::Offset && !(dense && aligned_to(y, sizeof(TY) * V) && D > 2048 && D <= LN_MAX_D - V))
        how = Access::Element;
#define XS_LN(VV, E, RING, OFF)                                                                   \
    norm_launch<TX, TY, VV, E, RING, OFF>(h, rows, D, x, ldx, w, b, eps, y, ldy, mean, rstd)
    if (D > LN_MAX_D) {
        const unsigned grid = (unsigned)std::min(rows, (int64_t)sm_count(h.device) * 4);
        layer_norm_wide_kernel<TX, TY>
            <<<grid, LN_WIDE, 0, h.stream>>>(rows, D, x, ldx, w, b, eps, y, ldy, mean, rstd);
        after_launch(h, "layer_norm_wide");
    } else if (how == Access::Wide) {
        if (more) XS_LN(V, 32, true, false);
        else XS_LN(4, 16, true, false);
    } else if (how == Access::Offset) {
        XS_LN(V, 32, true, true);
    } else if (how == Access::Element) {
        if (D > 8192) XS_LN(1, 32, true, false);
        else XS_LN(1, 16, true, false);
    } else {
        if (D > 8192) XS_LN(1, 32, false, false);
        else XS_LN(1, 16, false, false);
    }
#undef XS_LN
}

template <typename TX, typename TY>
void layer_norm_backward(Handle& h, int64_t rows, int64_t D, const TY* dy, int64_t lddy,
                         const TX* x, int64_t ldx, const float* w, const float* mean,
                         const float* rstd, TY* dx, int64_t lddx, float* dw, float* db) {
    if (rows == 0) {
        if (dw) XS_CHECK_CUDA(cudaMemsetAsync(dw, 0, D * sizeof(float), h.stream));
        if (db) XS_CHECK_CUDA(cudaMemsetAsync(db, 0, D * sizeof(float), h.stream));
        return;
    }
    constexpr int V = 16 / sizeof(TX);
    Access how = worst(access_of(x, ldx, rows, D), access_of(dy, lddy, rows, D));
    if (how == Access::Wide && !((!dx || (aligned_to(dx, sizeof(TY) * V) && (lddx % V == 0 || rows == 1))) &&
                                 aligned_to(w, 16)))
        how = (ldx == D && lddy == D) || rows == 1 ? Access::Element : Access::Direct;
    // with two inputs the offset form's edges cost more than it saves (4821 columns, bf16: 178 us against 156)
    if (how == Access::Offset) how = Access::Element;
#define XS_LN(VV, E, RING, SM)                                                                    \
    norm_grad_launch<TX, TY, VV, E, RING, SM>(h, rows, D, dy, lddy, x, ldx, w, mean, rstd, dx, lddx, \
                                              dw, db)
    if (D > LN_MAX_D) {
        if (dw || db) {
            layer_norm_wide_dw_kernel<TX, TY><<<(unsigned)ceil_div(D, 32), LN_WIDE, 0, h.stream>>>(
                rows, D, dy, lddy, x, ldx, mean, rstd, dw, db);
            after_launch(h, "layer_norm_wide_dw");
        }
        if (dx) {
            const unsigned grid = (unsigned)std::min(rows, (int64_t)sm_count(h.device) * 4);
            layer_norm_wide_dx_kernel<TX, TY><<<grid, LN_WIDE, 0, h.stream>>>(
                rows, D, dy, lddy, x, ldx, w, mean, rstd, dx, lddx);
            after_launch(h, "layer_norm_wide_dx");
        }
    } else if (D > LN_MAX_ACC) {  // the sums take the shared memory that a ring would need
        if (how == Access::Wide) XS_LN(4, 32, false, true);
        else XS_LN(1, 32, false, true);
    } else if (how == Access::Wide) {
        XS_LN(V, 16, true, false);
    } else if (how == Access::Element) {
        XS_LN(1, 16, true, false);
    } else {
        XS_LN(1, 16, false, false);
    }
#undef XS_LN
}

#define XS_INST_LN(TX, TY)                                                                        \
    template void layer_norm<TX, TY>(Handle&, int64_t, int64_t, const TX*, int64_t, const float*, \
                                     const float*, float, TY*, int64_t, float*, float*);          \
    template void layer_norm_backward<TX, TY>(Handle&, int64_t, int64_t, const TY*, int64_t,      \
                                              const TX*, int64_t, const float*, const float*,     \
                                              const float*, TY*, int64_t, float*, float*);
XS_INST_LN(__half, __half)
XS_INST_LN(__nv_bfloat16, __nv_bfloat16)
XS_INST_LN(float, float)
XS_INST_LN(float, __half)
XS_INST_LN(float, __nv_bfloat16)

}  // namespace xspmm_b200
