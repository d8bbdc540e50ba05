// orthogonalize.cu -- the orthogonalised update of a weight matrix by Newton-Schulz steps.
//
// X = g / (|g| + eps), then `steps` times X <- B' X, B' = a I + b A + c A A, A = X X^T, taken on the smaller side:
// for more rows than columns X <- X B' with A = X^T X. The coefficients (a, b, c) = (3.4445, -4.7750, 2.0315) were
// published by K. Jordan and others in 2024 with this use of the iteration. The polynomial p(s) = a s + b s^3 + c s^5 acts on the
// singular values, which start in [0, 1]; it is at most 1.2025 there (at s = 0.5545) and maps [0, 1.2025] into
// itself, so every entry of X stays below 1.21, of A below 1.45 and of B' (eigenvalues in [0.63, 3.4445]) below 3.45.
//
// Precision. A step multiplies small singular values by 3.4445, 485 in five steps, and what rounding X to 16 bits
// would add to those directions with them. X, A and B' are therefore held as two fp16 parts (22 bits), and the
// products are those of the parts with fp32 sums, joined from runs of at most 128 terms (tile_product.cuh): the error
// before y's rounding is about that of the steps in fp32. A and B' are symmetric: half of their tiles are computed. The
// norm is summed in fp64: squares of any fp32 gradient are in its range. A gradient far below eps makes an X_0 far below
// 1, of which 2^14 times would lose bits of the parts, or all: step i holds 2^(14 + e_i) X_i, e_i from the bound
// a^i |X_0| on its entries, 0 as soon as that passes 1/2. An X_0 of norm 2^-100 still has all its bits.
//
// 11008 x 4096: 7.8 to 8.1 ms; the three products of the parts' 3.1 TFLOP are 6.73 ms at the sustained bf16 rate. Below about 1000
// the launches and latencies of fifteen products (768 x 1232: 228 us).
#include "tile_product.cuh"

namespace xspmm_b200 {
namespace {

using namespace product;

// A matrix is walked in pieces of PIECE columns of a row, one a warp, V elements a lane at a time: f(row, first column).
constexpr int PIECE = 1024;
template <int V, typename F>
__device__ __forceinline__ void each_piece(int64_t rows, int64_t cols, F&& f) {
    const int64_t per = (cols + PIECE - 1) / PIECE, warps = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < rows * per; i += warps) {
        const int64_t r = i / per, c0 = (i - r * per) * PIECE, end = min(cols, c0 + PIECE);
#pragma unroll 4
        for (int64_t c = c0 + (threadIdx.x & 31) * V; c < end; c += 32 * V) f(r, c);
    }
}

// Sum of squares in fp64: one partial per CTA, added in a fixed order by the next kernel.
template <typename T, int V>
__global__ void __launch_bounds__(256) squares_kernel(int64_t rows, int64_t cols, const T* g, int64_t ldg, double* part) {
    __shared__ double red[8];
    cudaGridDependencySynchronize();
    double s = 0.0;
    each_piece<V>(rows, cols, [&](int64_t r, int64_t c) {
        float v[V];
        load_pack<T, V>(g + r * ldg + c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s += (double)v[e] * (double)v[e];
    });
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) s += red[i];
        part[blockIdx.x] = s;
    }
}

// The norm and 1 / (norm + eps), from the partial sums; the same in all threads of the CTA and in all CTAs.
__device__ __forceinline__ double2 norm_of(const double* part, int parts, float eps) {
    __shared__ double norm;
    if (threadIdx.x < 32) {
        double s = 0.0;
        for (int i = threadIdx.x; i < parts; i += 32) s += part[i];
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x == 0) norm = sqrt(s);
    }
    __syncthreads();
    return make_double2(norm, 1.0 / (norm + (double)eps));
}

// e_i from a^i |X_0|, and the bound of the next step.
__device__ __forceinline__ int exponent(double* bound) {
    int x;
    frexp(*bound, &x);  // below 2^x; 0 and what is not finite: no matter
    *bound *= (double)NS_A;
    return max(0, min(100, -x));
}

// X_0 in two parts; the padding of its rows becomes zeros. mul[i]: what step i's A and its X or y are multiplied by.
template <typename T, int V>
__global__ void __launch_bounds__(256)
start_kernel(int64_t rows, int64_t cols, const T* g, int64_t ldg, const double* part, int parts, float eps, __half* hi,
             __half* lo, int64_t ld, int steps, float2* mul) {
    cudaGridDependencySynchronize();
    const double2 norm = norm_of(part, parts, eps);
    double bound = norm.x * norm.y;
    int at = exponent(&bound);
    const double inv = norm.y * (double)(ldexpf(SPLIT_SCALE, at));
    if (blockIdx.x == 0 && threadIdx.x == 0)
        for (int i = 0; i < steps; ++i) {
            const int next = i + 1 < steps ? exponent(&bound) : 0;
            mul[i] = make_float2(ldexpf(1.0f, -2 * at), ldexpf(1.0f, next - at));
            at = next;
        }
    each_piece<4>(rows, ld, [&](int64_t r, int64_t c) {
        float v[4] = {};
        const T* from = g + r * ldg + c;
        if constexpr (V == 4) {
            if (c < cols) load_pack<T, 4>(from, v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < cols) v[e] = to_float(from[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)(v[e] * inv);
        uint2 h, l;
        split2(v[0], v[1], &h.x, &l.x);
        split2(v[2], v[3], &h.y, &l.y);
        *reinterpret_cast<uint2*>(hi + r * ld + c) = h;
        *reinterpret_cast<uint2*>(lo + r * ld + c) = l;
    });
}

// y = X_0: no steps.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256)
scaled_kernel(int64_t rows, int64_t cols, const TX* g, int64_t ldg, const double* part, int parts, float eps, TY* y,
              int64_t ldy) {
    cudaGridDependencySynchronize();
    const double inv = norm_of(part, parts, eps).y;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
        y[i / cols * ldy + i % cols] = from_float<TY>((float)(to_float(g[i / cols * ldg + i % cols]) * inv));
}

// ---- small matrices: all steps in one CTA -----------------------------------------------------------
// A side of at most 128 and another of at most 256: X (as a matrix of at most 128 rows, transposed if need be) and A
// stay in shared memory in two parts, in the SWIZZLE_128B layout: 64-column chunks of 128 rows of 128 bytes. Read along
// its rows a chunk is a K-major operand, along its columns an MN-major one, so X serves both products. A is replaced by
// B' in place and X by its successor, each after the MMAs that read it. Bound by the latency of 3 products a step, their
// MMAs on 1 of 148 SMs and the epilogues between (128 x 128, 5 steps: 64 us, on the large path 111; 100 x 200 75 and 121;
// 128 x 256, the largest that fits, 107 and 121).
constexpr int SMALL_THREADS = 512, SMALL_ROWS = 128, SMALL_COLS = 256;
constexpr int SMALL_CHUNK = SMALL_ROWS * 128;

__device__ __forceinline__ uint64_t small_desc_mn(uint32_t saddr) {  // 64-column chunks SMALL_CHUNK apart
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(SMALL_CHUNK >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Where 8 elements of row r from column c (a multiple of 8) on are.
__device__ __forceinline__ int small_at(int r, int c) {
    return (c >> 6) * SMALL_CHUNK + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4);
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(SMALL_THREADS, 1)
small_update_kernel(int rows, int cols, const TX* g, int64_t ldg, int steps, float eps, TY* y, int64_t ldy,
                    uint32_t square, uint32_t wide, unsigned* err) {  // descriptors: 128 x 128, 128 x X's columns
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ double red[SMALL_THREADS / 32];
    __shared__ uint64_t done;
    __shared__ uint32_t tmem_slot;
    const bool turned = rows > cols;
    const int m = min(rows, cols), n = max(rows, cols), chunks = (n + 63) / 64;
    uint8_t *xh = smem, *xl = xh + chunks * SMALL_CHUNK, *ah = xl + chunks * SMALL_CHUNK, *al = ah + 2 * SMALL_CHUNK;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc_all<1>(&tmem_slot);
    cudaGridDependencySynchronize();
    double s = 0.0;
    for (int i = threadIdx.x; i < rows * cols; i += SMALL_THREADS) {
        const int r = i / cols;
        const double v = to_float(g[r * ldg + i - r * cols]);
        s += v * v;
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int i = 0; i < SMALL_THREADS / 32; ++i) s += red[i];
    double bound = sqrt(s);
    double inv = 1.0 / (bound + (double)eps);
    bound *= inv;
    int at = exponent(&bound);
    inv *= (double)ldexpf(SPLIT_SCALE, at);
    for (int i = threadIdx.x; i < SMALL_ROWS * chunks * 32; i += SMALL_THREADS) {  // two columns of X, zeros outside
        const int r = i % SMALL_ROWS, c = i / SMALL_ROWS * 2;  // neighbouring threads: rows of X
        float v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const bool in = r < m && c + e < n;
            const int64_t from = turned ? (c + e) * ldg + r : r * ldg + c + e;
            v[e] = in ? (float)(to_float(g[from]) * inv) : 0.0f;
        }
        uint32_t hi, lo;
        split2(v[0], v[1], &hi, &lo);
        const int place = small_at(r, c & ~7) + (c & 7) * 2;
        *reinterpret_cast<uint32_t*>(xh + place) = hi;
        *reinterpret_cast<uint32_t*>(xl + place) = lo;
    }
    int phase = 0;
    uint32_t tmem = 0;
    // What was written to shared memory and read from TMEM before is done; `issue` runs in one thread, and its MMAs have
    // finished on return.
    auto products = [&](auto&& issue) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        tmem = tmem_slot;
        if (threadIdx.x == 0) {
            issue();
            tc_commit(&done);
        }
        mbar_wait(&done, phase, err);
        phase ^= 1;
        __syncwarp();
        tc_fence_after();
    };
    // The k-th MMAs of a sum. With up to 128 columns its second half goes to an accumulator of its own: an addition in the
    // tensor core truncates (tile_product.cuh).
    auto three = [&](uint64_t da, uint64_t la, uint64_t db, uint64_t lb, uint32_t idesc, int k, int half) {
        tc_mma(tmem + (k < half ? 0 : SMALL_ROWS), da, db, idesc, k != 0 && k != half);
        tc_mma(tmem + ACC_COLS, da, lb, idesc, k > 0);
        tc_mma(tmem + ACC_COLS, la, db, idesc, 1);
    };
    // f(row, first column, sums of MMAs' results) for 32 columns at a time of the accumulators' `width`: four warps a
    // quarter of the rows
    auto results = [&](int width, bool two, auto&& f) {
        for (int c = (warp >> 2) * 32; c < width; c += SMALL_THREADS / 128 * 32) {
            uint32_t v[32], u[32];
            const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c;
            tmem_ld32(at, v);
            tmem_ld32(at + ACC_COLS, u);
            tmem_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(u[e]));
            if (two) {
                tmem_ld32(at + SMALL_ROWS, u);
                tmem_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(u[e]));
            }
            f((warp & 3) * 32 + lane, c, v);
        }
    };
    auto put = [&](uint8_t* hi, uint8_t* lo, int r, int c, const float (&v)[8]) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split2(v[2 * e], v[2 * e + 1], &h[e], &l[e]);
        *reinterpret_cast<uint4*>(hi + small_at(r, c)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(lo + small_at(r, c)) = make_uint4(l[0], l[1], l[2], l[3]);
    };
    const int km = (m + 15) / 16, kn = (n + 15) / 16;  // MMAs that a sum over rows, or columns, of X takes
    auto along = [](const uint8_t* p, int k) { return desc_k(smem_u32(p) + (k >> 2) * SMALL_CHUNK) + (k & 3) * 2; };
    auto down = [](const uint8_t* p, int k) { return small_desc_mn(smem_u32(p)) + k * 128; };
    for (int i = 0; i < steps; ++i) {
        const int next = i + 1 < steps ? exponent(&bound) : 0;
        const float square_mul = ldexpf(1.0f, -2 * at), mul = ldexpf(1.0f, next - at);
        at = next;
        products([&] {  // A = X X^T
            for (int k = 0; k < kn; ++k) three(along(xh, k), along(xl, k), along(xh, k), along(xl, k), square, k, (kn + 1) / 2);
        });
        results(SMALL_ROWS, kn > 1, [&](int r, int c, const uint32_t (&v)[32]) {
#pragma unroll
            for (int b = 0; b < 32; b += 8) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = finish<Epi::Gram>(__uint_as_float(v[b + e]), 0.0f, false, square_mul);
                put(ah, al, r, c + b, t);
            }
        });
        products([&] {  // A A
            for (int k = 0; k < km; ++k) three(along(ah, k), along(al, k), along(ah, k), along(al, k), square, k, (km + 1) / 2);
        });
        results(SMALL_ROWS, km > 1, [&](int r, int c, const uint32_t (&v)[32]) {
#pragma unroll
            for (int b = 0; b < 32; b += 8) {
                const uint4 h = *reinterpret_cast<const uint4*>(ah + small_at(r, c + b));
                const uint4 l = *reinterpret_cast<const uint4*>(al + small_at(r, c + b));
                const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float2 fh = unpack2(hw[e / 2], __half()), fl = unpack2(lw[e / 2], __half());
                    t[e] = finish<Epi::Poly>(__uint_as_float(v[b + e]), fh.x + fl.x, r == c + b + e, 1.0f);
                    t[e + 1] = finish<Epi::Poly>(__uint_as_float(v[b + e + 1]), fh.y + fl.y, r == c + b + e + 1, 1.0f);
                }
                put(ah, al, r, c + b, t);
            }
        });
        products([&] {  // B' X
            const int half = chunks > 2 ? km : (km + 1) / 2;
            for (int k = 0; k < km; ++k) three(along(ah, k), along(al, k), down(xh, k), down(xl, k), wide, k, half);
        });
        results(chunks * 64, km > 1 && chunks <= 2, [&](int r, int c, const uint32_t (&v)[32]) {
            if (i + 1 < steps) {
#pragma unroll
                for (int b = 0; b < 32; b += 8) {
                    float t[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[e] = finish<Epi::Next>(__uint_as_float(v[b + e]), 0.0f, false, mul);
                    put(xh, xl, r, c + b, t);
                }
            } else if (r < m) {
                TY* to = turned ? y + c * ldy + r : y + r * ldy + c;
                const int64_t next = turned ? ldy : 1;
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (c + e < n) to[e * next] = from_float<TY>(finish<Epi::Last>(__uint_as_float(v[e]), 0.0f, false, mul));
            }
        });
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_free_all<1>(tmem_slot);
}

// A matrix in two parts, rows padded to whole 16-byte words.
struct Parts {
    __half *hi, *lo;
    int64_t rows, cols, ld;
    CUtensorMap map(int part, int box_rows) const {
        return make_map_2d(part ? lo : hi, (uint64_t)cols, (uint64_t)rows, (uint64_t)ld * 2, 64, (uint32_t)box_rows,
                           CU_TENSOR_MAP_SWIZZLE_128B);
    }
};

// out = the product of P and Q (P Q^T, with AMN P^T, with BMN Q) finished by E; y instead of `out` for Last.
template <Epi E, typename T, int CG, bool AMN, bool BMN>
void multiply(Handle& h, int64_t M, int64_t N, int64_t K, const Parts& P, const Parts& Q, const float* mul, const Parts* out,
              const Parts* A, T* y, int64_t ldy) {
    Args t = {};
    t.mul = mul;
    t.M = M;
    t.N = out ? out->ld : N;
    t.ksteps = (int)ceil_div(K, 64);
    t.cols_first = M > N;
    choose<E, CG>(h, t);
    for (int i = 0; i < 2; ++i) {
        t.a[i] = P.map(i, AMN ? 64 : TM);
        t.b[i] = Q.map(i, BMN ? 64 : t.acc_n / CG);
    }
    if constexpr (E == Epi::Poly) t.ah = A->hi, t.al = A->lo, t.lda = A->ld;
    if constexpr (E == Epi::Last) {
        set_output(t, 0, y, ldy);
    } else {
        set_output(t, 0, out->hi, out->ld);
        set_output(t, 1, out->lo, out->ld);
    }
    launch<E, T, CG, AMN, BMN>(h, t);
}
template <Epi E, typename T, bool AMN, bool BMN>
void multiply(Handle& h, int64_t M, int64_t N, int64_t K, const Parts& P, const Parts& Q, const float* mul, const Parts* out,
              const Parts* A = nullptr, T* y = nullptr, int64_t ldy = 0) {
    if (M > TM) multiply<E, T, 2, AMN, BMN>(h, M, N, K, P, Q, mul, out, A, y, ldy);
    else multiply<E, T, 1, AMN, BMN>(h, M, N, K, P, Q, mul, out, A, y, ldy);
}

}  // namespace

template <typename TX, typename TY>
void orthogonalize(Handle& h, int64_t rows, int64_t cols, const TX* g, int64_t ldg, int steps, float eps, TY* y,
                   int64_t ldy) {
    if (rows == 0 || cols == 0) return;
    const int64_t limit = (int64_t(1) << 31) - 512;  // TMA coordinates are 32 bits
    XS_REQUIRE(rows < limit && cols < limit, XSPMM_STATUS_UNSUPPORTED, "a dimension of the update passes 2^31");
    if (steps > 0 && std::min(rows, cols) <= SMALL_ROWS && std::max(rows, cols) <= SMALL_COLS) {
        auto kern = small_update_kernel<TX, TY>;
        allow_smem(kern);
        const int chunks = (int)ceil_div(std::max(rows, cols), 64);
        const size_t smem = 1024 + (size_t)(2 * chunks + 4) * SMALL_CHUNK;
        launch_dependent(h.stream, kern, 1, SMALL_THREADS, smem, 1, (int)rows, (int)cols, g, ldg, steps, eps, y, ldy,
                         make_idesc(false, false, false, SMALL_ROWS, SMALL_ROWS),
                         make_idesc(false, false, true, SMALL_ROWS, chunks * 64), h.d_err);
        after_launch(h, "update_small");
        return;
    }
    const int parts = (int)std::min<int64_t>(ceil_div(rows * ceil_div(cols, PIECE), 8), 8 * sm_count(h.device));
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows * cols, 512), 8 * sm_count(h.device));
    const bool wide = cols % 4 == 0 && aligned_to(g, 4 * sizeof(TX)) && (rows == 1 || ldg % 4 == 0);
    DevBuf<double> part((size_t)parts, h.stream);
    launch_dependent(h.stream, wide ? squares_kernel<TX, 4> : squares_kernel<TX, 1>, (unsigned)parts, 256, 0, 1, rows, cols, g,
                     ldg, part.get());
    after_launch(h, "update_squares");
    if (steps == 0) {
        launch_dependent(h.stream, scaled_kernel<TX, TY>, grid, 256, 0, 1, rows, cols, g, ldg, part.get(), parts, eps, y, ldy);
        after_launch(h, "update_scaled");
        return;
    }
    const bool tall = rows > cols;
    const int64_t m = std::min(rows, cols), ldx = ceil_div(cols, 8) * 8, lda = ceil_div(m, 8) * 8;
    DevBuf<float2> muls((size_t)steps, h.stream);
    DevBuf<__half> buf((size_t)(4 * rows * ldx + 4 * m * lda), h.stream);
    __half* at = buf.get();
    auto take = [&](int64_t r, int64_t c, int64_t ld) {
        const Parts p{at, at + r * ld, r, c, ld};
        at += 2 * r * ld;
        return p;
    };
    Parts X = take(rows, cols, ldx), next = take(rows, cols, ldx), A = take(m, m, lda), B = take(m, m, lda);
    launch_dependent(h.stream, wide ? start_kernel<TX, 4> : start_kernel<TX, 1>, (unsigned)parts, 256, 0, 1, rows, cols, g, ldg,
                     part.get(), parts, eps, X.hi, X.lo, ldx, steps, muls.get());
    after_launch(h, "update_start");
    for (int i = 0; i < steps; ++i) {
        const float *square = reinterpret_cast<const float*>(muls.get() + i), *mul = square + 1;
        if (tall) multiply<Epi::Gram, __half, true, true>(h, m, m, rows, X, X, square, &A);
        else multiply<Epi::Gram, __half, false, false>(h, m, m, cols, X, X, square, &A);
        multiply<Epi::Poly, __half, false, false>(h, m, m, m, A, A, nullptr, &B, &A);
        if (i + 1 == steps) {
            if (tall) multiply<Epi::Last, TY, false, false>(h, rows, m, m, X, B, mul, nullptr, nullptr, y, ldy);
            else multiply<Epi::Last, TY, false, true>(h, m, cols, m, B, X, mul, nullptr, nullptr, y, ldy);
        } else if (tall) {
            multiply<Epi::Next, __half, false, false>(h, rows, m, m, X, B, mul, &next);
        } else {
            multiply<Epi::Next, __half, false, true>(h, m, cols, m, B, X, mul, &next);
        }
        std::swap(X, next);
    }
}

#define XS_INST_UPDATE(TX, TY) \
    template void orthogonalize<TX, TY>(Handle&, int64_t, int64_t, const TX*, int64_t, int, float, TY*, int64_t);
XS_INST_UPDATE(__half, __half)
XS_INST_UPDATE(__nv_bfloat16, __nv_bfloat16)
XS_INST_UPDATE(float, __half)
XS_INST_UPDATE(float, __nv_bfloat16)

}  // namespace xspmm_b200
