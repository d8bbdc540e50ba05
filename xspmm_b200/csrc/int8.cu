// int8.cu -- rows in 8-bit integers with a scale each, and their product.
//
// Quantisation: scale = max|x| / 127, q = 127 x / max|x| rounded to the nearest whole number, ties to even, of
// the exact quotient. Product: y[r, f] = xs[r] * ws[f] * sum_k x[r, k] w[f, k] + bias[f], the sum exact in 32 bits.
//
// 2048 rows of 4096 -> 11008, to bf16: 78 us (2.4 POP/s; the library's product without scales 65), bound by the loads into
// each SM, 64 bytes a clock. One row: 9.4 us, 73 % of the copy bandwidth.
#include "tile_product.cuh"

namespace xspmm_b200 {
namespace {

constexpr int Q_THREADS = 256;  // of a CTA of several rows

// 127 v / most rounded to the nearest, ties to even, of V values. inv = 127 / most in fp32 puts the quotient p, at most
// 127.0001, within 2^-23 of itself, 1.6e-5, so only one that close to a border can be on its wrong side; such ones (one of
// 25000) are decided in 64 bits (127 v has 31 bits, (2 q + 1) most has 32). inv is infinite for the smallest subnormal
// `most`: 64 bits too. Adding 1.5 * 2^23 rounds to whole numbers and leaves them in the low bits.
__device__ __noinline__ uint32_t quantized_exactly(float v, float most) {
    return (uint32_t)(int)rint(127.0 * (double)v / (double)most);
}
template <int V>
__device__ __forceinline__ void quantized(Pack<int8_t, V>& out, const float (&v)[V], float most, float inv) {
    constexpr float WHOLE = 12582912.0f;
    bool clear = true;
    uint32_t t[V];
    auto off = [&](int e) {  // NaN where p is infinite
        const float p = v[e] * inv, w = p + WHOLE;
        t[e] = __float_as_uint(w);
        return fabsf(p - (w - WHOLE));
    };
#pragma unroll
    for (int e = 0; e < V; ++e) clear = clear && off(e) <= 0.49998f;
    if (__builtin_expect(!clear, 0))
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (!(off(e) <= 0.49998f)) t[e] = quantized_exactly(v[e], most);
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 4)  // the low bytes
            reinterpret_cast<uint32_t*>(&out)[e / 4] =
                __byte_perm(__byte_perm(t[e], t[e + 1], 0x0040), __byte_perm(t[e + 2], t[e + 3], 0x0040), 0x5410);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) out.v[e] = (int8_t)(t[e] & 0xff);
    }
}

// The largest magnitude over a row's threads: part of a warp, or the CTA. As whole numbers, magnitudes compare as the
// numbers do, infinity above all and NaN above that.
__device__ __forceinline__ uint32_t row_most(uint32_t v, int tpr) {
    __shared__ uint32_t part[32];
    if (tpr >= 32) {
        v = __reduce_max_sync(0xffffffffu, v);
    } else {
        for (int o = tpr >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    if (tpr <= 32) return v;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int i = 0; i < tpr / 32; ++i) v = max(v, part[i]);
    return v;
}

// tpr threads a row, a power of two: part of a warp, or a CTA of that many. A thread takes V consecutive elements at a
// time, HELD in registers (the loads of a row are all in flight together and x is read once; with 8 instead of 16 what a
// thread does once a row weighs more: 2^20 x 128 fp16 163 us, with 16 108); HELD = 0: longer rows, read again for the
// second pass. Bound by memory where rows start on 16 bytes (2^20 x 128 fp32: 132 to 146 us, 103 at the copy bandwidth);
// by the instructions of narrow loads and stores elsewhere.
template <typename T, int V, int HELD>
__global__ void __launch_bounds__(HELD == 16 ? Q_THREADS : 512)
quantize_kernel(int64_t rows, int cols, int tpr_log, const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                float* scale) {
    constexpr int LOADS = HELD > V ? HELD / V : 1;
    cudaGridDependencySynchronize();
    const int tpr = 1 << tpr_log, t = threadIdx.x & (tpr - 1);
    const int64_t r = (int64_t)blockIdx.x * (blockDim.x >> tpr_log) + (threadIdx.x >> tpr_log);
    const bool live = r < rows;
    const T* from = x + (live ? r : 0) * ldx;
    int8_t* to = q + (live ? r : 0) * ldq;
    Pack<T, V> raw[LOADS];
    uint32_t most = 0;
    auto look = [&](const Pack<T, V>& k) {
#pragma unroll
        for (int e = 0; e < V; ++e) most = max(most, __float_as_uint(to_float(k.v[e])) & 0x7fffffffu);
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int c = (i * tpr + t) * V;
            raw[i] = Pack<T, V>{};
            if (live && c < cols) raw[i] = *reinterpret_cast<const Pack<T, V>*>(from + c);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) look(raw[i]);
    } else {
#pragma unroll 4
        for (int c = t * V; live && c < cols; c += tpr * V) look(*reinterpret_cast<const Pack<T, V>*>(from + c));
    }
    most = row_most(most, tpr);
    const float top = __uint_as_float(most), inv = 127.0f / top;
    const bool odd = most >= 0x7f800000u, none = odd || most == 0;
    if (!live) return;
    auto put = [&](const Pack<T, V>& k, int c) {
        Pack<int8_t, V> out = {};
        if (!none) {
            float v[V];
            unpack<T, V>(k, v);
            quantized<V>(out, v, top, inv);
        }
        *reinterpret_cast<Pack<int8_t, V>*>(to + c) = out;
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            if ((i * tpr + t) * V < cols) put(raw[i], (i * tpr + t) * V);
    } else {
#pragma unroll 4
        for (int c = t * V; c < cols; c += tpr * V) put(*reinterpret_cast<const Pack<T, V>*>(from + c), c);
    }
    if (t == 0) scale[r] = odd ? __uint_as_float(0x7fc00000u) : top / 127.0f;
}

// 16 bytes from anywhere in a matrix (bytes [begin, end)): the two aligned 16-byte words that hold them, shifted
// together; words that reach outside, and the `valid` < 16 at a row's end, byte by byte, with zeros after them.
__device__ __forceinline__ uint4 load_bytes(const int8_t* src, int64_t valid, uintptr_t begin, uintptr_t end) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(src), low = at & ~uintptr_t(15);
    const int shift = (int)(at & 15);
    uint32_t out[4] = {0, 0, 0, 0};
    if (valid >= 16 && low >= begin && low + (shift ? 32 : 16) <= end) {
        const uint4 v0 = __ldg(reinterpret_cast<const uint4*>(low));
        const uint4 v1 = shift ? __ldg(reinterpret_cast<const uint4*>(low) + 1) : v0;
        uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        if (shift & 8)
#pragma unroll
            for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
        if (shift & 4)
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __funnelshift_r(w[i], w[i + 1], (shift & 3) * 8);
    } else {
        const uint8_t* e = reinterpret_cast<const uint8_t*>(src);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < valid) out[i / 4] |= (uint32_t)__ldg(e + i) << (i % 4 * 8);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// ---- a few rows: the weight's bytes, each used once ------------------------------------------------
// A CTA takes 16 features, its eight warps interleaved 128-byte slices of the sum. The weight goes from memory
// straight to registers as the A operand of mma.sync m16n8k32 (16 features; the tokens are the 8 columns). The
// sum's order is free, so a lane loads 32 contiguous bytes of a weight row (four lanes: a 128-byte line) and hands
// them to four MMAs as if they were the k positions the fragment layout asks for; x is loaded in the same order.
constexpr int FEW_WARPS = 8;

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 32 bytes of a row from column k on as 8 words; zeros from column K on. VEC: the row starts on 16 bytes and K is a
// multiple of 16.
template <bool VEC>
__device__ __forceinline__ void load32(uint32_t (&w)[8], const int8_t* row, int64_t k, int64_t K, bool live,
                                       uintptr_t begin, uintptr_t end) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint4 v = make_uint4(0, 0, 0, 0);
        const int64_t at = k + 16 * h;
        if (live && at < K) {
            if constexpr (VEC) v = __ldg(reinterpret_cast<const uint4*>(row + at));
            else v = load_bytes(row + at, K - at, begin, end);
        }
        w[4 * h] = v.x; w[4 * h + 1] = v.y; w[4 * h + 2] = v.z; w[4 * h + 3] = v.w;
    }
}

// NT: tokens by eights.
template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(32 * FEW_WARPS) few_rows_int8_kernel(const Int8Args p, T* y, int64_t ldy) {
    __shared__ int red[FEW_WARPS][NT * 8][16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int64_t f0 = (int64_t)blockIdx.x * 16;
    cudaGridDependencySynchronize();
    const int8_t* rows[2];  // a lane's two features; past the last: the last, not stored
#pragma unroll
    for (int h = 0; h < 2; ++h) rows[h] = p.w + min(f0 + g + 8 * h, p.F - 1) * p.ldw;
    const uintptr_t wb = reinterpret_cast<uintptr_t>(p.w), we = wb + (p.F - 1) * p.ldw + p.K;
    const uintptr_t xb = reinterpret_cast<uintptr_t>(p.x), xe = xb + (p.rows - 1) * p.ldx + p.K;
    int acc[NT][4] = {};
    const int64_t slices = (p.K + 127) / 128;
#pragma unroll 4
    for (int64_t s = warp; s < slices; s += FEW_WARPS) {
        const int64_t k = s * 128 + q * 32;
        uint32_t a[2][8], x[NT][8];
#pragma unroll
        for (int h = 0; h < 2; ++h) load32<VEC>(a[h], rows[h], k, p.K, true, wb, we);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int n = t * 8 + g;
            load32<VEC>(x[t], p.x + (n < p.rows ? n : 0) * p.ldx, k, p.K, n < p.rows, xb, xe);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t f[4] = {a[0][2 * i], a[1][2 * i], a[0][2 * i + 1], a[1][2 * i + 1]};
                mma_s8(acc[t], f, x[t][2 * i], x[t][2 * i + 1]);
            }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp][t * 8 + q * 2 + (i & 1)][g + (i >> 1) * 8] = acc[t][i];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * 16; i += 32 * FEW_WARPS) {
        const int n = i / 16, c = i % 16;
        if (n >= p.rows || f0 + c >= p.F) continue;
        int s = 0;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) s += red[w][n][c];
        y[n * ldy + f0 + c] = from_float<T>(fmaf((float)s * p.xs[n], p.ws[f0 + c], p.bias ? p.bias[f0 + c] : 0.0f));
    }
}

// ---- operands that TMA cannot address ----------------------------------------------------------------
struct Copies {
    struct {
        const int8_t* src;
        int8_t* dst;
        int64_t rows, cols, ld, ldp;
    } m[2];
};
// A warp per row, 16 bytes a lane. The row's padding becomes zeros.
__global__ void __launch_bounds__(256) restride_bytes_kernel(const __grid_constant__ Copies a) {
    const auto& m = a.m[blockIdx.y];
    cudaGridDependencySynchronize();
    const uintptr_t begin = reinterpret_cast<uintptr_t>(m.src), end = begin + (m.rows - 1) * m.ld + m.cols;
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < m.rows; r += (int64_t)gridDim.x * 8)
        for (int64_t c = (threadIdx.x & 31) * 16; c < m.cols; c += 512)
            *reinterpret_cast<uint4*>(m.dst + r * m.ldp + c) = load_bytes(m.src + r * m.ld + c, m.cols - c, begin, end);
}

bool tma_bytes(const void* p, int64_t ld) { return aligned_to(p, 16) && ld % 16 == 0 && ld < (int64_t(1) << 40); }

// x and w as TMA can read them: the caller's, or copies in scratch with rows on 16 bytes.
struct Operands {
    const int8_t* p[2];
    int64_t ld[2], rows[2], K;
    DevBuf<int8_t> copy[2];
    Operands(Handle& h, const Int8Args& a) : p{a.x, a.w}, ld{a.ldx, a.ldw}, rows{a.rows, a.F}, K(a.K) {
        Copies job = {};
        int jobs = 0;
        int64_t most = 0;
        for (int i = 0; i < 2; ++i) {
            const int64_t ldp = ceil_div(K, 16) * 16;
            if (rows[i] == 1) ld[i] = ldp;  // the stride of a single row is never taken
            if (tma_bytes(p[i], ld[i])) continue;
            copy[i] = DevBuf<int8_t>((size_t)(rows[i] * ldp), h.stream);
            job.m[jobs++] = {p[i], copy[i].get(), rows[i], K, ld[i], ldp};
            most = std::max(most, rows[i]);
            p[i] = copy[i].get();
            ld[i] = ldp;
        }
        if (jobs == 0) return;
        const dim3 grid((unsigned)std::min(ceil_div(most, 8), (int64_t)sm_count(h.device) * 8), (unsigned)jobs);
        launch_dependent(h.stream, restride_bytes_kernel, grid, 256, 0, 1, job);
        after_launch(h, "int8_restride");
    }
    CUtensorMap map(int i, int box_rows) const {
        return make_map_2d(p[i], (uint64_t)K, (uint64_t)rows[i], (uint64_t)ld[i], 128, (uint32_t)box_rows,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8);
    }
};

// y = bias: a sum of no terms.
template <typename T>
__global__ void __launch_bounds__(256) bias_kernel(int64_t rows, int64_t F, const float* bias, T* y, int64_t ldy) {
    cudaGridDependencySynchronize();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * F; i += (int64_t)gridDim.x * 256)
        y[i / F * ldy + i % F] = from_float<T>(bias ? bias[i % F] : 0.0f);
}

template <typename T, int CG>
void tiles(Handle& h, const Int8Args& a, T* y, int64_t ldy) {
    using namespace product;
    const Operands in(h, a);
    Args t = {};
    t.M = a.rows;
    t.N = a.F;
    t.ksteps = (int)ceil_div(a.K, 128);
    t.cols_first = a.rows > a.F;  // the operand of the inner index is read again and should fit L2
    choose<Epi::Int8, CG>(h, t);
    t.a[0] = in.map(0, TM);
    t.b[0] = in.map(1, t.acc_n / CG);
    t.xs = a.xs;
    t.ws = a.ws;
    t.bias = a.bias;
    if constexpr (sizeof(T) == 4) {
        if (a.rows == 1) ldy = a.F;
        t.out[0] = y;
        t.ld[0] = ldy;
        t.tma[0] = a.F % 4 == 0 && aligned_to(y, 16) && ldy % 4 == 0 && ldy < (int64_t(1) << 38);
        if (t.tma[0])
            t.omap[0] = make_map_2d(y, (uint64_t)a.F, (uint64_t)a.rows, (uint64_t)ldy * 4, 32, 32,
                                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_FLOAT32);
    } else {
        set_output(t, 0, y, ldy);
    }
    launch<Epi::Int8, T, CG, false, false>(h, t);
}

}  // namespace

template <typename T>
void quantize_rows(Handle& h, int64_t rows, int64_t cols, const T* x, int64_t ldx, int8_t* q, int64_t ldq,
                   float* scale) {
    if (rows == 0) return;
    XS_REQUIRE(cols < INT32_MAX - 65536, XSPMM_STATUS_UNSUPPORTED, "columns pass 2^31");
    auto launch = [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        const int held = cols <= 16 * Q_THREADS ? 16 : cols <= 32 * 512 ? 32 : 0;
        // enough threads to hold the row; in a small call as many as a warp can use
        int log = 0;
        while (log < 9 && ((held ? (int64_t)held << log < cols : true) || (log < 5 && V << log < cols && rows < 4096))) ++log;
        const int threads = log > 5 ? 1 << log : Q_THREADS;
        const int64_t grid = ceil_div(rows, threads >> log);
        XS_REQUIRE(grid < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "rows pass 2^31");
        auto kern = held == 16 ? quantize_kernel<T, V, 16> : held ? quantize_kernel<T, V, 32> : quantize_kernel<T, V, 0>;
        launch_dependent(h.stream, kern, (unsigned)grid, threads, 0, 1, rows, (int)cols, log, x, ldx, q, ldq, scale);
        after_launch(h, "quantize_rows");
    };
    // the widest loads that every row's start allows
    auto fits = [&](int v) {
        return cols % v == 0 && aligned_to(x, v * sizeof(T)) && aligned_to(q, v) && (rows == 1 || (ldx % v == 0 && ldq % v == 0));
    };
    constexpr int WIDE = 16 / sizeof(T);
    if (fits(WIDE)) launch(std::integral_constant<int, WIDE>{});
    else if (fits(WIDE / 2)) launch(std::integral_constant<int, WIDE / 2>{});
    else launch(std::integral_constant<int, 1>{});
}

template <typename T>
void linear_int8(Handle& h, const Int8Args& a, T* y, int64_t ldy) {
    if (a.rows == 0 || a.F == 0) return;
    const int64_t most = (int64_t(1) << 31) - 512;  // TMA coordinates are 32 bits
    XS_REQUIRE(a.rows < most && a.F < most, XSPMM_STATUS_UNSUPPORTED, "a dimension of the 8-bit product passes 2^31");
    if (a.K == 0) {
        const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(a.rows * a.F, 256), 8 * sm_count(h.device));
        launch_dependent(h.stream, bias_kernel<T>, grid, 256, 0, 1, a.rows, a.F, a.bias, y, ldy);
        after_launch(h, "int8_bias");
    } else if (a.rows <= 16) {  // 4096 -> 11008: 16 rows 15.0 us (tiles 20.2), 9 rows 13.1 (19.1), 17 rows by tiles 20.3
        const bool vec = a.K % 16 == 0 && tma_bytes(a.w, a.F > 1 ? a.ldw : 0) && tma_bytes(a.x, a.rows > 1 ? a.ldx : 0);
        auto kern = a.rows <= 8 ? (vec ? few_rows_int8_kernel<T, 1, true> : few_rows_int8_kernel<T, 1, false>)
                                : (vec ? few_rows_int8_kernel<T, 2, true> : few_rows_int8_kernel<T, 2, false>);
        launch_dependent(h.stream, kern, (unsigned)ceil_div(a.F, 16), 32 * FEW_WARPS, 0, 1, a, y, ldy);
        after_launch(h, "int8_few_rows");
    } else if (a.rows <= product::TM) {  // 128 rows 15.3 us (pairs 17.5), 129 rows by pairs 17.5 (single CTAs 16.1)
        tiles<T, 1>(h, a, y, ldy);
    } else {
        tiles<T, 2>(h, a, y, ldy);
    }
}

#define XS_INST_INT8(T)                                                                                        \
    template void quantize_rows<T>(Handle&, int64_t, int64_t, const T*, int64_t, int8_t*, int64_t, float*);     \
    template void linear_int8<T>(Handle&, const Int8Args&, T*, int64_t);
XS_INST_INT8(__half)
XS_INST_INT8(__nv_bfloat16)
XS_INST_INT8(float)

}  // namespace xspmm_b200
