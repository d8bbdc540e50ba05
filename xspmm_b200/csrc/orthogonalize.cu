// orthogonalize.cu -- the orthogonalised update of a weight matrix by Newton-Schulz steps.
//
// X = g / (|g| + eps), then `steps` times X <- B' X, B' = a I + b A + c A A, A = X X^T, taken on the smaller side:
// for more rows than columns X <- X B' with A = X^T X. The polynomial p(s) = a s + b s^3 + c s^5 acts on the
// singular values, which start in [0, 1]; it is at most 1.2025 there (at s = 0.5545) and maps [0, 1.2025] into
// itself, so every entry of X stays below 1.21, of A below 1.45 and of B' (eigenvalues in [0.63, 3.4445]) below 3.45.
//
// Precision. A step multiplies small singular values by 3.4445, 485 in five steps, and what rounding X to 16 bits
// would add to those directions with them. X, A and B' are therefore held as two fp16 parts (22 bits), and the
// products are those of the parts with fp32 sums (tile_product.cuh). A and B' are symmetric: half of their tiles
// are computed. The norm is summed in fp64: squares of any fp32 gradient are in its range.
#include "tile_product.cuh"

namespace xspmm_b200 {
namespace {

using namespace product;

// Sum of squares in fp64: one partial per CTA, added in order by the next kernel.
template <typename T>
__global__ void __launch_bounds__(256) squares_kernel(int64_t rows, int64_t cols, const T* g, int64_t ldg, double* part) {
    __shared__ double red[8];
    cudaGridDependencySynchronize();
    double s = 0.0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256) {
        const double v = to_float(g[i / cols * ldg + i % cols]);
        s += v * v;
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) s += red[i];
        part[blockIdx.x] = s;
    }
}

// The inverse of the norm, from the partial sums in their order; the same in all threads.
__device__ __forceinline__ double inverse_norm(const double* part, int parts, float eps) {
    __shared__ double inv;
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < parts; ++i) s += part[i];
        inv = 1.0 / (sqrt(s) + (double)eps);
    }
    __syncthreads();
    return inv;
}

// X_0 in two parts; the padding of its rows becomes zeros.
template <typename T>
__global__ void __launch_bounds__(256)
start_kernel(int64_t rows, int64_t cols, const T* g, int64_t ldg, const double* part, int parts, float eps, __half* hi,
             __half* lo, int64_t ld) {
    cudaGridDependencySynchronize();
    const double inv = inverse_norm(part, parts, eps);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * (ld / 2); i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / (ld / 2), c = (i - r * (ld / 2)) * 2;
        const float v0 = c < cols ? (float)(to_float(g[r * ldg + c]) * inv) * SPLIT_SCALE : 0.0f;
        const float v1 = c + 1 < cols ? (float)(to_float(g[r * ldg + c + 1]) * inv) * SPLIT_SCALE : 0.0f;
        uint32_t h, l;
        split2(v0, v1, &h, &l);
        *reinterpret_cast<uint32_t*>(hi + r * ld + c) = h;
        *reinterpret_cast<uint32_t*>(lo + r * ld + c) = l;
    }
}

// y = X_0: no steps.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256)
scaled_kernel(int64_t rows, int64_t cols, const TX* g, int64_t ldg, const double* part, int parts, float eps, TY* y,
              int64_t ldy) {
    cudaGridDependencySynchronize();
    const double inv = inverse_norm(part, parts, eps);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
        y[i / cols * ldy + i % cols] = from_float<TY>((float)(to_float(g[i / cols * ldg + i % cols]) * inv));
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
void multiply(Handle& h, int64_t M, int64_t N, int64_t K, const Parts& P, const Parts& Q, const Parts* out,
              const Parts* A, T* y, int64_t ldy) {
    Args t = {};
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
void multiply(Handle& h, int64_t M, int64_t N, int64_t K, const Parts& P, const Parts& Q, const Parts* out,
              const Parts* A = nullptr, T* y = nullptr, int64_t ldy = 0) {
    if (M > TM) multiply<E, T, 2, AMN, BMN>(h, M, N, K, P, Q, out, A, y, ldy);
    else multiply<E, T, 1, AMN, BMN>(h, M, N, K, P, Q, out, A, y, ldy);
}

}  // namespace

template <typename TX, typename TY>
void orthogonalize(Handle& h, int64_t rows, int64_t cols, const TX* g, int64_t ldg, int steps, float eps, TY* y,
                   int64_t ldy) {
    if (rows == 0 || cols == 0) return;
    const int64_t limit = (int64_t(1) << 31) - 512;  // TMA coordinates are 32 bits
    XS_REQUIRE(rows < limit && cols < limit, XSPMM_STATUS_UNSUPPORTED, "a dimension of the update passes 2^31");
    const int parts = (int)std::min<int64_t>(ceil_div(rows * cols, 4096), sm_count(h.device));
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows * cols, 512), 8 * sm_count(h.device));
    DevBuf<double> part((size_t)parts, h.stream);
    launch_dependent(h.stream, squares_kernel<TX>, (unsigned)parts, 256, 0, 1, rows, cols, g, ldg, part.get());
    after_launch(h, "update_squares");
    if (steps == 0) {
        launch_dependent(h.stream, scaled_kernel<TX, TY>, grid, 256, 0, 1, rows, cols, g, ldg, part.get(), parts, eps, y, ldy);
        after_launch(h, "update_scaled");
        return;
    }
    const bool tall = rows > cols;
    const int64_t m = std::min(rows, cols), ldx = ceil_div(cols, 8) * 8, lda = ceil_div(m, 8) * 8;
    DevBuf<__half> buf((size_t)(4 * rows * ldx + 4 * m * lda), h.stream);
    __half* at = buf.get();
    auto take = [&](int64_t r, int64_t c, int64_t ld) {
        const Parts p{at, at + r * ld, r, c, ld};
        at += 2 * r * ld;
        return p;
    };
    Parts X = take(rows, cols, ldx), next = take(rows, cols, ldx), A = take(m, m, lda), B = take(m, m, lda);
    launch_dependent(h.stream, start_kernel<TX>, grid, 256, 0, 1, rows, cols, g, ldg, part.get(), parts, eps, X.hi, X.lo, ldx);
    after_launch(h, "update_start");
    for (int i = 0; i < steps; ++i) {
        if (tall) multiply<Epi::Gram, __half, true, true>(h, m, m, rows, X, X, &A);
        else multiply<Epi::Gram, __half, false, false>(h, m, m, cols, X, X, &A);
        multiply<Epi::Poly, __half, false, false>(h, m, m, m, A, A, &B, &A);
        if (i + 1 == steps) {
            if (tall) multiply<Epi::Last, TY, false, false>(h, rows, m, m, X, B, nullptr, nullptr, y, ldy);
            else multiply<Epi::Last, TY, false, true>(h, m, cols, m, B, X, nullptr, nullptr, y, ldy);
        } else if (tall) {
            multiply<Epi::Next, __half, false, false>(h, rows, m, m, X, B, &next);
        } else {
            multiply<Epi::Next, __half, false, true>(h, m, cols, m, B, X, &next);
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
