// orthogonalize.cu -- the orthogonalised update of a weight matrix by Newton-Schulz steps.
//
// X = g / (|g| + eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T, taken on the smaller side:
// for more rows than columns X <- X (a I + b A + c A A) with A = X^T X. The polynomial p(s) = a s + b s^3 + c s^5
// acts on the singular values, which start in [0, 1]; it has p <= 1.2025 there (at s = 0.5545) and maps
// [0, 1.2025] into itself, so every entry of X stays below 1.21 and of A below 1.45.
#include "layers.cuh"

namespace xspmm_b200 {
namespace {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;

// Sum of squares in fp64: one partial per CTA, added in order by the next kernel.
template <typename T>
__global__ void __launch_bounds__(256) squares_kernel(int64_t rows, int64_t cols, const T* g, int64_t ldg, double* part) {
    __shared__ double red[8];
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

template <typename T>
__global__ void __launch_bounds__(256)
scale_kernel(int64_t rows, int64_t cols, const T* g, int64_t ldg, const double* part, int parts, float eps, float* x) {
    double s = 0.0;
    for (int i = 0; i < parts; ++i) s += part[i];
    const double inv = 1.0 / (sqrt(s) + (double)eps);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
        x[i] = (float)(to_float(g[i / cols * ldg + i % cols]) * inv);
}

// out = alpha * C + beta * op(A) op(B), 16 x 16 a CTA; element (i, k) of op(A) is at i * ai + k * ak.
__global__ void __launch_bounds__(256)
product_kernel(int64_t M, int64_t N, int64_t K, const float* A, int64_t ai, int64_t ak, const float* B, int64_t bk,
               int64_t bj, const float* C, float alpha, float beta, float* out) {
    __shared__ float as[16][17], bs[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t nt = (N + 15) / 16, i = blockIdx.x / nt * 16 + ty, j = blockIdx.x % nt * 16 + tx;
    float s = 0.0f;
    for (int64_t k0 = 0; k0 < K; k0 += 16) {
        as[ty][tx] = i < M && k0 + tx < K ? A[i * ai + (k0 + tx) * ak] : 0.0f;
        bs[ty][tx] = j < N && k0 + ty < K ? B[(k0 + ty) * bk + j * bj] : 0.0f;
        __syncthreads();
        for (int k = 0; k < 16; ++k) s = fmaf(as[ty][k], bs[k][tx], s);
        __syncthreads();
    }
    if (i < M && j < N) out[i * N + j] = beta * s + (C ? alpha * C[i * N + j] : 0.0f);
}

template <typename T>
__global__ void __launch_bounds__(256) store_kernel(int64_t rows, int64_t cols, const float* x, T* y, int64_t ldy) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
        y[i / cols * ldy + i % cols] = from_float<T>(x[i]);
}

}  // namespace

template <typename TX, typename TY>
void orthogonalize(Handle& h, int64_t rows, int64_t cols, const TX* g, int64_t ldg, int steps, float eps, TY* y,
                   int64_t ldy) {
    if (rows == 0 || cols == 0) return;
    const int parts = (int)std::min<int64_t>(ceil_div(rows * cols, 4096), sm_count(h.device));
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows * cols, 256), 8 * sm_count(h.device));
    const int64_t m = std::min(rows, cols);
    const bool tall = rows > cols;
    DevBuf<double> part((size_t)parts, h.stream);
    DevBuf<float> buf((size_t)(2 * rows * cols + 2 * m * m), h.stream);
    float *x = buf.get(), *next = x + rows * cols, *A = next + rows * cols, *B = A + m * m;
    squares_kernel<TX><<<parts, 256, 0, h.stream>>>(rows, cols, g, ldg, part.get());
    after_launch(h, "update_squares");
    scale_kernel<TX><<<grid, 256, 0, h.stream>>>(rows, cols, g, ldg, part.get(), parts, eps, x);
    after_launch(h, "update_scale");
    auto product = [&](int64_t M, int64_t N, int64_t K, const float* P, int64_t pi, int64_t pk, const float* Q,
                       int64_t qk, int64_t qj, const float* C, float alpha, float beta, float* out) {
        const int64_t tiles = ceil_div(M, 16) * ceil_div(N, 16);
        XS_REQUIRE(tiles < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "grid too large");
        product_kernel<<<(unsigned)tiles, 256, 0, h.stream>>>(M, N, K, P, pi, pk, Q, qk, qj, C, alpha, beta, out);
        after_launch(h, "update_product");
    };
    for (int i = 0; i < steps; ++i) {
        if (tall) product(m, m, rows, x, 1, cols, x, cols, 1, nullptr, 0.0f, 1.0f, A);
        else product(m, m, cols, x, cols, 1, x, 1, cols, nullptr, 0.0f, 1.0f, A);
        product(m, m, m, A, m, 1, A, m, 1, A, NS_B, NS_C, B);
        if (tall) product(rows, cols, m, x, cols, 1, B, m, 1, x, NS_A, 1.0f, next);
        else product(rows, cols, m, B, m, 1, x, cols, 1, x, NS_A, 1.0f, next);
        std::swap(x, next);
    }
    store_kernel<TY><<<grid, 256, 0, h.stream>>>(rows, cols, x, y, ldy);
    after_launch(h, "update_store");
}

#define XS_INST_UPDATE(TX, TY) \
    template void orthogonalize<TX, TY>(Handle&, int64_t, int64_t, const TX*, int64_t, int, float, TY*, int64_t);
XS_INST_UPDATE(__half, __half)
XS_INST_UPDATE(__nv_bfloat16, __nv_bfloat16)
XS_INST_UPDATE(float, __half)
XS_INST_UPDATE(float, __nv_bfloat16)

}  // namespace xspmm_b200
