// gated_ffn.cu -- the gated feed-forward block and its gradient.
//
// Forward: g = x wg^T, u = x wu^T, y = act(g) * u. Backward, from dy and the kept g and u:
// du = dy * act(g), dg = dy * u * act'(g), dx = dg wg + du wu, dwg = dg^T x, dwu = du^T x.
// Sums are held in fp32; dg and du are rounded to the operands' 16-bit type before the products,
// as any 16-bit matrix product's operand is.
#include "layers.cuh"

namespace xspmm_b200 {
namespace {

__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + __expf(-v)); }

template <Activation ACT>
__device__ __forceinline__ float act_value(float v) {
    if constexpr (ACT == Activation::Silu) return v * sigmoid(v);
    else if constexpr (ACT == Activation::Gelu) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    else if constexpr (ACT == Activation::Relu) return v > 0.0f ? v : (v != v ? v : 0.0f);
    else return sigmoid(v);
}
template <Activation ACT>
__device__ __forceinline__ float act_slope(float v) {
    if constexpr (ACT == Activation::Silu) {
        const float s = sigmoid(v);
        return s * (1.0f + v * (1.0f - s));
    } else if constexpr (ACT == Activation::Gelu) {
        return 0.5f * (1.0f + erff(v * 0.70710678118654752f)) +
               v * __expf(-0.5f * v * v) * 0.39894228040143268f;
    } else if constexpr (ACT == Activation::Relu) {
        return v > 0.0f ? 1.0f : 0.0f;
    } else {
        const float s = sigmoid(v);
        return s * (1.0f - s);
    }
}

// out[i, j] = sum over the segments s and k of a_s[i, k] * b_s[k, j], any element strides.
template <typename T>
struct Operand {
    const T* p;
    int64_t si, sk;  // strides of the output index and of the summed index
};
constexpr int PT = 64, PK = 16;  // output tile, summed slice; 256 threads of 4 x 4 outputs

template <typename T>
__device__ void product_tile(const Operand<T>& a, const Operand<T>& b, int64_t M, int64_t N,
                             int64_t K, int64_t i0, int64_t j0, float (&acc)[4][4]) {
    __shared__ float sa[PK][PT + 1], sb[PK][PT + 1];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int64_t k0 = 0; k0 < K; k0 += PK) {
        __syncthreads();
        for (int e = threadIdx.x; e < PT * PK; e += 256) {
            const int i = e / PK, k = e % PK;
            sa[k][i] = i0 + i < M && k0 + k < K ? to_float(a.p[(i0 + i) * a.si + (k0 + k) * a.sk]) : 0.0f;
            sb[k][i] = j0 + i < N && k0 + k < K ? to_float(b.p[(j0 + i) * b.si + (k0 + k) * b.sk]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += sa[k][ty + 16 * i] * sb[k][tx + 16 * j];
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
product_kernel(Operand<T> a0, Operand<T> b0, Operand<T> a1, Operand<T> b1, int64_t M, int64_t N,
               int64_t K, T* out, int64_t ldo) {
    const int64_t nt = (N + PT - 1) / PT;
    const int64_t i0 = blockIdx.x / nt * PT, j0 = blockIdx.x % nt * PT;
    float acc[4][4] = {};
    product_tile(a0, b0, M, N, K, i0, j0, acc);
    if (a1.p) product_tile(a1, b1, M, N, K, i0, j0, acc);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t r = i0 + ty + 16 * i, c = j0 + tx + 16 * j;
            if (r < M && c < N) out[r * ldo + c] = from_float<T>(acc[i][j]);
        }
}

template <typename T, Activation ACT>
__global__ void __launch_bounds__(256)
gated_kernel(GatedArgs<T> p, T* y, int64_t ldy, T* gate, T* up) {
    const int64_t nt = (p.F + PT - 1) / PT;
    const int64_t i0 = blockIdx.x / nt * PT, j0 = blockIdx.x % nt * PT;
    float g[4][4] = {}, u[4][4] = {};
    const Operand<T> x{p.x, p.ldx, 1};
    product_tile(x, Operand<T>{p.wg, p.ldwg, 1}, p.rows, p.F, p.K, i0, j0, g);
    product_tile(x, Operand<T>{p.wu, p.ldwu, 1}, p.rows, p.F, p.K, i0, j0, u);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t r = i0 + ty + 16 * i, c = j0 + tx + 16 * j;
            if (r >= p.rows || c >= p.F) continue;
            y[r * ldy + c] = from_float<T>(act_value<ACT>(g[i][j]) * u[i][j]);
            if (gate) gate[r * p.F + c] = from_float<T>(g[i][j]);
            if (up) up[r * p.F + c] = from_float<T>(u[i][j]);
        }
}

// dg and du, rows x F contiguous.
template <typename T, Activation ACT>
__global__ void __launch_bounds__(256)
gated_slopes_kernel(int64_t rows, int64_t F, const T* dy, int64_t lddy, const T* gate, const T* up,
                    T* dg, T* du) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * F;
         i += (int64_t)gridDim.x * 256) {
        const float d = to_float(dy[i / F * lddy + i % F]), g = to_float(gate[i]);
        du[i] = from_float<T>(d * act_value<ACT>(g));
        dg[i] = from_float<T>(d * to_float(up[i]) * act_slope<ACT>(g));
    }
}

template <typename F>
void with_activation(Activation a, F&& f) {
    switch (a) {
        case Activation::Silu: return f(std::integral_constant<Activation, Activation::Silu>{});
        case Activation::Gelu: return f(std::integral_constant<Activation, Activation::Gelu>{});
        case Activation::Relu: return f(std::integral_constant<Activation, Activation::Relu>{});
        case Activation::Sigmoid: return f(std::integral_constant<Activation, Activation::Sigmoid>{});
    }
}

unsigned tile_grid(int64_t M, int64_t N) {
    const int64_t t = ceil_div(M, PT) * ceil_div(N, PT);
    XS_REQUIRE(t < (int64_t(1) << 31), XSPMM_STATUS_UNSUPPORTED, "grid too large");
    return (unsigned)t;
}

}  // namespace

template <typename T>
void gated_ffn(Handle& h, const GatedArgs<T>& a, T* y, int64_t ldy, T* gate, T* up) {
    if (a.rows == 0 || a.F == 0) return;
    with_activation(a.act, [&](auto act) {
        gated_kernel<T, decltype(act)::value>
            <<<tile_grid(a.rows, a.F), 256, 0, h.stream>>>(a, y, ldy, gate, up);
    });
    after_launch(h, "gated_ffn");
}

template <typename T>
void gated_ffn_backward(Handle& h, const GatedArgs<T>& a, const T* dy, int64_t lddy, const T* gate,
                        const T* up, T* dx, int64_t lddx, T* dwg, T* dwu) {
    const int64_t n = a.rows * a.F;
    DevBuf<T> d(std::max<int64_t>(2 * n, 1), h.stream);
    T *dg = d.get(), *du = d.get() + n;
    if (n > 0) {
        const unsigned grid = (unsigned)std::min(ceil_div(n, 256), (int64_t)sm_count(h.device) * 8);
        with_activation(a.act, [&](auto act) {
            gated_slopes_kernel<T, decltype(act)::value>
                <<<grid, 256, 0, h.stream>>>(a.rows, a.F, dy, lddy, gate, up, dg, du);
        });
        after_launch(h, "gated_slopes");
    }
    const Operand<T> none{nullptr, 0, 0};
    if (dx && a.rows > 0) {
        product_kernel<T><<<tile_grid(a.rows, a.K), 256, 0, h.stream>>>(
            Operand<T>{dg, a.F, 1}, Operand<T>{a.wg, 1, a.ldwg}, Operand<T>{du, a.F, 1},
            Operand<T>{a.wu, 1, a.ldwu}, a.rows, a.K, a.F, dx, lddx);
        after_launch(h, "gated_dx");
    }
    if (dwg && a.F > 0) {
        const T* src[2] = {dg, du};
        T* dst[2] = {dwg, dwu};
        for (int i = 0; i < 2; ++i) {
            product_kernel<T><<<tile_grid(a.F, a.K), 256, 0, h.stream>>>(
                Operand<T>{src[i], 1, a.F}, Operand<T>{a.x, 1, a.ldx}, none, none, a.F, a.K, a.rows,
                dst[i], a.K);
            after_launch(h, "gated_dw");
        }
    }
}

#define XS_INST_FFN(T)                                                                            \
    template void gated_ffn<T>(Handle&, const GatedArgs<T>&, T*, int64_t, T*, T*);                \
    template void gated_ffn_backward<T>(Handle&, const GatedArgs<T>&, const T*, int64_t, const T*, \
                                        const T*, T*, int64_t, T*, T*);
XS_INST_FFN(__half)
XS_INST_FFN(__nv_bfloat16)

}  // namespace xspmm_b200
