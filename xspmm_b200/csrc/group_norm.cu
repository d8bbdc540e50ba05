// group_norm.cu -- group norm with an activation over the samples of a packed batch, forward and backward.
//
// Forward: over the n values of a sample's rows and a group's channels, mean = sum(x) / n,
// var = sum((x - mean)^2) / n, rstd = 1 / sqrt(var + eps); z = ((x - mean) * rstd) * w + b, y = act(z).
// Backward: dz = dy * act'(z), t = dz * w, dx = rstd * (t - mean(t) - xh * mean(t * xh)), dw = sum of dz * xh,
// db = sum of dz over all samples' rows.
//
// One CTA per sample and group, which reads the group's values three times.
#include "gated_tc.cuh"

namespace xspmm_b200 {
namespace {

constexpr int GN_THREADS = 256;

// A CTA's sum, the same in all its threads.
__device__ __forceinline__ float cta_sum(float v) {
    __shared__ float part[GN_THREADS / 32];
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < GN_THREADS / 32; ++i) v += part[i];
    return v;
}

// Sample s's rows, within the matrix whatever the offsets hold.
struct Span {
    int64_t begin, end;
};
__device__ __forceinline__ Span span_of(const int64_t* offsets, int64_t s, int64_t rows) {
    if (!offsets) return {0, rows};
    const int64_t b = max((int64_t)0, min(rows, offsets[s]));
    return {b, max(b, min(rows, offsets[s + 1]))};
}

// z, each operation rounded by itself: the sign of z, which decides relu's slope, is then the same however the
// compiler orders the code around it.
__device__ __forceinline__ float affine(float xh, float w, float b) { return __fadd_rn(__fmul_rn(xh, w), b); }
__device__ __forceinline__ float centred(float x, float mean, float rstd) {
    return __fmul_rn(__fsub_rn(x, mean), rstd);
}

// act(z) and its slope. 16-bit outputs take the block's approximate forms (errors far below their rounding),
// fp32 ones CUDA's accurate functions.
template <typename TY>
__device__ __forceinline__ float act_of(Activation act, float z) {
    constexpr bool FINE = sizeof(TY) == 4;
    if constexpr (FINE) {
        switch (act) {
            case Activation::Silu: return z > -gated::SILU_END ? z / (1.0f + expf(-z)) : (z != z ? z : 0.0f);
            case Activation::Gelu: return z > -gated::GELU_END ? z * normcdff(z) : (z != z ? z : 0.0f);
            case Activation::Sigmoid: return 1.0f / (1.0f + expf(-z));
            case Activation::Relu: return z > 0.0f ? z : (z != z ? z : 0.0f);
            default: return z;
        }
    } else {
        float v = z;
        if (act != Activation::None)
            gated::with_activation(act, [&](auto a) { v = gated::act_value<decltype(a)::value>(z); });
        return v;
    }
}
template <typename TY>
__device__ __forceinline__ float slope_of(Activation act, float z) {
    constexpr bool FINE = sizeof(TY) == 4;
    if (act == Activation::None) return 1.0f;
    if constexpr (FINE) {
        switch (act) {
            case Activation::Silu: {
                const float low = fmaxf(fminf(z, gated::SILU_END), -gated::SILU_END);
                const float e = expf(-low), s = 1.0f / (1.0f + e);
                return z != z ? z : s * (1.0f + low * (e * s));
            }
            case Activation::Gelu: {
                const float low = fmaxf(fminf(z, gated::GELU_END), -gated::GELU_END);
                return z != z ? z : normcdff(low) + low * 0.39894228040143268f * expf(-0.5f * low * low);
            }
            case Activation::Sigmoid: {
                const float e = expf(-fabsf(z)), high = 1.0f / (1.0f + e);
                return high * (e * high);
            }
            default: return z > 0.0f ? 1.0f : 0.0f;
        }
    } else {
        float v = 1.0f, value;
        gated::with_activation(act, [&](auto a) { gated::act_both<decltype(a)::value>(z, &value, &v); });
        return v;
    }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(GN_THREADS)
group_norm_kernel(const GroupNormArgs<TX> a, float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    const int64_t s = blockIdx.x / a.groups, g = blockIdx.x % a.groups, width = a.C / a.groups;
    const Span rows = span_of(a.offsets, s, a.rows);
    const int64_t n = (rows.end - rows.begin) * width;
    auto each = [&](auto&& f) {
        for (int64_t i = threadIdx.x; i < n; i += GN_THREADS) f(rows.begin + i / width, g * width + i % width);
    };
    float v = 0.0f;
    each([&](int64_t r, int64_t c) { v += to_float(a.x[r * a.ldx + c]); });
    const float m = n ? cta_sum(v) / (float)n : 0.0f;
    v = 0.0f;
    each([&](int64_t r, int64_t c) {
        const float d = to_float(a.x[r * a.ldx + c]) - m;
        v = fmaf(d, d, v);
    });
    const float rs = 1.0f / sqrtf((n ? cta_sum(v) / (float)n : 0.0f) + eps);
    each([&](int64_t r, int64_t c) {
        const float xh = centred(to_float(a.x[r * a.ldx + c]), m, rs);
        y[r * ldy + c] = from_float<TY>(act_of<TY>(a.act, affine(xh, a.w ? a.w[c] : 1.0f, a.b ? a.b[c] : 0.0f)));
    });
    if (threadIdx.x == 0) {
        if (mean) mean[blockIdx.x] = m;
        if (rstd) rstd[blockIdx.x] = rs;
    }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(GN_THREADS)
group_norm_grad_kernel(const GroupNormArgs<TX> a, const TY* dy, int64_t lddy, const float* mean, const float* rstd,
                       TY* dx, int64_t lddx) {
    const int64_t s = blockIdx.x / a.groups, g = blockIdx.x % a.groups, width = a.C / a.groups;
    const Span rows = span_of(a.offsets, s, a.rows);
    const int64_t n = (rows.end - rows.begin) * width;
    const float m = mean[blockIdx.x], rs = rstd[blockIdx.x];
    auto each = [&](auto&& f) {
        for (int64_t i = threadIdx.x; i < n; i += GN_THREADS) {
            const int64_t r = rows.begin + i / width, c = g * width + i % width;
            const float xh = centred(to_float(a.x[r * a.ldx + c]), m, rs), w = a.w ? a.w[c] : 1.0f;
            const float z = affine(xh, w, a.b ? a.b[c] : 0.0f);
            f(r, c, xh, to_float(dy[r * lddy + c]) * slope_of<TY>(a.act, z) * w);
        }
    };
    float s1 = 0.0f, s2 = 0.0f;
    each([&](int64_t, int64_t, float xh, float t) { s1 += t, s2 = fmaf(t, xh, s2); });
    if (n == 0) return;
    s1 = cta_sum(s1) / (float)n;
    s2 = cta_sum(s2) / (float)n;
    each([&](int64_t r, int64_t c, float xh, float t) { dx[r * lddx + c] = from_float<TY>(rs * (t - s1 - xh * s2)); });
}

// A CTA per channel.
template <typename TX, typename TY>
__global__ void __launch_bounds__(GN_THREADS)
group_norm_weight_kernel(const GroupNormArgs<TX> a, const TY* dy, int64_t lddy, const float* mean, const float* rstd,
                         float* dw, float* db) {
    const int64_t c = blockIdx.x, g = c / (a.C / a.groups);
    const float w = a.w ? a.w[c] : 1.0f, b = a.b ? a.b[c] : 0.0f;
    float sw = 0.0f, sb = 0.0f;
    for (int64_t s = 0; s < a.samples; ++s) {
        const Span rows = span_of(a.offsets, s, a.rows);
        const float m = mean[s * a.groups + g], rs = rstd[s * a.groups + g];
        for (int64_t r = rows.begin + threadIdx.x; r < rows.end; r += GN_THREADS) {
            const float xh = centred(to_float(a.x[r * a.ldx + c]), m, rs);
            const float dz = to_float(dy[r * lddy + c]) * slope_of<TY>(a.act, affine(xh, w, b));
            sw = fmaf(dz, xh, sw);
            sb += dz;
        }
    }
    sw = cta_sum(sw);
    sb = cta_sum(sb);
    if (threadIdx.x == 0) {
        if (dw) dw[c] = sw;
        if (db) db[c] = sb;
    }
}

}  // namespace

template <typename TX, typename TY>
void group_norm(Handle& h, const GroupNormArgs<TX>& a, float eps, TY* y, int64_t ldy, float* mean, float* rstd) {
    if (a.samples == 0) return;
    XS_REQUIRE(a.samples * a.groups < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "too many samples and groups");
    group_norm_kernel<TX, TY><<<(unsigned)(a.samples * a.groups), GN_THREADS, 0, h.stream>>>(a, eps, y, ldy, mean, rstd);
    after_launch(h, "group_norm");
}

template <typename TX, typename TY>
void group_norm_backward(Handle& h, const GroupNormArgs<TX>& a, const TY* dy, int64_t lddy, const float* mean,
                         const float* rstd, TY* dx, int64_t lddx, float* dw, float* db) {
    XS_REQUIRE(a.samples * a.groups < INT32_MAX, XSPMM_STATUS_UNSUPPORTED, "too many samples and groups");
    if (dw || db) {
        group_norm_weight_kernel<TX, TY><<<(unsigned)a.C, GN_THREADS, 0, h.stream>>>(a, dy, lddy, mean, rstd, dw, db);
        after_launch(h, "group_norm_weight");
    }
    if (dx && a.samples > 0) {
        group_norm_grad_kernel<TX, TY>
            <<<(unsigned)(a.samples * a.groups), GN_THREADS, 0, h.stream>>>(a, dy, lddy, mean, rstd, dx, lddx);
        after_launch(h, "group_norm_grad");
    }
}

#define XS_INST_GROUP_NORM(TX, TY)                                                                              \
    template void group_norm<TX, TY>(Handle&, const GroupNormArgs<TX>&, float, TY*, int64_t, float*, float*);    \
    template void group_norm_backward<TX, TY>(Handle&, const GroupNormArgs<TX>&, const TY*, int64_t,             \
                                              const float*, const float*, TY*, int64_t, float*, float*);
XS_INST_GROUP_NORM(__half, __half)
XS_INST_GROUP_NORM(__nv_bfloat16, __nv_bfloat16)
XS_INST_GROUP_NORM(float, float)
XS_INST_GROUP_NORM(float, __half)
XS_INST_GROUP_NORM(float, __nv_bfloat16)

}  // namespace xspmm_b200
