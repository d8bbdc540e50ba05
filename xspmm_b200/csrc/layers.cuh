// layers.cuh -- internal host entry points of the layer operators that stand next to the sparse
// product (layer norm, dropout, gated feed-forward) and the device pieces they share. Rows are
// nodes or tokens, features are contiguous; ld* are row strides in elements.
#pragma once

#include "ops.cuh"

namespace xspmm_b200 {

// Layer norm over each row's D features (layer_norm.cu). w, b, mean, rstd may be null.
template <typename TX, typename TY>
void layer_norm(Handle& h, int64_t rows, int64_t D, const TX* x, int64_t ldx, const float* w,
                const float* b, float eps, TY* y, int64_t ldy, float* mean, float* rstd);
// Its gradient; any of dx, dw, db may be null. dy and dx have the output's type.
template <typename TX, typename TY>
void layer_norm_backward(Handle& h, int64_t rows, int64_t D, const TY* dy, int64_t lddy,
                         const TX* x, int64_t ldx, const float* w, const float* mean,
                         const float* rstd, TY* dx, int64_t lddx, float* dw, float* db);

// y = residual + keep * x / (1 - p) over n contiguous elements (dropout.cu).
template <typename T>
void dropout(Handle& h, int64_t n, const T* x, const T* residual, double p, uint64_t seed,
             uint64_t offset, T* y);

// Gated feed-forward block (gated_ffn.cu).
enum class Activation { Silu = 0, Gelu = 1, Relu = 2, Sigmoid = 3 };
template <typename T>
struct GatedArgs {
    int64_t rows, K, F;  // x is rows x K, the weights F x K, the block's output rows x F
    Activation act;
    const T* x;
    int64_t ldx;
    const T* wg;
    int64_t ldwg;
    const T* wu;
    int64_t ldwu;
};
// y = act(x wg^T) * (x wu^T); gate and up (rows x F, contiguous) receive the two projections when
// they are not null.
template <typename T>
void gated_ffn(Handle& h, const GatedArgs<T>& a, T* y, int64_t ldy, T* gate, T* up);
// Gradients from dy and the kept projections. dx may be null; dwg and dwu (F x K, contiguous) are
// both null or both given.
template <typename T>
void gated_ffn_backward(Handle& h, const GatedArgs<T>& a, const T* dy, int64_t lddy, const T* gate,
                        const T* up, T* dx, int64_t lddx, T* dwg, T* dwu);

// ---- device pieces ------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// V consecutive elements, moved with the widest loads and stores their size allows (the caller
// guarantees that alignment).
template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
    T v[V];
};
// Two values as one word, the first in the low half.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {  // bf16 is fp32's high half
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
// A pack's values as floats and back: one instruction per value, or per two when narrowing.
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& k, float (&out)[V]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 f = unpack2(reinterpret_cast<const uint32_t*>(&k)[i / 2], T());
            out[i] = f.x;
            out[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = to_float(k.v[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&out)[V]) {
    unpack<T, V>(*reinterpret_cast<const Pack<T, V>*>(p), out);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[V]) {
    Pack<T, V> k;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2)
            reinterpret_cast<uint32_t*>(&k)[i / 2] = pack2(in[i], in[i + 1], T());
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) k.v[i] = from_float<T>(in[i]);
    }
    *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

inline bool aligned_to(const void* p, size_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace xspmm_b200
