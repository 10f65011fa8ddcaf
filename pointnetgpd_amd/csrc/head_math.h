// Element types, activations and reductions shared by the classification-head kernels.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "pngpd.h"

namespace pngpd {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }      // rounds to nearest even

// act(z) and act'(z).  gelu: z Phi(z); gelu_tanh: z sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3), which is
// 0.5 z (1 + tanh u) without tanh's cancellation for large negative z; silu: z sigmoid(z).  z = -inf gives 0 and slope
// 0 in all of them (the limits; the plain formulas give -inf * 0), NaN stays NaN.
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_f(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float sigmoid_f(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_f(-LOG2E * v)); }
// z times a gate that has reached 0 where z is -inf (NaN stays in the gate)
__device__ __forceinline__ float gated(float z, float gate) { return __builtin_fmaxf(z, -3.0e38f) * gate; }
// sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3)
__device__ __forceinline__ float gelu_gate(float z) {
    const float k = -2.f * LOG2E * 0.7978845608028654f;
    return __builtin_amdgcn_rcpf(1.f + exp2_f(z * __builtin_fmaf(k * 0.044715f, z * z, k)));
}

constexpr float GELU_C = 0.7978845608028654f;      // sqrt(2 / pi)

// Phi(z), and exp(-z^2 / 2) on the way.  Phi(-|z|) = exp(-z^2 / 2) Q(t), t = 1 / (1 + 0.297 |z|): Q is a least-squares fit of
// erfcx's scaled form in t, reweighted towards equal relative error over |z| <= 14 (4e-8 in exact arithmetic, 3e-7 in 32 bits);
// one exponential and one reciprocal, where the library's erfcf takes some 60 instructions.  The exponential's argument is
// rounded to 32 bits, which Phi sees as an error growing with z^2: 1e-6 of its value at z = -3, 7e-6 at -12.
__device__ __forceinline__ float normal_cdf(float z, float* bell) {
    const float e = exp2_f(-0.5f * LOG2E * z * z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.2969848480983499f, __builtin_fabsf(z), 1.f));
    float q = 0.0391947381f;
    q = __builtin_fmaf(q, t, -0.178475707f);
    q = __builtin_fmaf(q, t, 0.255165062f);
    q = __builtin_fmaf(q, t, -0.101603871f);
    q = __builtin_fmaf(q, t, 0.157105486f);
    q = __builtin_fmaf(q, t, 0.0886519629f);
    q = __builtin_fmaf(q, t, 0.121786028f);
    q = __builtin_fmaf(q, t, 0.118163349f);
    q = __builtin_fmaf(q, t, 1.29719759e-05f);
    q *= e;
    *bell = e;
    return z < 0.f ? q : 1.f - q;
}

template <int ACT>
__device__ __forceinline__ float act_f(float z) {
    if constexpr (ACT == PNGPD_ACT_RELU) return z < 0.f ? 0.f : z;
    if constexpr (ACT == PNGPD_ACT_GELU) {
        float bell;
        return gated(z, normal_cdf(z, &bell));
    }
    if constexpr (ACT == PNGPD_ACT_GELU_TANH)
        return gated(z, gelu_gate(z));
    if constexpr (ACT == PNGPD_ACT_SILU) return gated(z, sigmoid_f(z));
    return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == PNGPD_ACT_RELU) return z > 0.f ? 1.f : z == z ? 0.f : z;
    if constexpr (ACT == PNGPD_ACT_GELU) {
        float bell;
        const float s = normal_cdf(z, &bell);
        // beyond 16 the bell is below 1e-55 (and an infinite z would make 0 * inf of it)
        return __builtin_fabsf(z) > 16.f ? (z > 0.f ? 1.f : 0.f) : __builtin_fmaf(z * 0.3989422804014327f, bell, s);
    }
    if constexpr (ACT == PNGPD_ACT_GELU_TANH) {
        const float s = gelu_gate(z);
        const float v = s + z * s * (1.f - s) * 2.f * GELU_C * (1.f + 0.134145f * z * z);
        return __builtin_fabsf(z) > 16.f ? (z > 0.f ? 1.f : 0.f) : v;
    }
    if constexpr (ACT == PNGPD_ACT_SILU) {
        const float s = sigmoid_f(z);
        const float v = s + z * s * (1.f - s);
        return __builtin_fabsf(z) > 100.f ? (z > 0.f ? 1.f : 0.f) : v;
    }
    return z == z ? 1.f : z;
}

// The pre-activation kept for the backward pass, rounded to the operands' type: 32 bits would cost as much memory again, for an
// error of dx and dW of 0.00235 of their norm instead of 0.00242 in bfloat16 (dz's own rounding makes the most of it).  A ReLU's slope is its sign, so a sum
// that the type would round to zero keeps it: it becomes the type's smallest number.
template <typename T, int ACT>
__device__ __forceinline__ T keep_z(float z) {
    T r = (T)z;
    if constexpr (ACT == PNGPD_ACT_RELU && sizeof(T) == 2) {
        if (z > 0.f && (float)r == 0.f) r = __builtin_bit_cast(T, (unsigned short)1);
    }
    return r;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// fmaxf drops NaN; a row that holds one has to come out NaN, which the sum of exponentials sees to
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, o));
    return v;
}

}  // namespace pngpd
