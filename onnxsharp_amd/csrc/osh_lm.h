// osh_lm.h -- element types and conversions of the language-model operators
// (osh_norm_quant.hip, osh_block_norm.hip, osh_quant_matmul.hip, osh_int4_matmul.hip,
// osh_window_attn.hip, osh_kv4_attn.hip).
#pragma once

#include "osh_common.h"

namespace osh {

template <int N> struct IntC {
    static constexpr int value = N;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Vec8;
template <> struct Vec8<float> { using type = f32x8; };
template <> struct Vec8<_Float16> { using type = f16x8; };
template <> struct Vec8<__bf16> { using type = bf16x8; };

// Eight neighbouring values at any alignment of whole elements: global memory
// takes 16-byte accesses at every byte address, so one form serves odd widths.
template <typename T>
__device__ __forceinline__ f32x8 load8(const T *p) {
    typename Vec8<T>::type v;
    __builtin_memcpy(&v, p, sizeof(v));
    return __builtin_convertvector(v, f32x8);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, f32x8 f) {
    const typename Vec8<T>::type v = __builtin_convertvector(f, typename Vec8<T>::type);
    __builtin_memcpy(p, &v, sizeof(v));
}

__host__ __device__ constexpr int cdiv(int a, int b) { return a / b + (a % b != 0); }

// An RMS norm's row whose squares leave FP32's range is taken times the power of two that brings the larger of its largest
// |h| and sqrt(eps) (of biased exponent eps_exp) to [1, 2), as far as floats go: y is that of
// the row times it, with eps times its square.
__device__ __forceinline__ float row_shift(float hmax, int eps_exp) {
    const int e = max((int)(__float_as_uint(hmax) >> 23), eps_exp);
    return __uint_as_float((unsigned)min(max(254 - e, 1), 253) << 23);
}
// 1 / sqrt; 0 for a row of zeros without eps, NaN for a row that is not finite.
__device__ __forceinline__ float row_inv(float hmax, float mean, float eps) {
    if (!(hmax < __builtin_inff())) return __builtin_nanf("");
    return mean + eps == 0.0f ? 0.0f : 1.0f / __builtin_sqrtf(mean + eps);
}

// Activations.  EXACT ones are for FP32 outputs: GELU is x erfc(-x / sqrt 2) / 2, since
// 1 + erf cancels below zero (4% off at -5, 0 from -5.6 on).  For 16-bit outputs SiLU takes
// the hardware's reciprocal, and GELU, x - x Q(x) for x > 0 and x Q(-x) below with Q(z) =
// erfc(z / sqrt 2) / 2, a least-maximum fit of erfc(z) e^(z^2) by t P(t), t = 1 / (1 +
// 0.4 z): within 7e-8 of erfc in exact arithmetic, and GELU within 8e-8 in FP32.  Of its own
// size it is 5e-7 off for x > -1, 2e-6 at -3, 3e-5 at -5 (1/16 of f16's half step where f16
// has normal numbers, from -4 up), 5e-4 at -8 and 2e-3 at -12 (1/8 and 1/2 of bf16's).
// erff is 45 instructions a value against 17: 8 us of 1028 x 5120 x 1280.
template <bool EXACT>
__device__ __forceinline__ float apply_act(int act, float v) {
    switch (act) {
    case OSH_ACT_RELU: return v > 0.0f || v != v ? v : 0.0f;
    case OSH_ACT_SILU: {
        const float e = 1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f);
        return EXACT ? v / e : v * __builtin_amdgcn_rcpf(e);
    }
    case OSH_ACT_GELU: {
        if (EXACT) {
            const float c = v < -64.0f ? -64.0f : v;  // -0 from there on, at -infinity too
            return 0.5f * c * erfcf(c * -0.70710678118654752f);
        }
        const float z = __builtin_fabsf(v) * 0.70710678118654752f;
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.4f, z, 1.0f));
        float q = -0.20526915788650513f;
        q = __builtin_fmaf(q, t, 0.7297442555427551f);
        q = __builtin_fmaf(q, t, -0.4045509994029999f);
        q = __builtin_fmaf(q, t, 0.4955560863018036f);
        q = __builtin_fmaf(q, t, 0.15084387362003326f);
        q = __builtin_fmaf(q, t, 0.23367586731910706f);
        q *= t * __builtin_amdgcn_exp2f(z * z * -1.4426950408889634f);
        const float h = 0.5f * __builtin_fminf(__builtin_fabsf(v), 64.0f) * q;  // q is 0 from 64 on
        return v > 0.0f ? v - h : -h;
    }
    default: return v;
    }
}

template <int ACT, bool EXACT>
__device__ __forceinline__ void act8(f32x8 &v) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = apply_act<EXACT>(ACT, v[i]);
}

// Bytes of an element type of the C ABI, 0 if there is no such type.
inline int elem_bytes(int t) {
    switch (t) {
    case OSH_T_F32: return 4;
    case OSH_T_F16: case OSH_T_BF16: return 2;
    case OSH_T_I8: case OSH_T_E4M3: return 1;
    default: return 0;
    }
}

}  // namespace osh
