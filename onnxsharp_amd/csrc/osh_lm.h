// osh_lm.h -- element types and conversions of the language-model operators
// (osh_norm_quant.hip, osh_quant_matmul.hip, osh_window_attn.hip).
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
