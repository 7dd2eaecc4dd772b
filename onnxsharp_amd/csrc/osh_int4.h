// osh_int4.h -- matrix instructions, direct copies to LDS, and codes of 4 bits as they take them.
#pragma once

#include "osh_lm.h"

namespace osh {

template <typename T> struct Half8;
template <> struct Half8<_Float16> { using type = f16x8; };
template <> struct Half8<__bf16> { using type = bf16x8; };
// FP32 rows are multiplied as three bf16 pieces
template <> struct Half8<float> { using type = bf16x8; };

__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// N bytes (4 or 16) a lane from `from` to LDS: lane i's to dst + N i.
template <int N = 16>
__device__ __forceinline__ void copy_to_lds(const void *from, unsigned char *dst) {
    const auto *src = (const __attribute__((address_space(1))) void *)from;
    auto *to = (__attribute__((address_space(3))) void *)dst;
    static_assert(N == 4 || N == 16);
    if constexpr (N == 4) __builtin_amdgcn_global_load_lds(src, to, 4, 0, 0);
    else __builtin_amdgcn_global_load_lds(src, to, 16, 0, 0);
}
// 16 bytes of LDS, read as four words: a read that may be of any type would wait for all
// direct copies in flight.
template <typename H8>
__device__ __forceinline__ H8 lds_chunk(const unsigned char *at) {
    const unsigned *u = static_cast<const unsigned *>(__builtin_assume_aligned(at, 16));
    const unsigned w[4] = {u[0], u[1], u[2], u[3]};
    return __builtin_bit_cast(H8, w);
}

// The codes of a word, 0..15 each, times a power of two, as 16-bit floats: those at even
// places (0, 2, 4, 6), then those at odd ones.  A byte 0..15 is code * 2^-9 as e4m3 (its
// subnormal numbers and the first binade lie evenly), so that the hardware's conversion, two a
// time and at full rate, does it: 7 instructions for 8 codes.  times512: 512 times the power.
__device__ __forceinline__ void codes8(unsigned w, f16x8 &v, float times512 = 512.0f) {
    const int b[2] = {(int)(w & 0x0f0f0f0fu), (int)(w >> 4 & 0x0f0f0f0fu)};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 p = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b[h], times512, false));
        const f16x2 q = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b[h], times512, true));
        v[4 * h] = p[0], v[4 * h + 1] = p[1], v[4 * h + 2] = q[0], v[4 * h + 3] = q[1];
    }
}
__device__ __forceinline__ void codes8(unsigned w, bf16x8 &v, float times512 = 512.0f) {
    const int b[2] = {(int)(w & 0x0f0f0f0fu), (int)(w >> 4 & 0x0f0f0f0fu)};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        const bf16x2 p = __builtin_bit_cast(bf16x2, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[h], times512, false));
        const bf16x2 q = __builtin_bit_cast(bf16x2, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b[h], times512, true));
        v[4 * h] = p[0], v[4 * h + 1] = p[1], v[4 * h + 2] = q[0], v[4 * h + 3] = q[1];
    }
}
// The same less z, a whole number up to 15: exact in bf16 too.  20 instructions for 8 codes.
__device__ __forceinline__ void codes8_less(unsigned w, float z, bf16x8 &v) {
    const int b[2] = {(int)(w & 0x0f0f0f0fu), (int)(w >> 4 & 0x0f0f0f0fu)};
    f32x8 f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 p = __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b[h], 512.0f, false));
        const f32x2 q = __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b[h], 512.0f, true));
        f[4 * h] = p[0] - z, f[4 * h + 1] = p[1] - z, f[4 * h + 2] = q[0] - z, f[4 * h + 3] = q[1] - z;
    }
    v = __builtin_convertvector(f, bf16x8);
}

}  // namespace osh
