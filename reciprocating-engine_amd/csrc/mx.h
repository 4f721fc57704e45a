// mx.h - MXFP4 on the device: e2m1 codes with a power-of-two scale for 32 values.
//
//   m = max |x| of a block        s = the smallest power of two with m / s < 7
//   code = e2m1(x / s), to nearest, ties to the even code
//
// A quotient below 7 rounds to 6 at most, so nothing is clipped; a scale one step
// smaller would clip, one larger would lose a bit. The conversions of gfx950 take the
// scale's exponent byte in the place of a float's exponent, its 0 for 2^-127 and its 255
// for NaN (checked on the card over all bf16 values and scale bytes whose quotient is
// below 7, and over all codes and scale bytes).
#pragma once

#include "common.h"

namespace reng {
namespace mx {

constexpr uint32_t BLOCK = RENG_HIP_MX_BLOCK;
constexpr uint32_t NAN_BYTE = 255, ONE_BYTE = 127;

// Bytes of a row's scales: four blocks a word.
__host__ __device__ constexpr size_t scale_pitch(size_t cols) { return (cols + 127) / 128 * 4; }

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// The scale byte of a block from its largest magnitude's f32 bits (NaN patterns sort above
// infinity's): the exponent of m, one more from 1.75 on, less that of 4.
__device__ __forceinline__ uint32_t scale_byte(uint32_t mbits) {
    if (mbits >= 0x7f800000u) return NAN_BYTE;
    if (mbits == 0) return ONE_BYTE;
    const uint32_t e = (mbits + 0x00200000u) >> 23;
    return e > 2 ? e - 2 : 0;
}

__device__ __forceinline__ float scale_operand(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes of f32 values, in a dword; zeros for a NaN block.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t byte) {
    const float s = scale_operand(byte);
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[0], x[1], s, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[2], x[3], s, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[4], x[5], s, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[6], x[7], s, 3);
    return byte == NAN_BYTE ? 0u : d;
}

// Eight codes as bf16.
__device__ __forceinline__ u32x4_t decode8(uint32_t d, float s) {
    u32x4_t r;
    r.x = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 0));
    r.y = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 1));
    r.z = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 2));
    r.w = __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 3));
    return r;
}

// The largest of a value over the four lanes of an aligned quad.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));   // quad_perm [1, 0, 3, 2]
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));   // quad_perm [2, 3, 0, 1]
}

// The scale bytes of four quads (16 lanes, aligned) as their word, in every lane.
__device__ __forceinline__ uint32_t scale_word(uint32_t byte) {
    uint32_t w = byte << (8 * (threadIdx.x / 4 % 4));
    w |= (uint32_t)__builtin_amdgcn_ds_swizzle((int)w, 0x101f);   // lane ^ 4
    w |= (uint32_t)__builtin_amdgcn_ds_swizzle((int)w, 0x201f);   // lane ^ 8
    return w;
}

}  // namespace mx

// The checks every call that takes a cache makes of it.
int check_mx_cache(const reng_hip_mx_cache *c);

}  // namespace reng
