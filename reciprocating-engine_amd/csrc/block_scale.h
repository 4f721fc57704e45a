// block_scale.h - one fp8 scale for a block of values: the device pieces shared
// by the block quantizer (block_quantize.hip) and the norm that writes its
// output as codes (residual_norm.hip).
//
//   m = max |x| over the block (NaN ignored, infinities counted)
//   s = m / (max_finite * backoff), 1 where that is 0 in f32
//   code = encode(x / s)
//
// which is the per-channel scheme of reng_fp8::quantize_with
// (crates/reng-fp8/src/lib.rs:519-563) with a block in the place of a row, and
// the same bits: the quotient is the IEEE one, the encoder the exact one. (But a
// row there has scale 0, and NaN for its zeros, where m is not 0 and m / full is:
// m up to 2^-150 full, f32's smallest subnormals.)
#pragma once

#include "common.h"

namespace reng {
namespace blk {

constexpr uint32_t BLOCK = 128;   // columns of a block; rows too, in a weight

constexpr uint32_t F32_INF = 0x7f800000u;

// |x|'s bits as the absmax counts them: 0 for NaN.
__device__ __forceinline__ uint32_t mag_no_nan(float x) {
    const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
    return a > F32_INF ? 0u : a;
}

__device__ __forceinline__ float scale_of(uint32_t mbits, float full) {
    const float s = __uint_as_float(mbits) / full;
    return s == 0.0f ? 1.0f : s;
}

// Four codes in a dword. With a normal, finite s the f32 quotient is taken as
// RN32(x * RN64(1 / s)) through f64, which is the IEEE quotient for every finite
// x (quantize.hip proves it) at a fifth of the instructions of a division, and
// v_cvt_pk encodes it after a clamp; other scales, and a quad that holds a NaN,
// take the division and the integer encoder.
struct Encoder {
    float s;
    double r;
    bool fast;
    __device__ __forceinline__ explicit Encoder(float scale)
        : s(scale), r(0.0), fast(scale >= 1.17549435e-38f && scale < __builtin_inff()) {
        if (fast) r = 1.0 / (double)scale;
    }
    // Of a fast scale and four values without a NaN.
    template <int F>
    __device__ __forceinline__ uint32_t quad_fast(float x0, float x1, float x2, float x3) const {
        return cvt4<F, true>((float)((double)x0 * r), (float)((double)x1 * r), (float)((double)x2 * r),
                             (float)((double)x3 * r));
    }
    template <int F>
    __device__ __forceinline__ uint32_t quad(float x0, float x1, float x2, float x3) const {
        const bool nan = __builtin_isnan(x0) | __builtin_isnan(x1) | __builtin_isnan(x2) | __builtin_isnan(x3);
        if (fast && !nan) return quad_fast<F>(x0, x1, x2, x3);
        return encode_div<F>(x0, s) | (encode_div<F>(x1, s) << 8) | (encode_div<F>(x2, s) << 16) |
               (encode_div<F>(x3, s) << 24);
    }
};

// Max over the 16 or 32 lanes (aligned) a lane belongs to.
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        const uint32_t w = (uint32_t)__shfl_xor((int)v, o, 64);
        v = v > w ? v : w;
    }
    return v;
}

}  // namespace blk
}  // namespace reng
