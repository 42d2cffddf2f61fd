// Device helpers of the 8-bit floating point operators (e4m3 codes; k_q8_*.hip).
//
// Rows: codes [rows, n], one bf16 scale per row and 128 columns.  Weights:
// codes [E][out][in], one scale (F32, F16 or BF16) per 128 x 128 block.
// A value is code * scale.
#pragma once
#include "device_common.hpp"

namespace moehip {

typedef float f32x4q __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4q __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2q __attribute__((ext_vector_type(2)));

constexpr float kQ8Top = 448.0f;              // the largest e4m3 value
constexpr float kQ8Least = 1.17549435e-38f;   // 2^-126: the smallest scale

// |x| as an order-preserving word in which NaN is above infinity, so that a
// maximum of words keeps a NaN (a maximum of floats drops it).
__device__ __forceinline__ uint32_t abs_word(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// F32 to bf16 bits, nearest even; NaN stays NaN.
__device__ __forceinline__ uint32_t bf16_bits(float x) {
    const uint32_t b = __float_as_uint(x);
    return abs_word(x) > 0x7f800000u ? (b >> 16) | 0x40u : (b + 0x7fffu + ((b >> 16) & 1u)) >> 16;
}

// The maximum over each aligned row of 16 lanes, all of which are active.
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = max(v, dpp_u<kDppQuad1>(v));
    v = max(v, dpp_u<kDppQuad2>(v));
    v = max(v, dpp_u<kDppHalfMirror>(v));
    return max(v, dpp_u<kDppMirror>(v));
}

// The stored scale of 128 values whose largest magnitude (abs_word) is `top`.
// A group that holds an infinity or a NaN gets a scale of infinity or NaN, so
// each of its values reads back as NaN (0 * inf, NaN * inf).
__device__ __forceinline__ uint32_t q8_scale_bits(uint32_t top) {
    const float s = __uint_as_float(top) / kQ8Top;
    return bf16_bits(s < kQ8Least ? kQ8Least : s);
}
// Four values as e4m3 codes (nearest even; r: 1 / scale).  |v| * r is at most
// 448 * (1 + 2^-8), which rounds to 448.
__device__ __forceinline__ uint32_t q8_codes4(float a, float b, float c, float d, float r) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a * r, b * r, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * r, d * r, v, true);
}

}  // namespace moehip
