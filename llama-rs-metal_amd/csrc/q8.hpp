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
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
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
// each of its values reads back as NaN (0 * inf, NaN * inf).  The quotient of the
// product with 1/448 and one correction is the division's for every finite `top`
// whose quotient is kQ8Least or more.
__device__ __forceinline__ uint32_t q8_scale_bits(uint32_t top) {
    const float x = __uint_as_float(top), q = x * (1.0f / kQ8Top);
    const float s = fmaf(fmaf(-q, kQ8Top, x), 1.0f / kQ8Top, q);
    return bf16_bits(x < kQ8Least * kQ8Top ? kQ8Least : top >= 0x7f800000u ? x : s);
}
// 1 / scale, within 2^-23 of it (a scale is at least 2^-126)
__device__ __forceinline__ float q8_inverse(uint32_t sb) { return __builtin_amdgcn_rcpf(bf16_to_f32(sb)); }
// Four quotients v / scale as e4m3 codes (nearest even).  They are at most
// 448 * (1 + 2^-8), which rounds to 448.
__device__ __forceinline__ uint32_t q8_codes4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
// Four values, r = 1 / scale: each product is within 2^-22 of the quotient.  For
// values that are seen in 8 bits only, and are further off than that themselves.
__device__ __forceinline__ uint32_t q8_codes4(float a, float b, float c, float d, float r) {
    return q8_codes4(a * r, b * r, c * r, d * r);
}

}  // namespace moehip
