// The 8-bit paged cache's number format. A row is the D values of one (token, kv head), keys and values apart; it is held as D
// codes in float8 (e4m3, finite: 448 is the largest, there is no infinity) and one power of two 2^e, kept as the byte e + 127:
//
//   e = the smallest power with max |x| / 2^e <= 448, at least -126;   code = round(x / 2^e), ties to even
//
// A power of two makes every step but the code's rounding exact: the division, the way back (code * 2^e has four significant
// bits), and the scale's way into a product of sums. A code keeps a row's values to 2^-4 of themselves down to 2^-15 of the
// row's largest, so a finer scale than one a row would change little. What is not finite has the code NaN and takes no part in
// the maximum; a row of zeros has e = 0.
//
// A page of the pool: codes [2, Hkv, P * D], keys as rows [P, D], values transposed [D, P]; scales [2, Hkv, P].
#pragma once
#include "common.h"

typedef uint32_t q8x4_t __attribute__((ext_vector_type(4)));      // 16 codes
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// e + 127 for a row whose largest finite value is `amax`: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t q8_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax == 0.f ? 127u : (uint32_t)(max(e, -126) + 127);
}
__device__ __forceinline__ float q8_power(uint32_t byte) { return __uint_as_float(byte << 23); }          // 2^e (byte >= 1)
__device__ __forceinline__ float q8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }  // 2^-e, e <= 120

// What a value counts for in its row's maximum.
__device__ __forceinline__ float q8_size(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}
// The codes of four values already divided by 2^e, lowest byte first.
__device__ __forceinline__ uint32_t q8_codes(float a, float b, float c, float d) {
  const auto kept = [](float v) { return fabsf(v) <= 448.f ? v : __uint_as_float(0x7fc00000u); };
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(kept(a), kept(b), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(kept(c), kept(d), w, true);
  return (uint32_t)w;
}
