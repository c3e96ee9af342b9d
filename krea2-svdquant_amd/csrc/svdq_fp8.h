// 8-bit floating point with a scale per block: E4M3 codes (OCP, largest value 448, 0x7F not a number, no infinity) and
// float32 scales.  A block's scale is the smallest power of two from 2^-126 under which its largest finite magnitude is at
// most 448: E4M3 keeps its relative precision over 2^15, so a scale of 24 bits would gain nothing, and under a power of two each
// value is rounded once and a code read back is exact in bf16.  Values that are not finite become the code that is not a number, and
// say nothing about the scale.
#pragma once
#include "svdq_common.h"

namespace svdq {

__host__ __device__ constexpr long fp8_kp(long K) { return (K + 127) / 128 * 128; }

// The float32 bits of |v|, 0 where v is not finite.
__device__ __forceinline__ uint32_t fp8_magnitude(float v) {
  const uint32_t a = __float_as_uint(v) & 0x7FFFFFFFu;
  return a >= 0x7F800000u ? 0u : a;
}

// The scale of a block whose largest magnitude has the float32 bits `top`: 448 = 1.75 x 2^8, so a mantissa above 1.75 takes
// the next power.
__device__ __forceinline__ float fp8_scale(uint32_t top) {
  const int e = (int)((top + 0x1FFFFFu) >> 23) - 8;
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// Four values as E4M3 codes under a power-of-two scale, to nearest even.
__device__ __forceinline__ uint32_t fp8_encode4(float a, float b, float c, float d, float scale) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  i16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, r);
}

// Four bf16 values of two registers as E4M3 codes under a power-of-two scale, to nearest even.
__device__ __forceinline__ uint32_t fp8_encode_bf16x4(uint32_t lo, uint32_t hi, float scale) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  i16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, lo), scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, hi), scale, true);
  return __builtin_bit_cast(uint32_t, r);
}

// Eight codes as bf16 (exact).
__device__ __forceinline__ u32x4 fp8_to_bf16x8(uint32_t lo, uint32_t hi) {
  u32x4 o;
  o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
  o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
  o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
  o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  return o;
}

}  // namespace svdq
