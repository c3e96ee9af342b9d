// Microscaled (MX) blocks: 32 consecutive values of a row share an E8M0 scale byte s (2^(s - 127); 255:
// not a number), elements are E2M1 (4 bits, two per byte, the even column in the low half) or E4M3
// (8 bits).  The formats are those of the OCP Microscaling specification v1.0; gfx950's scaled matrix
// instructions take them as they are.
//
// Storage of R rows of K values: codes [R, kp] elements with kp = K rounded up to 128 (a matrix
// instruction's K and a half cache line of E2M1 codes; the padding holds zero codes), scales [R, sp]
// bytes with sp = 16 per 512 columns, so that a row's scales of four steps of 128 columns are one
// aligned 16-byte load (bytes beyond kp / 32 hold 0).
#pragma once
#include "svdq_common.h"

namespace svdq {

constexpr int MX_E2M1 = 0, MX_E4M3 = 1;

__host__ __device__ constexpr long mx_kp(long K) { return (K + 127) / 128 * 128; }
__host__ __device__ constexpr long mx_sp(long K) { return (K + 511) / 512 * 16; }
__host__ __device__ constexpr long mx_row_bytes(long K, int fmt) { return fmt == MX_E4M3 ? mx_kp(K) : mx_kp(K) / 2; }

// The scale byte of a block whose largest magnitude has the float32 bits `top`: the exponent floor(log2)
// minus the element type's own (2: 6 = 1.5 x 2^2; 8: 448 = 1.75 x 2^8), not below the type's smallest.
// Infinities and NaN (which are >= 0x7F800000 as integers) make the block not a number.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const int e = (int)(top >> 23) - (FMT == MX_E4M3 ? 8 : 2);
  return top >= 0x7F800000u ? 255u : (uint32_t)max(e, 0);
}

// Eight float32 values as E2M1 (one dword) or E4M3 (two dwords) codes under the scale byte s, rounded to
// nearest even, beyond the type's range to its largest value; zero codes in a block that is not a number.
// The conversion reads the scale's exponent field alone, so field 0 is 2^-127.  E2M1 saturates by itself; E4M3
// would give NaN beyond 464 x 2^(s - 127), so values are clamped to 448 x 2^(s - 127) first (exact in float32).
template <int FMT>
__device__ __forceinline__ u32x2 mx_encode8(const float (&v)[8], uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  u32x2 o = {0, 0};
  if (FMT == MX_E2M1) {
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[0], v[1], scale, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[2], v[3], scale, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[4], v[5], scale, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[6], v[7], scale, 3);
    o[0] = d;
  } else {
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    const float most = __uint_as_float(((s + 8) << 23) | 0x600000u);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      i16x2 d = {0, 0};
      d = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(d, __builtin_amdgcn_fmed3f(v[4 * i], -most, most),
                                                   __builtin_amdgcn_fmed3f(v[4 * i + 1], -most, most), scale, false);
      d = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(d, __builtin_amdgcn_fmed3f(v[4 * i + 2], -most, most),
                                                   __builtin_amdgcn_fmed3f(v[4 * i + 3], -most, most), scale, true);
      o[i] = __builtin_bit_cast(uint32_t, d);
    }
  }
  return s == 255u ? u32x2{0, 0} : o;
}

// The largest magnitude (float32 bits; a NaN's pass infinity's) of eight values.
__device__ __forceinline__ uint32_t mx_chunk_top(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return top;
}

// The largest of the four lanes 4 i .. 4 i + 3 that hold a block.
__device__ __forceinline__ uint32_t mx_block_top(uint32_t top) {
  // quad_perm [1, 0, 3, 2], then [2, 3, 0, 1]
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));
  return top;
}

// Chunk c (eight columns from 8 c) of a row into MX blocks: the four lanes of a block call it together.
// top: mx_chunk_top(v).  Chunks beyond kp write only their share of the scales' padding (v is zero there).  PAST: E4M3 codes past the L2.
template <int FMT, bool PAST = false>
__device__ __forceinline__ void mx_store8(const float (&v)[8], uint32_t top, int c, int kp, uint8_t* __restrict__ codes,
                                          uint8_t* __restrict__ scales) {
  const uint32_t s = mx_scale_byte<FMT>(mx_block_top(top));
  const u32x2 o = mx_encode8<FMT>(v, s);
  if (8 * c < kp) {
    if (FMT == MX_E2M1) *reinterpret_cast<uint32_t*>(codes + 4 * c) = o[0];
    else if (PAST) __builtin_nontemporal_store(o, reinterpret_cast<u32x2*>(codes + 8 * c));
    else *reinterpret_cast<u32x2*>(codes + 8 * c) = o;
  }
  if ((c & 3) == 0) scales[c >> 2] = (uint8_t)s;
}

}  // namespace svdq
