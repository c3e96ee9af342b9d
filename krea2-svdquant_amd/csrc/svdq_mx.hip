// Into MX blocks and back: quantising a bf16 activation, the SwiGLU product and the block's adaptive RMS norm
// (with the gated residual ahead of it) with their results in MX blocks, and reading blocks back as bf16.
//
//   block of 32 values:  s = max(floor(log2(max |v|)) - E, -127)   (E = 2: E2M1, 8: E4M3)
//                        q = the element type's nearest value to v / 2^s, ties to even, saturating
//
// The values v are float32 here (a bf16 input as it is; the norm's and the product's results are not rounded to
// bf16 first), so each value is rounded once.  All of these passes are HBM-bound: one read of the inputs, one
// write of the codes.  A lane holds 8 consecutive columns (one 16-byte load), the four lanes of a block find
// its largest magnitude by two quad permutes and write 4 (E2M1) or 8 (E4M3) bytes of codes each, so loads and
// stores of a wave are contiguous.
#include "svdq_kernels.h"
#include "svdq_mx.h"

namespace svdq {
namespace {

__device__ __forceinline__ u32x4 ld16(const void* p) { return *reinterpret_cast<const u32x4*>(p); }

__device__ __forceinline__ void unpack8(u32x4 r, float (&v)[8]) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    v[2 * d] = bf16lo(r[d]);
    v[2 * d + 1] = bf16hi(r[d]);
  }
}

// Columns 8 c .. 8 c + 7 of a row of K bf16 values, zeros beyond K.  VEC: rows start on 16 bytes and K % 8 == 0.
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t* __restrict__ row, int c, int K, float (&v)[8]) {
  if (VEC) {
    unpack8(8 * c < K ? ld16(row + 8 * c) : u32x4{}, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 8 * c + i < K ? bf16f(row[8 * c + i]) : 0.0f;
  }
}

// silu(g) u = g u / (1 + exp(-g)) in float32 for g >= -87.  exp(-g) = 2^t, t = -g log2(e) as the rounded product t0 and
// what it and the rounded constant leave, 2^t = 2^t0 (1 + ln(2) (t - t0)), within 1.5 units of 2^-23; the reciprocal of
// 1 + exp(-g) by v_rcp_f32 and one Newton step; g u is exact unless it overflows, so the result rounds once more.  Few
// instructions, because the pass is close to being bound by them: with expf and the correctly rounded quotient M = 4352,
// K = 16384, E4M3 took 74.9 us, so 65.4 with the check for the range's ends below (62.9 without).  Above g = 87 the exponent is held there: 1 + exp(-g) is 1.
__device__ __forceinline__ float silu_factor(float g) {   // 1 / (1 + exp(-g))
  const float c = __builtin_amdgcn_fmed3f(g, -87.0f, 87.0f);
  const float t0 = c * -1.44269502f;
  const float rest = __builtin_fmaf(c, -1.92596303e-8f, __builtin_fmaf(c, -1.44269502f, -t0));
  const float e0 = __builtin_amdgcn_exp2f(t0), e = __builtin_fmaf(e0, 0.693147181f * rest, e0);
  const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.0f), r);
}

// The same product for every g and u, by way of u's exponent: u = m 2^x, g m is of ordinary size.  Below g = -87,
// 1 / (1 + exp(-g)) is exp(g) to 2^-125 = 2^t0 as above, t0 = n + f with the whole n into the exponent; below -10000 the result is
// 0 as there.
__device__ __forceinline__ float silu_mul_any(float g, float u) {
  const float m = __builtin_amdgcn_frexp_mantf(u);
  const int x = __builtin_amdgcn_frexp_expf(u);
  const float c = fmaxf(g, -10000.0f), t0 = c * 1.44269502f, n = rintf(t0);
  const float rest = __builtin_fmaf(c, 1.92596303e-8f, __builtin_fmaf(c, 1.44269502f, -t0));
  const float e0 = __builtin_amdgcn_exp2f(t0 - n), e = __builtin_fmaf(e0, 0.693147181f * rest, e0);
  const bool far = g < -87.0f;
  return ldexpf(g * m * (far ? e : silu_factor(g)), (far ? (int)n : 0) + x);
}

// v[i] = silu(v[i]) u[i]; returns mx_chunk_top(v).  The longer way round only where a gate is below -87 or a product left
// float32's range.
__device__ __forceinline__ uint32_t silu_mul8(float (&v)[8], const float (&u)[8]) {
  float least = 0.0f, y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = v[i] * u[i] * silu_factor(v[i]);
    least = fminf(least, v[i]);
  }
  uint32_t top = mx_chunk_top(y);
  if (__builtin_expect(least < -87.0f || top >= 0x7F800000u, 0)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = silu_mul_any(v[i], u[i]);
    top = mx_chunk_top(y);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = y[i];
  return top;
}

// A wave takes units of 64 chunks (512 columns: 16 bytes of scales) of one row, UNITS of them at a time, whose loads are
// all under way before the first is used; rows and columns are wave-uniform (scalar) arithmetic.
// GATE: the SwiGLU product silu(x) * u, else x itself.
template <int FMT, bool VEC, bool GATE, int UNITS>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const uint16_t* __restrict__ x, long ldx,
                                                          const uint16_t* __restrict__ u, long ldu, long units, int K,
                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int kp = (int)mx_kp(K), sp = (int)mx_sp(K), per_row = sp / 16, lane = threadIdx.x & 63;
  const long first = ((long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * UNITS;
  float v[UNITS][8], w[UNITS][8];
  long row = first / per_row;
  int part = (int)(first - row * per_row);
  const long row0 = row;
  const int part0 = part;
  auto next = [&] {
    if (++part == per_row) {
      part = 0;
      ++row;
    }
  };
#pragma unroll
  for (int i = 0; i < UNITS; ++i, next())
    if (first + i < units) {
      load8<VEC>(x + row * ldx, 64 * part + lane, K, v[i]);
      if (GATE) load8<VEC>(u + row * ldu, 64 * part + lane, K, w[i]);
    }
  row = row0;
  part = part0;
#pragma unroll
  for (int i = 0; i < UNITS; ++i, next())
    if (first + i < units) {
      const int c = 64 * part + lane;
      const uint32_t top = GATE ? silu_mul8(v[i], w[i]) : mx_chunk_top(v[i]);   // columns beyond K: 0 times 0
      mx_store8<FMT>(v[i], top, c, kp, codes + row * mx_row_bytes(K, FMT), scales + row * sp);
    }
}

// Codes and scales back to bf16 [M, K]: code times 2^(s - 127), exact in bf16 but for values below its normal range.  A wave
// takes units of 64 chunks as above; a lane's eight codes are converted under their scale by four instructions.
template <int FMT, bool VEC, int UNITS>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, long units, int K,
                                                            uint16_t* __restrict__ y) {
  const int sp = (int)mx_sp(K), per_row = sp / 16, lane = threadIdx.x & 63;
  const long first = ((long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * UNITS;
  u32x2 q[UNITS];
  uint32_t s[UNITS];
  long row = first / per_row;
  int part = (int)(first - row * per_row);
  const long row0 = row;
  const int part0 = part;
  auto next = [&] {
    if (++part == per_row) {
      part = 0;
      ++row;
    }
  };
#pragma unroll
  for (int i = 0; i < UNITS; ++i, next()) {
    const int c = 64 * part + lane;
    q[i] = u32x2{0, 0};
    s[i] = 0;
    if (first + i < units && 8 * c < K) {
      const uint8_t* src = codes + row * mx_row_bytes(K, FMT);
      if (FMT == MX_E2M1) q[i][0] = *reinterpret_cast<const uint32_t*>(src + 4 * c);
      else q[i] = *reinterpret_cast<const u32x2*>(src + 8 * c);
      s[i] = scales[row * sp + (c >> 2)];
    }
  }
  row = row0;
  part = part0;
#pragma unroll
  for (int i = 0; i < UNITS; ++i, next()) {
    const int c = 64 * part + lane;
    if (first + i >= units || 8 * c >= K) continue;
    const float scale = __uint_as_float(s[i] << 23);
    u32x4 o;
    if (FMT == MX_E2M1) {
      o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[i][0], scale, 0));
      o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[i][0], scale, 1));
      o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[i][0], scale, 2));
      o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[i][0], scale, 3));
    } else {
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        o[2 * d] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i][d], scale, false));
        o[2 * d + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i][d], scale, true));
      }
    }
    if (s[i] == 255u) o = u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
    uint16_t* dst = y + row * K + 8 * c;
    if (VEC) {
      *reinterpret_cast<u32x4*>(dst) = o;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (8 * c + k < K) dst[k] = (uint16_t)(o[k / 2] >> (16 * (k % 2)));
    }
  }
}

// v as a float32 that rounds to fewer bits as v itself does: where v lies between two float32 values, the odd one.
__device__ __forceinline__ float to_odd(double v) {
  const float r = (float)v;
  const double back = (double)r;
  const uint32_t bits = __float_as_uint(r);
  if (back == v || (bits & 1) || !(fabsf(r) < __builtin_inff())) return r;
  return __uint_as_float(fabs(v) > fabs(back) ? bits + 1 : bits - 1);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Adaptive RMS norm into MX blocks, one 256-thread workgroup per row of H (H % 8 == 0):
//   RES: xo = bf16(x + g v) (one rounding; written, and the row that is normalized), else xo = x
//   y = xo rsqrt(mean(xo^2) + eps) w + shift, quantised from the exact value
// A value near the middle of two codes takes the other one for an error in its last bits, and the whole row shares its
// mean: the mean is summed in 64 bits, its root's reciprocal kept as r0 + r1, xo w (with a power of two) is exact (but for
// values under 2^-126 of the row's root mean square), and y = (xo w) r0 + shift + (xo w) r1 by two fused products, within one unit in its
// last place.  Codes and scales change only at values whose last 19 bits are zero, so a chunk with a value at most one
// unit from such (three in 2^19 of them) is evaluated again in 64 bits and rounded to odd: codes and scales are those
// of the exact y to 2^-46 of its terms.  On float32's y alone 324 of 6.4e8 codes (24 inputs of 4352 x 6144, E4M3)
// were the neighbours'; with the whole formula in float32 733.
// Thread t takes chunks t, t + 256, ...: the first NR stay in registers between the passes, those beyond are read
// again (RES: from xo, written by the same thread).  HBM-bound: RES, 3.03 (E4M3) or 2.53 bytes a value beside x and v.
// NR is the row's own count, so that short rows keep few registers, and stores of what is not read again here go past
// the L2: M = 4352, H = 6144, RES, E4M3, on inputs that the cache in front of HBM holds 39.7 -> 30.8 us; on inputs from
// HBM (eight sets in turn) 39.4 us, 39.7 with the values next to borders in 64 bits, 4.7 TB/s (T = 128 4.7 and 4.9).
// xo may be x, so neither is restrict: each thread reads a chunk of x before it writes that chunk of xo.
template <int FMT, int NR, bool RES>
__global__ void __launch_bounds__(256) rms_norm_mx_kernel(const uint16_t* x, long ldx, const uint16_t* __restrict__ v,
                                                          long ldv, const uint16_t* __restrict__ g,
                                                          const uint16_t* __restrict__ w,
                                                          const uint16_t* __restrict__ shift, int H, float eps,
                                                          uint16_t* xo, long ldxo, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  __shared__ double part[4];
  const int tid = threadIdx.x, nc = H / 8, kp = (int)mx_kp(H), sp = (int)mx_sp(H);
  const uint16_t* xr = x + (long)blockIdx.x * ldx;
  uint16_t* xor_ = RES ? xo + (long)blockIdx.x * ldxo : nullptr;
  auto row_chunk = [&](int c, bool again) {   // again: the chunk will be read again
    u32x4 r = ld16(xr + 8 * c);
    if (RES) {
      const u32x4 gv = ld16(g + 8 * c), vv = ld16(v + (long)blockIdx.x * ldv + 8 * c);
#pragma unroll
      for (int d = 0; d < 4; ++d)
        r[d] = pack_bf16x2(__builtin_fmaf(bf16lo(gv[d]), bf16lo(vv[d]), bf16lo(r[d])),
                           __builtin_fmaf(bf16hi(gv[d]), bf16hi(vv[d]), bf16hi(r[d])));
      if (again) *reinterpret_cast<u32x4*>(xor_ + 8 * c) = r;
      else __builtin_nontemporal_store(r, reinterpret_cast<u32x4*>(xor_ + 8 * c));
    }
    return r;
  };
  double ss = 0.0;
  auto add = [&](u32x4 r) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const double a = bf16lo(r[d]), b = bf16hi(r[d]);
      ss = __builtin_fma(a, a, ss);
      ss = __builtin_fma(b, b, ss);
    }
  };
  u32x4 keep[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int c = tid + 256 * i;
    keep[i] = c < nc ? row_chunk(c, false) : u32x4{};
    add(keep[i]);
  }
  for (int c = tid + 256 * NR; c < nc; c += 256) add(row_chunk(c, true));
  ss = wave_sum(ss);
  if ((tid & 63) == 0) part[tid >> 6] = ss;
  __syncthreads();
  const double mean = (part[0] + part[1] + part[2] + part[3]) / (double)H + (double)eps;
  // The root's reciprocal as 2^k (r0 + r1), so that x 2^k w is of ordinary size whatever the row's.  k within -126 .. 127: rows
  // of bf16 subnormals without eps have reciprocals up to 2^148, whose rest r0 and r1 take (r0 in [1, 2) otherwise).
  const double root = rsqrt(mean);
  const float pow2 = fminf(fmaxf(__uint_as_float(__float_as_uint((float)root) & 0x7F800000u), 0x1p-126f), 0x1p127f);
  const double scaled = root / (double)pow2;
  const float r0 = (float)scaled, r1 = (float)(scaled - (double)r0);
  uint8_t* crow = codes + (long)blockIdx.x * mx_row_bytes(H, FMT);
  uint8_t* srow = scales + (long)blockIdx.x * sp;
  auto put = [&](int c, u32x4 raw) {
    float f[8] = {};
    if (c < nc) {
      float wv[8], sv[8];
      uint32_t least = ~0u;
      unpack8(raw, f);
      unpack8(ld16(w + 8 * c), wv);
      unpack8(ld16(shift + 8 * c), sv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = f[i] * pow2 * wv[i];
        f[i] = __builtin_fmaf(t, r1, __builtin_fmaf(t, r0, sv[i]));
        least = min(least, (__float_as_uint(f[i]) + 1) << 13);
      }
      if (__builtin_expect(least <= 2u << 13, 0)) {
        unpack8(raw, f);
        unpack8(ld16(w + 8 * c), wv);
        unpack8(ld16(shift + 8 * c), sv);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_odd(__builtin_fma((double)(f[i] * pow2 * wv[i]), scaled, (double)sv[i]));
      }
    }
    mx_store8<FMT, true>(f, mx_chunk_top(f), c, kp, crow, srow);
  };
  // 4 sp chunks a row, the scales' padding included; 4 sp % 64 == 0, so a wave's lanes are in or out together
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int c = tid + 256 * i;
    if (c < 4 * sp) put(c, keep[i]);
  }
  for (int c = tid + 256 * NR; c < 4 * sp; c += 256)
    put(c, c < nc ? ld16((RES ? xor_ : xr) + 8 * c) : u32x4{});
}

template <int FMT, bool GATE, int UNITS>
hipError_t quantize_by(bool vec, const uint16_t* x, long ldx, const uint16_t* u, long ldu, long units, int K,
                       uint8_t* codes, uint8_t* scales, hipStream_t st) {
  const long blocks = (units + 4 * UNITS - 1) / (4 * UNITS);
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  if (vec)
    mx_quantize_kernel<FMT, true, GATE, UNITS><<<(unsigned)blocks, 256, 0, st>>>(x, ldx, u, ldu, units, K, codes, scales);
  else
    mx_quantize_kernel<FMT, false, GATE, UNITS><<<(unsigned)blocks, 256, 0, st>>>(x, ldx, u, ldu, units, K, codes, scales);
  return hipGetLastError();
}

template <int FMT, bool GATE>
hipError_t quantize(const uint16_t* x, long ldx, const uint16_t* u, long ldu, long M, int K, uint8_t* codes,
                    uint8_t* scales, hipStream_t st) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | (GATE ? reinterpret_cast<uintptr_t>(u) : 0);
  const bool vec = at % 16 == 0 && ldx % 8 == 0 && (!GATE || ldu % 8 == 0) && K % 8 == 0;
  const long units = M * (mx_sp(K) / 16);
  // Two units a wave where there are waves enough: M = 4352, K = 6144 and 16384, E4M3, 1 / 2 / 4 units: quantising 14.8 13.9
  // 14.8 and 40.6 35.3 38.8 us, the SwiGLU product (before it looked for the range's ends) 21.4 23.9 - and 62.0 66.1 -.
  // Between 8000 and 25000 units one and two differ by 3% either way (K = 6144, E2M1, 1 / 2 units: 8196 units 3.54 3.59, 12288
  // 4.55 4.42, 16392 5.24 5.33, 24576 7.09 7.09, 32772 10.59 10.31, 52224 15.91 14.93; reading back the same).
  if (!GATE && units >= 16384) return quantize_by<FMT, GATE, 2>(vec, x, ldx, u, ldu, units, K, codes, scales, st);
  return quantize_by<FMT, GATE, 1>(vec, x, ldx, u, ldu, units, K, codes, scales, st);
}

template <int FMT, bool RES, class... A>
hipError_t norm(int T, int H, hipStream_t st, A... a) {
  switch ((int)((4 * mx_sp(H) + 255) / 256)) {   // the row's chunks per thread
    case 1: rms_norm_mx_kernel<FMT, 1, RES><<<T, 256, 0, st>>>(a...); break;
    case 2: rms_norm_mx_kernel<FMT, 2, RES><<<T, 256, 0, st>>>(a...); break;
    case 3: rms_norm_mx_kernel<FMT, 3, RES><<<T, 256, 0, st>>>(a...); break;
    case 4: rms_norm_mx_kernel<FMT, 4, RES><<<T, 256, 0, st>>>(a...); break;
    case 5: rms_norm_mx_kernel<FMT, 5, RES><<<T, 256, 0, st>>>(a...); break;
    case 6: rms_norm_mx_kernel<FMT, 6, RES><<<T, 256, 0, st>>>(a...); break;
    default: rms_norm_mx_kernel<FMT, 8, RES><<<T, 256, 0, st>>>(a...);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_quantize(const uint16_t* x, long ldx, long M, int K, int fmt, uint8_t* codes, uint8_t* scales,
                              hipStream_t st) {
  return fmt == MX_E4M3 ? quantize<MX_E4M3, false>(x, ldx, nullptr, 0, M, K, codes, scales, st)
                        : quantize<MX_E2M1, false>(x, ldx, nullptr, 0, M, K, codes, scales, st);
}

hipError_t launch_silu_mul_mx(const uint16_t* g, long ldg, const uint16_t* u, long ldu, long M, int K, int fmt,
                              uint8_t* codes, uint8_t* scales, hipStream_t st) {
  return fmt == MX_E4M3 ? quantize<MX_E4M3, true>(g, ldg, u, ldu, M, K, codes, scales, st)
                        : quantize<MX_E2M1, true>(g, ldg, u, ldu, M, K, codes, scales, st);
}

template <int FMT, int UNITS>
static hipError_t dequantize_by(const uint8_t* codes, const uint8_t* scales, long units, int K, uint16_t* y,
                                hipStream_t st) {
  const long blocks = (units + 4 * UNITS - 1) / (4 * UNITS);
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  if (K % 8 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0)
    mx_dequantize_kernel<FMT, true, UNITS><<<(unsigned)blocks, 256, 0, st>>>(codes, scales, units, K, y);
  else
    mx_dequantize_kernel<FMT, false, UNITS><<<(unsigned)blocks, 256, 0, st>>>(codes, scales, units, K, y);
  return hipGetLastError();
}

template <int FMT>
static hipError_t dequantize(const uint8_t* codes, const uint8_t* scales, long M, int K, uint16_t* y, hipStream_t st) {
  const long units = M * (mx_sp(K) / 16);
  return units >= 16384 ? dequantize_by<FMT, 2>(codes, scales, units, K, y, st)
                        : dequantize_by<FMT, 1>(codes, scales, units, K, y, st);
}

hipError_t launch_mx_dequantize(const uint8_t* codes, const uint8_t* scales, long M, int K, int fmt, uint16_t* y,
                                hipStream_t st) {
  return fmt == MX_E4M3 ? dequantize<MX_E4M3>(codes, scales, M, K, y, st) : dequantize<MX_E2M1>(codes, scales, M, K, y, st);
}

hipError_t launch_rms_norm_mx(const uint16_t* x, long ldx, const uint16_t* v, long ldv, const uint16_t* g,
                              const uint16_t* w, const uint16_t* shift, int T, int H, float eps, int fmt, uint16_t* xo,
                              long ldxo, uint8_t* codes, uint8_t* scales, hipStream_t st) {
  if (v)
    return fmt == MX_E4M3
               ? norm<MX_E4M3, true>(T, H, st, x, ldx, v, ldv, g, w, shift, H, eps, xo, ldxo, codes, scales)
               : norm<MX_E2M1, true>(T, H, st, x, ldx, v, ldv, g, w, shift, H, eps, xo, ldxo, codes, scales);
  return fmt == MX_E4M3
             ? norm<MX_E4M3, false>(T, H, st, x, ldx, v, ldv, g, w, shift, H, eps, xo, ldxo, codes, scales)
             : norm<MX_E2M1, false>(T, H, st, x, ldx, v, ldv, g, w, shift, H, eps, xo, ldxo, codes, scales);
}

}  // namespace svdq
