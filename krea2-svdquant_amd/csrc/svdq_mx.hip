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

// silu(g) u = g u / (1 + exp(-g)) in float32.  exp(-g) overflows to infinity for g < -88.7, where the quotient is -0
// as it should be to float32's smallest normal; g = -infinity gives NaN (as in torch's float32 formula).
__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// One thread per chunk of 8 columns, sp * 4 chunks a row (the scales' padding included).  A workgroup takes 256
// consecutive chunks of the row-major list, its first one's row by one uniform 64-bit division.
// GATE: the SwiGLU product silu(x) * u, else x itself.
template <int FMT, bool VEC, bool GATE>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const uint16_t* __restrict__ x, long ldx,
                                                          const uint16_t* __restrict__ u, long ldu, long M, int K,
                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int kp = (int)mx_kp(K), sp = (int)mx_sp(K), per_row = 4 * sp;
  const long first = (long)blockIdx.x * 256;
  const long row0 = first / per_row;
  const uint32_t in = (uint32_t)(first - row0 * per_row) + threadIdx.x;
  const long row = row0 + in / (uint32_t)per_row;
  const int c = (int)(in % (uint32_t)per_row);
  if (row >= M) return;   // per_row % 64 == 0: the four lanes of a block leave together
  float v[8];
  load8<VEC>(x + row * ldx, c, K, v);
  if (GATE) {
    float w[8];
    load8<VEC>(u + row * ldu, c, K, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 8 * c + i < K ? silu_mul(v[i], w[i]) : 0.0f;
  }
  mx_store8<FMT>(v, c, kp, codes + row * mx_row_bytes(K, FMT), scales + row * sp);
}

// Eight E2M1 or E4M3 codes as float32, without their scale.
template <int FMT>
__device__ __forceinline__ void decode8(u32x2 q, float (&v)[8]) {
  if (FMT == MX_E2M1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = (q[0] >> (4 * i)) & 7u;
      // 0, 0.5, 1, 1.5, 2, 3, 4, 6: exponent m / 2, mantissa bit m % 2; the first two are 0 and 0.5
      const float a = m < 2 ? 0.5f * m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
      v[i] = __uint_as_float(__float_as_uint(a) | ((q[0] >> (4 * i + 3)) & 1u) << 31);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], true);
      v[4 * i] = a[0];
      v[4 * i + 1] = a[1];
      v[4 * i + 2] = b[0];
      v[4 * i + 3] = b[1];
    }
  }
}

// Codes and scales back to bf16 [M, K]: code times 2^(s - 127), exact in bf16 but for values below its normal range.
template <int FMT, bool VEC>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, long M, int K,
                                                            uint16_t* __restrict__ y) {
  const int per_row = (K + 7) / 8;
  const long first = (long)blockIdx.x * 256;
  const long row0 = first / per_row;
  const uint32_t in = (uint32_t)(first - row0 * per_row) + threadIdx.x;
  const long row = row0 + in / (uint32_t)per_row;
  const int c = (int)(in % (uint32_t)per_row);
  if (row >= M) return;
  const uint8_t* src = codes + row * mx_row_bytes(K, FMT);
  u32x2 q = {0, 0};
  if (FMT == MX_E2M1) q[0] = *reinterpret_cast<const uint32_t*>(src + 4 * c);
  else q = *reinterpret_cast<const u32x2*>(src + 8 * c);
  const uint32_t s = scales[row * mx_sp(K) + (c >> 2)];
  float v[8];
  decode8<FMT>(q, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = s == 255u ? __builtin_nanf("") : ldexpf(v[i], (int)s - 127);
  uint16_t* dst = y + row * K + 8 * c;
  u32x4 o;
#pragma unroll
  for (int d = 0; d < 4; ++d) o[d] = pack_bf16x2(v[2 * d], v[2 * d + 1]);
  if (VEC) {
    *reinterpret_cast<u32x4*>(dst) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * c + i < K) dst[i] = (uint16_t)(o[i / 2] >> (16 * (i % 2)));
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Adaptive RMS norm into MX blocks, one 256-thread workgroup per row of H (H % 8 == 0):
//   RES: xo = bf16(x + g v) (one rounding; written, and the row that is normalized), else xo = x
//   y = xo rsqrt(mean(xo^2) + eps) w + shift in float32, quantised
// Thread t takes chunks t, t + 256, ...: the first NR stay in registers between the passes, those beyond are read
// again (RES: from xo, written by the same thread).
template <int FMT, int NR, bool RES>
__global__ void __launch_bounds__(256) rms_norm_mx_kernel(const uint16_t* __restrict__ x, long ldx,
                                                          const uint16_t* __restrict__ v, long ldv,
                                                          const uint16_t* __restrict__ g, const uint16_t* __restrict__ w,
                                                          const uint16_t* __restrict__ shift, int H, float eps,
                                                          uint16_t* __restrict__ xo, long ldxo,
                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  __shared__ float part[4];
  const int tid = threadIdx.x, nc = H / 8, kp = (int)mx_kp(H), sp = (int)mx_sp(H);
  const uint16_t* xr = x + (long)blockIdx.x * ldx;
  uint16_t* xor_ = RES ? xo + (long)blockIdx.x * ldxo : nullptr;
  auto row_chunk = [&](int c) {
    u32x4 r = ld16(xr + 8 * c);
    if (RES) {
      const u32x4 gv = ld16(g + 8 * c), vv = ld16(v + (long)blockIdx.x * ldv + 8 * c);
#pragma unroll
      for (int d = 0; d < 4; ++d)
        r[d] = pack_bf16x2(__builtin_fmaf(bf16lo(gv[d]), bf16lo(vv[d]), bf16lo(r[d])),
                           __builtin_fmaf(bf16hi(gv[d]), bf16hi(vv[d]), bf16hi(r[d])));
      *reinterpret_cast<u32x4*>(xor_ + 8 * c) = r;
    }
    return r;
  };
  float ss = 0.0f;
  auto add = [&](u32x4 r) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      ss = __builtin_fmaf(bf16lo(r[d]), bf16lo(r[d]), ss);
      ss = __builtin_fmaf(bf16hi(r[d]), bf16hi(r[d]), ss);
    }
  };
  u32x4 keep[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int c = tid + 256 * i;
    keep[i] = c < nc ? row_chunk(c) : u32x4{};
    add(keep[i]);
  }
  for (int c = tid + 256 * NR; c < nc; c += 256) add(row_chunk(c));
  ss = wave_sum(ss);
  if ((tid & 63) == 0) part[tid >> 6] = ss;
  __syncthreads();
  const float r = 1.0f / sqrtf((part[0] + part[1] + part[2] + part[3]) / (float)H + eps);
  uint8_t* crow = codes + (long)blockIdx.x * mx_row_bytes(H, FMT);
  uint8_t* srow = scales + (long)blockIdx.x * sp;
  auto put = [&](int c, u32x4 raw) {
    float f[8] = {};
    if (c < nc) {
      float wv[8], sv[8];
      unpack8(raw, f);
      unpack8(ld16(w + 8 * c), wv);
      unpack8(ld16(shift + 8 * c), sv);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __builtin_fmaf(f[i] * r, wv[i], sv[i]);
    }
    mx_store8<FMT>(f, c, kp, crow, srow);
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

template <int FMT, bool GATE>
hipError_t quantize(const uint16_t* x, long ldx, const uint16_t* u, long ldu, long M, int K, uint8_t* codes,
                    uint8_t* scales, hipStream_t st) {
  const long blocks = (M * 4 * mx_sp(K) + 255) / 256;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | (GATE ? reinterpret_cast<uintptr_t>(u) : 0);
  const bool vec = at % 16 == 0 && ldx % 8 == 0 && (!GATE || ldu % 8 == 0) && K % 8 == 0;
  if (vec)
    mx_quantize_kernel<FMT, true, GATE><<<(unsigned)blocks, 256, 0, st>>>(x, ldx, u, ldu, M, K, codes, scales);
  else
    mx_quantize_kernel<FMT, false, GATE><<<(unsigned)blocks, 256, 0, st>>>(x, ldx, u, ldu, M, K, codes, scales);
  return hipGetLastError();
}

template <int FMT, bool RES, class... A>
hipError_t norm(int T, int H, hipStream_t st, A... a) {
  switch ((int)((4 * mx_sp(H) + 255) / 256)) {   // the row's chunks per thread
    case 1: rms_norm_mx_kernel<FMT, 1, RES><<<T, 256, 0, st>>>(a...); break;
    case 2: rms_norm_mx_kernel<FMT, 2, RES><<<T, 256, 0, st>>>(a...); break;
    case 3: rms_norm_mx_kernel<FMT, 3, RES><<<T, 256, 0, st>>>(a...); break;
    default: rms_norm_mx_kernel<FMT, 4, RES><<<T, 256, 0, st>>>(a...);
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

hipError_t launch_mx_dequantize(const uint8_t* codes, const uint8_t* scales, long M, int K, int fmt, uint16_t* y,
                                hipStream_t st) {
  const long blocks = (M * ((K + 7) / 8) + 255) / 256;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  const bool vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  const unsigned n = (unsigned)blocks;
  if (fmt == MX_E4M3) {
    if (vec) mx_dequantize_kernel<MX_E4M3, true><<<n, 256, 0, st>>>(codes, scales, M, K, y);
    else mx_dequantize_kernel<MX_E4M3, false><<<n, 256, 0, st>>>(codes, scales, M, K, y);
  } else {
    if (vec) mx_dequantize_kernel<MX_E2M1, true><<<n, 256, 0, st>>>(codes, scales, M, K, y);
    else mx_dequantize_kernel<MX_E2M1, false><<<n, 256, 0, st>>>(codes, scales, M, K, y);
  }
  return hipGetLastError();
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
