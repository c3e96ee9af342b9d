// Product of an MX activation a [M, K] (E2M1 or E4M3 codes) with an MX weight w [N, K] (E2M1 codes):
//   y[m, n] = sum over blocks b of 2^(sa[m, b] + sw[n, b] - 254) sum over 32 k of a[m, k] w[n, k]  (+ bias[n])
// in float32 on the scaled matrix instructions, rounded once to bf16 or stored as float32.
//
// v_mfma_scale_f32_32x32x64 takes the weight as its first operand and the activation as its second, so a lane
// holds one row m of the output and runs of four consecutive n.  Lane l (half h = l / 32) supplies row
// l % 32 of each: E2M1 the 32 codes k = 32 h .. of a step of 64 (16 bytes), E4M3 k = 16 h .. + 15 and
// 32 + 16 h .. + 15 (two runs of 16 bytes); the scale of its row's block h.  (Checked on the card, as is that
// a scale byte of 255 makes the product NaN and that 0 is 2^-127.)
//
// Precision.  E2M1 x E2M1: the instruction's sums over a block are exact.  E4M3 x E2M1: within each group of 8
// consecutive k it drops what lies below 2^-13 of the largest product's power of two (measured: 2688 + 0.125 is
// exact, 2688 + 0.0625 is 2688, a ninth k apart it is exact again), about 1.2e-5 of a result in the 2-norm.
// Under a bf16 output's own 2^-8 that is left so.  With float32 output each E4M3 operand is split by the top bit
// of its exponent into codes of magnitude 2 and more and codes below 2, and multiplied in two instructions: the
// products of either half are multiples of 2^-3 up to 2^11, or of 2^-10 up to 2^4, so neither drops anything.
#include "svdq_kernels.h"
#include "svdq_mx.h"

namespace svdq {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int FMT>
struct MxFrag {
  u32x4 q[FMT == MX_E4M3 ? 2 : 1];
};

__device__ __forceinline__ i32x8 operand(const MxFrag<MX_E2M1>& f) {
  return __builtin_bit_cast(i32x8, __builtin_shufflevector(f.q[0], f.q[0], 0, 1, 2, 3, -1, -1, -1, -1));
}
__device__ __forceinline__ i32x8 operand(const MxFrag<MX_E4M3>& f) {
  return __builtin_bit_cast(i32x8, __builtin_shufflevector(f.q[0], f.q[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

// acc += w a on one step of 64: scale byte SEL of ws and of as.  EXACT: in two halves by the E4M3 exponent.
template <int AF, bool EXACT, int SEL>
__device__ __forceinline__ f32x16 mx_mfma(const MxFrag<MX_E2M1>& w, const MxFrag<AF>& a, f32x16 acc, uint32_t ws,
                                          uint32_t as) {
  if constexpr (EXACT && AF == MX_E4M3) {
    MxFrag<AF> hi, lo;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t b = a.q[i][d] >> 6 & 0x01010101u, mask = (b << 8) - b;   // 0xFF where the exponent is 8 or more
        hi.q[i][d] = a.q[i][d] & mask;
        lo.q[i][d] = a.q[i][d] & ~mask;
      }
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(lo), acc, 4, 0, SEL, (int)ws, SEL, (int)as);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(hi), acc, 4, 0, SEL, (int)ws, SEL, (int)as);
  } else {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(a), acc, 4, AF == MX_E4M3 ? 0 : 4, SEL,
                                                           (int)ws, SEL, (int)as);
  }
}

// One wave per 32 x 32 tile of the output, operands loaded from memory as the matrix instruction takes them.
template <int AF, bool F32>
__global__ void __launch_bounds__(256) mx_gemm_simple_kernel(MxGemmParams p) {
  const int lane = threadIdx.x & 63, lr = lane & 31, h = lane >> 5, wave = threadIdx.x >> 6;
  const long m0 = (long)blockIdx.y * 64 + 32 * (wave & 1), n0 = (long)blockIdx.x * 64 + 32 * (wave >> 1);
  const long m = min(m0 + lr, (long)p.M - 1), n = min(n0 + lr, (long)p.N - 1);
  const int kp = (int)mx_kp(p.K), sp = (int)mx_sp(p.K);
  const uint8_t* a = p.a + m * mx_row_bytes(p.K, AF) + 16 * h;
  const uint8_t* w = p.w + n * (kp / 2) + 16 * h;
  const uint8_t *as = p.as + m * sp + h, *ws = p.ws + n * sp + h;
  f32x16 acc = {};
  for (int k = 0; k < kp; k += 64) {
    MxFrag<AF> fa;
    MxFrag<MX_E2M1> fw;
    fw.q[0] = *reinterpret_cast<const u32x4*>(w + k / 2);
    if (AF == MX_E4M3) {
      fa.q[0] = *reinterpret_cast<const u32x4*>(a + k);
      fa.q[AF == MX_E4M3] = *reinterpret_cast<const u32x4*>(a + k + 32);
    } else {
      fa.q[0] = *reinterpret_cast<const u32x4*>(a + k / 2);
    }
    acc = mx_mfma<AF, F32, 0>(fw, fa, acc, ws[k / 32], as[k / 32]);
  }
  if (m0 + lr >= p.M) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const long col = n0 + 8 * (r / 4) + 4 * h + r % 4;
    if (col < p.N) {
      const float v = acc[r] + (p.bias ? bf16f(p.bias[col]) : 0.0f);
      if (F32) static_cast<float*>(p.y)[m * p.ldy + col] = v;
      else static_cast<uint16_t*>(p.y)[m * p.ldy + col] = (uint16_t)pack_bf16x2(v, 0.0f);
    }
  }
}

}  // namespace

hipError_t launch_mx_gemm(const MxGemmParams& p, int fmt, bool out_f32, hipStream_t st) {
  const dim3 grid((unsigned)((p.N + 63) / 64), (unsigned)((p.M + 63) / 64));
  if (grid.y > 65535) return hipErrorInvalidValue;
  if (fmt == MX_E4M3) {
    if (out_f32) mx_gemm_simple_kernel<MX_E4M3, true><<<grid, 256, 0, st>>>(p);
    else mx_gemm_simple_kernel<MX_E4M3, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (out_f32) mx_gemm_simple_kernel<MX_E2M1, true><<<grid, 256, 0, st>>>(p);
    else mx_gemm_simple_kernel<MX_E2M1, false><<<grid, 256, 0, st>>>(p);
  }
  return hipGetLastError();
}

}  // namespace svdq
