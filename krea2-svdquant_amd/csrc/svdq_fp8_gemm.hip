// Product of an E4M3 activation a [M, kp] (a float32 scale for each row and 128 columns, [kp / 128, M]) with an E4M3 weight
// w [N, kp] (a float32 scale for each 128 x 128 block, [ceil(N / 128), kp / 128]):
//   y[m, n] = sum over blocks b of sa[b, m] sw[n / 128, b] (sum over the block's 128 k of a[m, k] w[n, k])  (+ bias[n])
// in float32, rounded once to bf16.
//
// v_mfma_f32_16x16x128 sums exactly one block: its result is scaled and added to the accumulator by one FMA per value
// (the scales are any float32, so the matrix instruction's own power-of-two scales cannot take them).  The weight is the
// first operand, so a lane holds one row m and four consecutive n: its scales are one value per row of tiles, times one per
// block that is the same for the whole wave.
#include <type_traits>
#include <utility>

#include "svdq_fp8.h"
#include "svdq_kernels.h"

namespace svdq {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Frag {
  u32x4 q[2];
};

__device__ __forceinline__ f32x4 fp8_mfma16(const Fp8Frag& w, const Fp8Frag& a) {
  const i32x8 wv = __builtin_bit_cast(i32x8, __builtin_shufflevector(w.q[0], w.q[1], 0, 1, 2, 3, 4, 5, 6, 7));
  const i32x8 av = __builtin_bit_cast(i32x8, __builtin_shufflevector(a.q[0], a.q[1], 0, 1, 2, 3, 4, 5, 6, 7));
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, av, f32x4{}, 0, 0, 0, 127, 0, 127);
}

template <int N>
__device__ __forceinline__ void landed_and_met() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ __forceinline__ void dma4_at(const void* at, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(at), "{m0}"(lds) : "memory");
}

// Block tile BM x BN (BM = 16 TM WM rows of a, BN = 16 TN WN rows of w, a wave's 16 TN within one block of 128), WM x WN
// waves, a ring of NB stages of 128 columns in LDS filled by DMA.  Rows of 128 bytes lie in chunks of 16, chunk c at slot
// c ^ (row / 2 mod 8).
template <int TM, int TN, int WM, int WN, int NB>
struct Fp8Tile {
  static constexpr int NW = WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN;
  static constexpr int TA = BM / 8, TB = BN / 8;                            // DMA instructions of 1024 bytes
  static constexpr int DA = TA / NW, D = DA + TB / NW;                      // per wave and stage, and one of scales
  static constexpr int BUF = (TA + TB) * 1024, OS = NB * BUF, LDS = OS + NB * NW * 256;
  static_assert(LDS <= 160 * 1024, "LDS");
  static_assert(TA % NW == 0 && TB % NW == 0 && 128 % (16 * TN) == 0 && TM <= 4 && NB >= 2, "whole instructions");
  static_assert(NB * (D + 1) <= 63, "vmcnt counts to 63");
};

template <int TM, int TN, int WM, int WN, int NB>
__global__ void __launch_bounds__(64 * WM * WN, 2) fp8_gemm_tile_kernel(Fp8GemmParams p, int nbm, int nbn, int group_m) {
  using T = Fp8Tile<TM, TN, WM, WN, NB>;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
  int bm, bn;
  tile_coords(blockIdx.x, nbm, nbn, group_m, bm, bn);
  const int m0 = bm * T::BM, n0 = bn * T::BN, kp = (int)fp8_kp(p.K), nst = kp / 128;
  const uint32_t lds0 = lds_offset(sm);
  const int chunk = lane % 8 ^ (lane / 8 >> 1 & 3), turned = 4;   // row / 2 mod 8 of row 8 i + lane / 8: 4 (i & 1) more
  uint32_t off[T::D];
#pragma unroll
  for (int d = 0; d < T::D; ++d) {
    const bool a = d < T::DA;
    const int i = wave + T::NW * (a ? d : d - T::DA), row = 8 * i + lane / 8;
    off[d] = (uint32_t)((long)min(row, (a ? p.M - m0 : p.N - n0) - 1) * kp + 16 * (chunk ^ (i & 1 ? turned : 0)));
  }
  const uint8_t *src_a = p.a + (long)m0 * kp, *src_w = p.w + (long)n0 * kp;
  const int mw = m0 + 16 * TM * wm, nw = n0 + 16 * TN * wn;
  const float* src_s = p.as + min(mw + min(lane, 16 * TM - 1), p.M - 1);
  int ahead = 0;
  // the stage `ahead`; past the last one that again, so that the waits count the same loads throughout
  auto fetch = [&](int buf) {
#pragma unroll
    for (int d = 0; d < T::D; ++d)
      dma16(d < T::DA ? src_a : src_w, off[d],
            lds0 + buf * T::BUF + 1024 * (d < T::DA ? wave + T::NW * d : T::TA + wave + T::NW * (d - T::DA)));
    dma4_at(src_s, lds0 + T::OS + 256 * (buf * T::NW + wave));
    if (++ahead < nst) {
      src_a += 128;
      src_w += 128;
      src_s += p.M;
    }
  };
  const float* wsrow = p.ws + (long)min(nw / 128, (p.N - 1) / 128) * nst;
  float wscales = wsrow[min(lane, nst - 1)];
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(wscales)::"memory");

  f32x4 acc[TN][TM] = {};
#pragma unroll
  for (int i = 0; i < NB - 1; ++i) fetch(i);
  int cur = 0, nxt = NB - 1;
#pragma unroll 1
  for (int s = 0; s < nst; ++s) {
    landed_and_met<(NB - 2) * (T::D + 1)>();
    if ((s & 63) == 0 && s) {   // waited for in here: a wait behind it would be for every stage's loads
      wscales = wsrow[min(s + lane, nst - 1)];
      asm volatile("s_waitcnt vmcnt(0)" : "+v"(wscales)::"memory");
    }
    fetch(nxt);
    const uint8_t* ba = sm + cur * T::BUF + (16 * TM * wm + lr) * 128;
    const uint8_t* bw = sm + cur * T::BUF + T::TA * 1024 + (16 * TN * wn + lr) * 128;
    const float* bs = reinterpret_cast<const float*>(sm + T::OS + 256 * (cur * T::NW + wave)) + lr;
    const float sw = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wscales), s & 63));
    const int o0 = 16 * (b ^ (lr >> 1 & 7)), o1 = 16 * ((4 + b) ^ (lr >> 1 & 7));
    Fp8Frag fa[TM];
    float sc[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      fa[t].q[0] = *reinterpret_cast<const u32x4*>(ba + 2048 * t + o0);
      fa[t].q[1] = *reinterpret_cast<const u32x4*>(ba + 2048 * t + o1);
      sc[t] = bs[16 * t] * sw;
    }
#pragma unroll
    for (int x = 0; x < TN; ++x) {
      Fp8Frag fw;
      fw.q[0] = *reinterpret_cast<const u32x4*>(bw + 2048 * x + o0);
      fw.q[1] = *reinterpret_cast<const u32x4*>(bw + 2048 * x + o1);
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        const f32x4 v = fp8_mfma16(fw, fa[t]);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[x][t][r] = __builtin_fmaf(v[r], sc[t], acc[x][t][r]);
      }
    }
    cur = cur + 1 == NB ? 0 : cur + 1;
    nxt = nxt + 1 == NB ? 0 : nxt + 1;
  }
  // nothing of the DMA may be under way when the next workgroup takes this LDS
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  // register r of lane (lr, b): row lr of a, column 4 b + r of w
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int m = mw + 16 * t + lr;
#pragma unroll
    for (int x = 0; x < TN; ++x) {
      const int n = nw + 16 * x + 4 * b;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (m < p.M && n + r < p.N)
          p.y[(long)m * p.ldy + n + r] =
              (uint16_t)pack_bf16x2(acc[x][t][r] + (p.bias ? bf16f(p.bias[n + r]) : 0.0f), 0.0f);
    }
  }
}

template <int TM, int TN, int WM, int WN, int NB>
hipError_t launch_tile(const Fp8GemmParams& p, hipStream_t st) {
  using T = Fp8Tile<TM, TN, WM, WN, NB>;
  const long nbm = (p.M + T::BM - 1) / T::BM, nbn = (p.N + T::BN - 1) / T::BN;
  fp8_gemm_tile_kernel<TM, TN, WM, WN, NB><<<(unsigned)(nbm * nbn), 64 * WM * WN, 0, st>>>(p, (int)nbm, (int)nbn, 4);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_gemm(const Fp8GemmParams& p, hipStream_t st) {
  const long large = (p.M + 255L) / 256 * ((p.N + 255L) / 256);
  return large >= 256 ? launch_tile<4, 8, 4, 2, 2>(p, st) : launch_tile<2, 2, 2, 2, 4>(p, st);
}

}  // namespace svdq
