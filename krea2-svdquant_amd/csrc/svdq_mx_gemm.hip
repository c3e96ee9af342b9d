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
#include <cstdlib>
#include <type_traits>
#include <utility>

#include "svdq_kernels.h"
#include "svdq_mx.h"

namespace svdq {

int mx_gemm_tile_choice(int M, int N, int K, int fmt);

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
        // 0xFF where the exponent is 8 or more: v_perm's selectors 8 and 9 (10 and 11) repeat the top bits of bytes 1 and 3 of
        // its second (first) operand
        const uint32_t x = a.q[i][d], mask = __builtin_amdgcn_perm(x << 9, x << 1, 0x090B080Au);
        hi.q[i][d] = x & mask;
        lo.q[i][d] = x & ~mask;
      }
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(lo), acc, 4, 0, SEL, (int)ws, SEL, (int)as);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(hi), acc, 4, 0, SEL, (int)ws, SEL, (int)as);
  } else {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(a), acc, 4, AF == MX_E4M3 ? 0 : 4, SEL,
                                                           (int)ws, SEL, (int)as);
  }
}

template <class F, int... B>
__device__ __forceinline__ void for_each_index(F&& f, std::integer_sequence<int, B...>) {
  (f(std::integral_constant<int, B>{}), ...);
}

// Block tile BM x BN (BM = 32 TM WM rows of a, BN = 32 TN WN rows of w), WM x WN waves of TM x TN accumulators.
//
// A stage is 128 columns of K in a ring of NBUF LDS buffers filled by DMA: rows of a (64 bytes E2M1, 128 bytes
// E4M3) and of w (64 bytes) in chunks of 16 bytes, a row's chunk c at slot c ^ f(row), which spreads sixteen
// consecutive rows' chunk over the 64 banks (f = row / 4 mod 4 in rows of 64 bytes, row / 2 mod 8 in rows of 128) while
// the DMA's lanes still read whole rows.  Scales come four stages at a time, 16 bytes a row, and are taken into
// registers at once, so they need no second buffer.
//
// A stage is two matrix steps of 64.  Its first step's operands are read during the stage before, its second's
// during its first step's products; between the two ("mid-stage") the wave waits for the next stage's bytes and for
// the other waves, after which everything of this stage has been read: its buffer takes stage s + NBUF.  So the one
// barrier per stage has matrix instructions queued on both sides.
template <int AF, bool F32, int TM, int TN, int WM, int WN, int NB>
struct MxTile {
  static constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, NBUF = NB;
  static constexpr int RA = AF == MX_E4M3 ? 128 : 64;                       // bytes of a row of a per stage
  static constexpr int TA = BM * RA / 1024, TB = BN * 64 / 1024;            // DMA instructions of 1024 bytes
  static constexpr int DA = TA / NW, D = DA + TB / NW;                      // per wave and stage
  static constexpr int TS = (BM + BN + 63) / 64, E = (TS + NW - 1) / NW;    // of scales, per four stages
  static constexpr int OB = TA * 1024, BUF = (TA + TB) * 1024, OS = NBUF * BUF;
  static constexpr int LDS = OS + TS * 1024;
  static constexpr int GROUPS = 160 * 1024 / LDS;                           // workgroups that a CU's LDS holds
  static_assert(LDS <= 160 * 1024, "LDS");
  static_assert(NBUF >= 3 && TA % NW == 0 && TB % NW == 0, "whole instructions per wave");
  static_assert(NBUF * D + E <= 63, "vmcnt counts to 63");
};

template <int N>
__device__ __forceinline__ void landed_and_met() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// the same with a per-lane 64-bit address
__device__ __forceinline__ void dma16_at(const void* at, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(at), "{m0}"(lds) : "memory");
}

template <int AF, bool F32, int TM, int TN, int WM, int WN, int NB>
__global__ void __launch_bounds__(64 * WM * WN, (MxTile<AF, F32, TM, TN, WM, WN, NB>::GROUPS > 1 ? 2 : 1))
    mx_gemm_tile_kernel(MxGemmParams p, int nbm, int nbn, int group_m) {
  using T = MxTile<AF, F32, TM, TN, WM, WN, NB>;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
  int bm, bn;
  tile_coords(blockIdx.x, nbm, nbn, group_m, bm, bn);
  const int m0 = bm * T::BM, n0 = bn * T::BN;
  const int nst = (int)(mx_kp(p.K) / 128), sp = (int)mx_sp(p.K);
  const long pa = mx_row_bytes(p.K, AF), pw = mx_kp(p.K) / 2;
  const uint32_t lds0 = lds_offset(sm);

  // Instruction i of a stage moves 1024 bytes: 16 (8) rows of 4 (8) chunks, a's rows first.  A wave's d-th is
  // wave + NW d: DA of a's, then w's.
  const uint8_t *src_a = p.a + (long)m0 * pa, *src_w = p.w + (long)n0 * pw;
  const uint32_t ldsw = lds0 + 1024 * wave;
  uint32_t off[T::D];
#pragma unroll
  for (int d = 0; d < T::D; ++d) {
    const bool a = d < T::DA;
    const int rows = a ? 1024 / T::RA : 16, cpr = a ? T::RA / 16 : 4;
    const int row = (wave + T::NW * (a ? d : d - T::DA)) * rows + lane / cpr, slot = lane % cpr;
    const int chunk = slot ^ (cpr == 8 ? row >> 1 & 7 : row >> 2 & 3);
    off[d] = (uint32_t)(min(row, (a ? p.M - m0 : p.N - n0) - 1) * (a ? pa : pw) + 16 * chunk);
  }
  const uint8_t* ssrc[T::E];
#pragma unroll
  for (int e = 0; e < T::E; ++e) {
    const int r = 64 * min(wave + T::NW * e, T::TS - 1) + lane;
    ssrc[e] = r < T::BM ? p.as + (long)min(m0 + r, p.M - 1) * sp : p.ws + (long)min(n0 + r - T::BM, p.N - 1) * sp;
  }
  // Every stage fetches the one NBUF further on; past the last stage the last one again, into a buffer that nothing
  // reads any more, so that the number of loads under way, which the waits count, is the same throughout.
  int ahead = 1;
  auto fetch = [&](uint32_t buf, int d) {   // this wave's instruction d, into the buffer at byte buf
    dma16(d < T::DA ? src_a : src_w, off[d], ldsw + 1024 * T::NW * d + buf);
    if (d == T::D - 1) {
      src_a += ahead < nst ? T::RA : 0;
      src_w += ahead < nst ? 64 : 0;
      ++ahead;
    }
  };
  auto fetch_scales = [&](int super) {
    const int more = 4 * (super + 1) < nst ? 16 : 0;
#pragma unroll
    for (int e = 0; e < T::E; ++e) {
      dma16_at(ssrc[e], lds0 + T::OS + 1024 * min(wave + T::NW * e, T::TS - 1));
      ssrc[e] += more;
    }
  };

  const int ra = 32 * TM * wm + lr, rw = 32 * TN * wn + lr;   // this lane's row of its first tiles
  MxFrag<AF> fa[2][TM];
  MxFrag<MX_E2M1> fw[2][TN];
  u32x4 sa[TM], sw[TN];
  // LDS read r of step j of the stage in the buffer at byte buf: the w operands, then the a operands (E4M3: two each)
  constexpr int AR = AF == MX_E4M3 ? 2 : 1, READS = TN + AR * TM, PRODUCTS = TN * TM;
  auto read = [&](uint32_t buf, int j, int r) {
    const uint8_t* b = sm + buf;
    if (r < TN) {
      fw[j][r].q[0] = *reinterpret_cast<const u32x4*>(b + T::OB + (rw + 32 * r) * 64 + 16 * ((2 * j + h) ^ (lr >> 2 & 3)));
    } else {
      const int t = (r - TN) / AR, u = (r - TN) % AR;
      const uint8_t* row = b + (ra + 32 * t) * T::RA;
      if (AF == MX_E4M3) fa[j][t].q[u] = *reinterpret_cast<const u32x4*>(row + 16 * ((4 * j + 2 * u + h) ^ (lr >> 1 & 7)));
      else fa[j][t].q[0] = *reinterpret_cast<const u32x4*>(row + 16 * ((2 * j + h) ^ (lr >> 2 & 3)));
    }
  };
  auto read_scales = [&] {   // of the next four stages
    const uint8_t* b = sm + T::OS;
#pragma unroll
    for (int t = 0; t < TM; ++t) sa[t] = *reinterpret_cast<const u32x4*>(b + (ra + 32 * t) * 16);
#pragma unroll
    for (int t = 0; t < TN; ++t) sw[t] = *reinterpret_cast<const u32x4*>(b + (T::BM + rw + 32 * t) * 16);
  };

  f32x16 acc[TN][TM] = {};
  fetch_scales(0);
#pragma unroll
  for (int s = 0; s < T::NBUF - 1; ++s)
#pragma unroll
    for (int d = 0; d < T::D; ++d) fetch(s * T::BUF, d);
#pragma unroll
  for (int d = 0; d < (T::D + 1) / 2; ++d) fetch((T::NBUF - 1) * T::BUF, d);
  landed_and_met<(T::NBUF - 2) * T::D + (T::D + 1) / 2>();
  read_scales();
#pragma unroll
  for (int r = 0; r < READS; ++r) read(0, 0, r);

  // One stage, from the buffer at cur, with the scales in element S of sa and sw.  Memory instructions are spread over
  // the products: a wave issues in order, and a block of them ahead of the products leaves the matrix unit idle while
  // their queues drain.  The LDS reads go first, one behind each product, so that they are over when they are needed;
  // the DMA instructions of stage s + NBUF - 1 are issued half in the second step of stage s - 1, after its mid-stage
  // freed their buffer, half in the first step of stage s.  No branch in between: the compiler would move the first
  // step's products below it, past the barrier.
  constexpr int D1 = (T::D + 1) / 2, D0 = T::D - D1;   // in a second step, in the first step that follows
  uint32_t cur = 0, nxt = T::BUF, free_ = (T::NBUF - 1) * T::BUF;
  auto stage = [&](auto sub, auto wait, auto next_scales) {
    constexpr int S = decltype(sub)::value;
    // this lane's blocks are h and 2 + h of the stage's four: bytes 0 and 2 after the shift
    uint32_t ca[TM], cw[TN];
#pragma unroll
    for (int t = 0; t < TM; ++t) ca[t] = sa[t][S] >> (8 * h);
#pragma unroll
    for (int t = 0; t < TN; ++t) cw[t] = sw[t][S] >> (8 * h);
    auto products = [&](auto step, auto nd, auto&& rd, auto&& dma) {
      constexpr int J = decltype(step)::value, ND = decltype(nd)::value, OPS = READS + ND;
      constexpr int PER = (OPS + PRODUCTS - 1) / PRODUCTS;   // behind each product
      // DMA instructions as far apart as the products behind the reads allow
      constexpr int LEFT = PRODUCTS - (READS + PER - 1) / PER, GAP = PER == 1 && ND && LEFT / ND > 1 ? LEFT / ND : 1;
#pragma unroll
      for (int i = 0; i < PRODUCTS; ++i) {
        const int x = i / TM, t = i % TM;
        acc[x][t] = mx_mfma<AF, F32, 2 * J>(fw[J][x], fa[J][t], acc[x][t], cw[x], ca[t]);
        if (GAP > 1) {
          if (i < READS) rd(i);
          else if ((i - READS) % GAP == 0 && (i - READS) / GAP < ND) dma((i - READS) / GAP);
        } else {
#pragma unroll
          for (int o = i * PER; o < (i + 1) * PER && o < OPS; ++o) {
            if (o < READS) rd(o);
            else dma(o - READS);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    products(std::integral_constant<int, 0>{}, std::integral_constant<int, D0>{}, [&](int r) { read(cur, 1, r); },
             [&](int d) { fetch(free_, D1 + d); });
    landed_and_met<decltype(wait)::value>();
    next_scales();
    products(std::integral_constant<int, 1>{}, std::integral_constant<int, D1>{}, [&](int r) { read(nxt, 0, r); },
             [&](int d) { fetch(cur, d); });
    free_ = cur;
    cur = nxt;
    nxt = nxt + T::BUF == T::OS ? 0 : nxt + T::BUF;
  };
  // Mid-stage of s, everything up to stage s + NBUF - 1 has been issued, and stage s + 1 has landed when only what was
  // issued after it is under way: NBUF - 2 stages, and the scales, which are issued at the mid-stage of S = 0.
  constexpr int WAIT = (T::NBUF - 2) * T::D;
  int s0 = 0;
  for (; s0 + 4 <= nst; s0 += 4)
    for_each_index([&](auto sub) {
      constexpr int S = decltype(sub)::value;
      stage(sub, std::integral_constant<int, WAIT + (S >= 1 && S <= T::NBUF - 2 ? T::E : 0)>{}, [&] {
        if (S == 0) fetch_scales(s0 / 4 + 1);
        if (S == 3) read_scales();
      });
    }, std::make_integer_sequence<int, 4>{});
  // up to three more; no further scales to fetch
#pragma unroll 1
  for (int s = s0; s < nst; ++s) {
    stage(std::integral_constant<int, 0>{}, std::integral_constant<int, WAIT>{}, [] {});
#pragma unroll
    for (int t = 0; t < TM; ++t) sa[t] = __builtin_shufflevector(sa[t], sa[t], 1, 2, 3, 0);
#pragma unroll
    for (int t = 0; t < TN; ++t) sw[t] = __builtin_shufflevector(sw[t], sw[t], 1, 2, 3, 0);
  }
  // nothing of the DMA may be under way when the next workgroup takes this one's LDS
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // Register 4 q + r of lane (lr, h): row lr of a, column 8 q + 4 h + r of w.  bf16: the halves of a row exchange
  // runs of four, so that a lane stores eight consecutive columns.
  const int mrow = m0 + 32 * TM * wm + lr, ncol = n0 + 32 * TN * wn;
  const bool wide = p.ldy % 8 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int c0 = ncol + 32 * i;
    if (c0 >= p.N) continue;
    float b[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = c0 + 8 * (r / 4) + 4 * h + r % 4;
      b[r] = p.bias && c < p.N ? bf16f(p.bias[c]) : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      const int m = mrow + 32 * t;
      float v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = acc[i][t][r] + b[r];
      if (F32) {
        float* row = static_cast<float*>(p.y) + (long)m * p.ldy;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = c0 + 8 * q + 4 * h;
          if (m < p.M) {
            if (wide && c + 4 <= p.N) *reinterpret_cast<f32x4*>(row + c) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            else
              for (int r = 0; r < 4; ++r)
                if (c + r < p.N) row[c + r] = v[4 * q + r];
          }
        }
      } else {
        uint16_t* row = static_cast<uint16_t*>(p.y) + (long)m * p.ldy;
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          u32x4 o = {pack_bf16x2(v[4 * q], v[4 * q + 1]), pack_bf16x2(v[4 * q + 2], v[4 * q + 3]),
                     pack_bf16x2(v[4 * q + 4], v[4 * q + 5]), pack_bf16x2(v[4 * q + 6], v[4 * q + 7])};
          // lanes h = 0: columns 8 q .. + 3 and (from the other half) + 4 .. 7; h = 1: 8 (q + 1) ..
          uint32_t x0 = o[0], x1 = o[1], y0 = o[2], y1 = o[3];
          permlane32_swap(x0, y0);
          permlane32_swap(x1, y1);
          const u32x4 w = {x0, x1, y0, y1};
          const int c = c0 + 8 * (q + h);
          if (m < p.M) {
            if (wide && c + 8 <= p.N) *reinterpret_cast<u32x4*>(row + c) = w;
            else
              for (int r = 0; r < 8; ++r)
                if (c + r < p.N) row[c + r] = (uint16_t)(w[r / 2] >> (16 * (r % 2)));
          }
        }
      }
    }
  }
}

template <int AF, bool F32, int TM, int TN, int WM, int WN, int NB>
hipError_t launch_tile(const MxGemmParams& p, hipStream_t st) {
  using T = MxTile<AF, F32, TM, TN, WM, WN, NB>;
  const long nbm = (p.M + T::BM - 1) / T::BM, nbn = (p.N + T::BN - 1) / T::BN;
  if (nbm * nbn > INT32_MAX) return hipErrorInvalidValue;
  mx_gemm_tile_kernel<AF, F32, TM, TN, WM, WN, NB>
      <<<(unsigned)(nbm * nbn), 64 * WM * WN, 0, st>>>(p, (int)nbm, (int)nbn, 4);
  return hipGetLastError();
}

// Block tiles: 64 x 64, 128 x 128, 256 x 256 rows of a by rows of w.
template <int AF, bool F32>
hipError_t launch_any(const MxGemmParams& p, hipStream_t st) {
  constexpr bool E8 = AF == MX_E4M3;
  switch (mx_gemm_tile_choice(p.M, p.N, p.K, AF)) {
    case 0: return launch_tile<AF, F32, 1, 1, 2, 2, 4>(p, st);
    case 1: return launch_tile<AF, F32, 2, 2, 2, 2, E8 ? 3 : 4>(p, st);
    // E4M3 with float32 output needs registers for the halves of its operands
    default: return launch_tile<AF, F32, E8 && F32 ? 2 : 4, 4, 2, 2, E8 && !F32 ? 3 : 4>(p, st);
  }
}

}  // namespace

int mx_gemm_tile_choice(int M, int N, int K, int fmt) {
  const long big = (long)((M + 255) / 256) * ((N + 255) / 256), mid = (long)((M + 127) / 128) * ((N + 127) / 128);
  return big >= 200 ? 2 : mid >= 200 ? 1 : 0;
}

hipError_t launch_mx_gemm(const MxGemmParams& p, int fmt, bool out_f32, hipStream_t st) {
  if (fmt == MX_E4M3) return out_f32 ? launch_any<MX_E4M3, true>(p, st) : launch_any<MX_E4M3, false>(p, st);
  return out_f32 ? launch_any<MX_E2M1, true>(p, st) : launch_any<MX_E2M1, false>(p, st);
}

}  // namespace svdq
