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
// exact, 2688 + 0.0625 is 2688, a ninth k apart it is exact again): less than 2^-12 of the largest product for each
// of the other seven.  For normal operands that is about 1.2e-5 of the results in the 2-norm, for a result that its
// products cancel to it can be any share.  Beside a bf16 output's own half step of 2^-8 that is left so.  With
// float32 output each E4M3 operand is split by the top bit of its exponent into codes of magnitude 2 and more and
// codes below 2, and multiplied in two instructions: the products of either half are multiples of 2^-3 up to 2^11, or
// of 2^-10 up to 2^4, so neither drops anything.
#include <type_traits>
#include <utility>

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

// a = hi + lo by the top bit of the E4M3 exponents
__device__ __forceinline__ void split(const MxFrag<MX_E4M3>& a, MxFrag<MX_E4M3>& hi, MxFrag<MX_E4M3>& lo) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      // 0xFF where the exponent is 8 or more: v_perm's selectors 8 and 9 (10 and 11) repeat the top bits of bytes 1 and 3
      // of its second (first) operand
      const uint32_t x = a.q[i][d], mask = __builtin_amdgcn_perm(x << 9, x << 1, 0x090B080Au);
      hi.q[i][d] = x & mask;
      lo.q[i][d] = x & ~mask;
    }
}

// acc += w a on one step of 64: scale byte SEL of ws and of as.  EXACT: in two halves by the E4M3 exponent.
template <int AF, bool EXACT, int SEL>
__device__ __forceinline__ f32x16 mx_mfma(const MxFrag<MX_E2M1>& w, const MxFrag<AF>& a, f32x16 acc, uint32_t ws,
                                          uint32_t as) {
  if constexpr (EXACT && AF == MX_E4M3) {
    MxFrag<AF> hi, lo;
    split(a, hi, lo);
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
// A stage is SPS matrix steps of 64 columns of K, 2 or 4, in a ring of NB LDS buffers filled by DMA.  Rows lie in chunks
// of 16 bytes, chunk c at slot c ^ f(row), which spreads sixteen consecutive rows' chunk over the 64 banks (rows of 64
// bytes: f = row / 4 mod 4, of 128: row / 2 mod 8, of 256: row mod 16) while the DMA's lanes still read whole rows.
// Scales come CH 16-byte groups a row at a time (a group: 512 columns), and are taken into registers a group at a time,
// so they need no second buffer.
//
// A load fills a cache line of 128 bytes.  Two steps of E2M1 codes are half a line, so stages of two steps read every
// line twice, and what bounds the large tiles is what the L2 delivers (M = 4352, N = 16384, K = 6144, 256 x 256: 248 us,
// on lines read once 224).  Stages of four steps read whole lines; the 256 x 256 tiles, whose LDS holds only two of
// those, take four of two steps and fetch the rows of every second stage in reverse order, so that its first half finds
// the lines of the stage before in the 32 KB of L1: 236 us.  For the same reason scales come in CH = 2 groups (one
// group at a time, a line of 128 bytes for 16: 248, none at all 232).
//
// A step's operands are read during the step before it.  Ahead of a stage's last step the wave waits for the next
// stage's bytes and for the other waves: by then everything of this stage has been read, its buffer takes stage s + NB,
// and the last step reads the next stage's first operands.  So the one barrier per stage has matrix instructions
// queued on both sides.
template <int AF, bool F32, int TM, int TN, int WM, int WN, int SPS, int NB>
struct MxTile {
  static constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, CH = 2;
  static constexpr int RW = 32 * SPS, RA = AF == MX_E4M3 ? 2 * RW : RW;     // bytes of a row of w and of a per stage
  static constexpr int TA = BM * RA / 1024, TB = BN * RW / 1024;            // DMA instructions of 1024 bytes
  static constexpr int DA = TA / NW, D = DA + TB / NW;                      // per wave and stage
  static constexpr int TS = (BM + BN) * CH / 64, E = (TS + NW - 1) / NW;    // of scales, per CH groups
  static constexpr int OB = TA * 1024, BUF = (TA + TB) * 1024, OS = NB * BUF, LDS = OS + TS * 1024;
  static constexpr int GROUPS = 160 * 1024 / LDS;                           // workgroups that a CU's LDS holds
  static constexpr bool TURN = RW < 128;                                    // every second stage in reverse order
  static_assert(LDS <= 160 * 1024, "LDS");
  static_assert(NB >= 2 && TA % NW == 0 && TB % NW == 0 && (BM + BN) * CH % 64 == 0 && NW % 4 == 0, "whole instructions");
  static_assert(NB * D + E <= 63, "vmcnt counts to 63");
};

// f(row) of rows of `bytes`
template <int BYTES>
__device__ __forceinline__ int mx_turn(int row) {
  return BYTES == 64 ? row >> 2 & 3 : BYTES == 128 ? row >> 1 & 7 : row & 15;
}

template <int N>
__device__ __forceinline__ void landed_and_met() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// the same with a per-lane 64-bit address
__device__ __forceinline__ void dma16_at(const void* at, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(at), "{m0}"(lds) : "memory");
}

template <int AF, bool F32, int TM, int TN, int WM, int WN, int SPS, int NB>
__global__ void __launch_bounds__(64 * WM * WN, (MxTile<AF, F32, TM, TN, WM, WN, SPS, NB>::GROUPS > 1 ? 2 : 1))
    mx_gemm_tile_kernel(MxGemmParams p, int nbm, int nbn, int group_m) {
  using T = MxTile<AF, F32, TM, TN, WM, WN, SPS, NB>;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
  int bm, bn;
  tile_coords(blockIdx.x, nbm, nbn, group_m, bm, bn);
  const int m0 = bm * T::BM, n0 = bn * T::BN;
  const int steps = (int)(mx_kp(p.K) / 64), nst = (steps + SPS - 1) / SPS, sp = (int)mx_sp(p.K);   // steps is even
  const long pa = mx_row_bytes(p.K, AF), pw = mx_kp(p.K) / 2;
  const uint32_t lds0 = lds_offset(sm);

  // Instruction i of a stage moves 1024 bytes, 1024 / RA rows of a or 1024 / RW of w, a's first.  A wave's d-th is
  // wave + NW d: DA of a's, then w's.  The chunk of a lane is the same in all of a's, and in all of w's.
  constexpr int CA = T::RA / 16, CW = T::RW / 16;
  const uint8_t *src_a = p.a + (long)m0 * pa, *src_w = p.w + (long)n0 * pw;
  const uint32_t ldsw = lds0 + 1024 * wave;
  const int chunk_a = lane % CA ^ mx_turn<T::RA>(64 / CA * wave + lane / CA);
  const int chunk_w = lane % CW ^ mx_turn<T::RW>(64 / CW * wave + lane / CW);
  uint32_t off[T::D];
#pragma unroll
  for (int d = 0; d < T::D; ++d) {
    const bool a = d < T::DA;
    const int cpr = a ? CA : CW, row = (wave + T::NW * (a ? d : d - T::DA)) * (64 / cpr) + lane / cpr;
    off[d] = (uint32_t)(min(row, (a ? p.M - m0 : p.N - n0) - 1) * (a ? pa : pw) + 16 * (a ? chunk_a : chunk_w));
  }
  // a last stage of two steps out of four has no second half to read: its first half again
  const uint32_t back_a = chunk_a >= CA / 2 ? T::RA / 2 : 0, back_w = chunk_w >= CW / 2 ? T::RW / 2 : 0;
  const uint8_t* ssrc[T::E];
  int spart = lane % T::CH;   // this lane's 16 bytes of a row's 16 CH
#pragma unroll
  for (int e = 0; e < T::E; ++e) {
    const int r = (64 * min(wave + T::NW * e, T::TS - 1) + lane) / T::CH;
    ssrc[e] = r < T::BM ? p.as + (long)min(m0 + r, p.M - 1) * sp : p.ws + (long)min(n0 + r - T::BM, p.N - 1) * sp;
  }
  // Every stage fetches the one NB further on; past the last stage the last one again, into a buffer that nothing
  // reads any more, so that the number of loads under way, which the waits count, is the same throughout.
  int ahead = 0;
  const bool odd = SPS == 4 && steps % 4;
  uint32_t half = odd && nst == 1 ? ~0u : 0u;
  auto fetch = [&](uint32_t buf, int i, bool turned) {   // this wave's i-th instruction, into the buffer at byte buf
    const int d = T::TURN && turned ? T::D - 1 - i : i;
    const uint32_t o = SPS == 4 ? off[d] - (half & (d < T::DA ? back_a : back_w)) : off[d];
    dma16(d < T::DA ? src_a : src_w, o, ldsw + 1024 * T::NW * d + buf);
    if (i == T::D - 1) {
      ++ahead;
      src_a += ahead < nst ? T::RA : 0;
      src_w += ahead < nst ? T::RW : 0;
      if (SPS == 4) half = odd && ahead >= nst - 1 ? ~0u : 0u;
    }
  };
  auto fetch_scales = [&](int chunk) {   // the chunk-th CH groups; beyond a row's scales its last again
    const int at = 16 * min(T::CH * chunk + spart, sp / 16 - 1);
#pragma unroll
    for (int e = 0; e < T::E; ++e) dma16_at(ssrc[e] + at, lds0 + T::OS + 1024 * min(wave + T::NW * e, T::TS - 1));
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
      fw[j & 1][r].q[0] = *reinterpret_cast<const u32x4*>(b + T::OB + (rw + 32 * r) * T::RW + 16 * ((2 * j + h) ^ mx_turn<T::RW>(lr)));
    } else {
      const int t = (r - TN) / AR, u = (r - TN) % AR;
      const uint8_t* row = b + (ra + 32 * t) * T::RA;
      if (AF == MX_E4M3) fa[j & 1][t].q[u] = *reinterpret_cast<const u32x4*>(row + 16 * ((4 * j + 2 * u + h) ^ mx_turn<T::RA>(lr)));
      else fa[j & 1][t].q[0] = *reinterpret_cast<const u32x4*>(row + 16 * ((2 * j + h) ^ mx_turn<T::RA>(lr)));
    }
  };
  auto read_scales = [&](int part) {   // the part-th group of the chunk
    const uint8_t* b = sm + T::OS + 16 * part;
#pragma unroll
    for (int t = 0; t < TM; ++t) sa[t] = *reinterpret_cast<const u32x4*>(b + (ra + 32 * t) * 16 * T::CH);
#pragma unroll
    for (int t = 0; t < TN; ++t) sw[t] = *reinterpret_cast<const u32x4*>(b + (T::BM + rw + 32 * t) * 16 * T::CH);
  };

  f32x16 acc[TN][TM] = {};
  constexpr int D1 = (T::D + 1) / 2, D0 = T::D - D1;   // issued in a last step, in the first that follows
  fetch_scales(0);
#pragma unroll
  for (int s = 0; s < NB; ++s)
#pragma unroll
    for (int d = 0; d < (s == NB - 1 ? D1 : T::D); ++d) fetch(s * T::BUF, d, s & 1);
  landed_and_met<(NB - 2) * T::D + D1>();
  read_scales(0);
#pragma unroll
  for (int r = 0; r < READS; ++r) read(0, 0, r);

  // Step J: its products, with a memory instruction or more behind each: a wave issues in order, and a block of them
  // ahead of the products leaves the matrix unit idle while their queues drain.  The READS reads of the next step go
  // first, so that they are over when they are needed, then ND DMA instructions.  The scales are in dword Q of sa and sw.
  uint32_t cur = 0, nxt = T::BUF, free_ = (NB - 1) * T::BUF;
  uint32_t ca[TM], cw[TN];
  auto pick = [&](int q) {   // this lane's blocks of a pair of steps are h and 2 + h of dword q: bytes 0 and 2 after the shift
#pragma unroll
    for (int t = 0; t < TM; ++t) ca[t] = sa[t][q] >> (8 * h);
#pragma unroll
    for (int t = 0; t < TN; ++t) cw[t] = sw[t][q] >> (8 * h);
  };
  auto step = [&](auto jj, auto nd, auto&& rd, auto&& dma) {
    constexpr int J = decltype(jj)::value, ND = decltype(nd)::value, OPS = READS + ND;
    constexpr int PER = (OPS + PRODUCTS - 1) / PRODUCTS;   // behind each product
    constexpr int EVERY = ND == 0 ? PRODUCTS + 1 : ND > PRODUCTS ? 1 : PRODUCTS / (ND ? ND : 1);   // PER = 1: a DMA instruction behind every so manyth
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
      const int x = i / TM, t = i % TM;
      acc[x][t] = mx_mfma<AF, F32, 2 * (J & 1)>(fw[J & 1][x], fa[J & 1][t], acc[x][t], cw[x], ca[t]);
      if (PER == 1) {
        if (i % EVERY == EVERY - 1 && i / EVERY < ND) dma(i / EVERY);
        else if (i - (i / EVERY < ND ? i / EVERY : ND) < READS) rd(i - (i / EVERY < ND ? i / EVERY : ND));
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
  using None = std::integral_constant<int, 0>;
  // One stage of parity PAR, its scales in dwords q .. of sa and sw.  No branch in it: the compiler would move products
  // below it, past the barrier.  At the barrier everything up to stage s + NB - 1 has been issued, and scales ahead of
  // the last of it, so stage s + 1 has landed when at most the stages after that are under way.
  auto stage = [&](auto par, int q, auto&& scales) {
    constexpr int PAR = decltype(par)::value;
    auto late = [&](int d) { fetch(free_, D1 + d, (PAR + NB - 1) & 1); };   // what the step before left of its stage
    auto inner = [&](auto jj) {
      constexpr int J = decltype(jj)::value;
      if (J % 2 == 0) pick(q + J / 2);
      step(jj, std::integral_constant<int, J == 0 ? D0 : 0>{}, [&](int r) { read(cur, J + 1, r); }, late);
    };
    for_each_index(inner, std::make_integer_sequence<int, SPS - 1>{});
    landed_and_met<(NB - 2) * T::D>();
    scales();   // the last step's are picked
    step(std::integral_constant<int, SPS - 1>{}, std::integral_constant<int, D1>{}, [&](int r) { read(nxt, 0, r); },
         [&](int d) { fetch(cur, d, (PAR + NB) & 1); });
    free_ = cur;
    cur = nxt;
    nxt = nxt + T::BUF == T::OS ? 0 : nxt + T::BUF;
  };
  // A group of scales lasts PG stages.  A chunk's last group is read at the end of the group before; a stage later
  // (every wave has read it) the next chunk is fetched, and lands by the end of the chunk.
  constexpr int PG = 8 / SPS, PC = T::CH * PG, QS = SPS / 2;   // stages per group and per chunk, dwords per stage
  const int full = steps / SPS;
  int s = 0;
  for (; s + PC <= full; s += PC)
    for_each_index([&](auto ii) {
      constexpr int I = decltype(ii)::value;
      stage(std::integral_constant<int, I % 2>{}, I % PG * QS, [&] {
        if (I % PG == PG - 1) read_scales((I / PG + 1) % T::CH);
        if (I == PC - PG) fetch_scales(s / PC + 1);
      });
    }, std::make_integer_sequence<int, PC>{});
  // what is left of the last chunk, a stage's scales at a time from LDS
  int left = 1;
  auto next_scales = [&] {
    const uint8_t* b = sm + T::OS + 4 * QS * left++;
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int k = 0; k < QS; ++k) sa[t][k] = *reinterpret_cast<const uint32_t*>(b + (ra + 32 * t) * 16 * T::CH + 4 * k);
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int k = 0; k < QS; ++k) sw[t][k] = *reinterpret_cast<const uint32_t*>(b + (T::BM + rw + 32 * t) * 16 * T::CH + 4 * k);
  };
#pragma unroll 1
  for (; s + 2 <= full; s += 2) {
    stage(std::integral_constant<int, 0>{}, 0, next_scales);
    stage(std::integral_constant<int, 1>{}, 0, next_scales);
  }
  if (s < full) stage(std::integral_constant<int, 0>{}, 0, next_scales);
  if (odd) {
    pick(0);
    step(std::integral_constant<int, 0>{}, None{}, [&](int r) { read(cur, 1, r); }, [](int) {});
    step(std::integral_constant<int, 1>{}, None{}, [](int) {}, [](int) {});
  }
  // Register 4 q + r of lane (lr, h): row lr of a, column 8 q + 4 h + r of w.  32 rows at a time go through LDS, each wave
  // in a part of its own, and out as whole rows of its tile (stored from the registers, 32 bytes to each of 32 rows an
  // instruction: M = 4352, N = 16384, K = 6144 235 us, so 231), past the L2, whose lines the operands need and which
  // would be written back in one go at the kernel's end (231 -> 221).  Nothing of the DMA may be under way when LDS is
  // used again, here or by the next workgroup.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  constexpr int ES = F32 ? 4 : 2, COLS = 32 * TN, PITCH = COLS * ES + 16, PER = 16 / ES;   // bytes; elements in 16
  static_assert(T::NW * 32 * PITCH <= T::LDS, "LDS");
  uint8_t* stage_out = sm + wave * 32 * PITCH;
  const int mw = m0 + 32 * TM * wm, nw = n0 + COLS * wn;
  const bool wide = p.ldy % PER == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
  f32x4 bias[TN][4];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = nw + 32 * i + 8 * (r / 4) + 4 * h + r % 4;
      bias[i][r / 4][r % 4] = p.bias && c < p.N ? bf16f(p.bias[c]) : 0.0f;
    }
#pragma unroll
  for (int t = 0; t < TM; ++t) {
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[i][t][4 * q + r] + bias[i][q][r];
        uint8_t* to = stage_out + lr * PITCH + (32 * i + 8 * q + 4 * h) * ES;
        if (F32) *reinterpret_cast<f32x4*>(to) = v;
        else *reinterpret_cast<u32x2*>(to) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own writes, read by its other lanes
    const int rows = min(32, p.M - (mw + 32 * t)), cols = min(COLS, p.N - nw);
    uint8_t* out = static_cast<uint8_t*>(p.y) + ((long)(mw + 32 * t) * p.ldy + nw) * ES;
    if (wide && cols % PER == 0) {
      constexpr int LPR = COLS / PER;   // lanes per row
#pragma unroll
      for (int k = 0; k < 32 * LPR / 64; ++k) {
        const int row = (64 * k + lane) / LPR, c = (64 * k + lane) % LPR;
        const u32x4 v = *reinterpret_cast<const u32x4*>(stage_out + row * PITCH + 16 * c);
        if (row < rows && PER * c < cols) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(out + (long)row * p.ldy * ES + 16 * c));
      }
    } else {
#pragma unroll 4
      for (int k = 0; k < 32 * COLS / 64; ++k) {
        const int row = (64 * k + lane) / COLS, c = (64 * k + lane) % COLS;
        const uint8_t* from = stage_out + row * PITCH + c * ES;
        if (row < rows && c < cols) {
          uint8_t* to = out + (long)row * p.ldy * ES + c * ES;
          if (F32) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
          else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// acc += w a of 16 x 16 on a step of 128: lane l supplies row l % 16 of each, E2M1 the 32 codes k = 32 (l / 16) ..,
// E4M3 k = 16 (l / 16) .. + 15 and 64 + 16 (l / 16) .. + 15; the scale (byte 0) of its row's block l / 16.
template <int AF, bool EXACT>
__device__ __forceinline__ f32x4 mx_mfma16(const MxFrag<MX_E2M1>& w, const MxFrag<AF>& a, f32x4 acc, uint32_t ws,
                                           uint32_t as) {
  if constexpr (EXACT && AF == MX_E4M3) {
    MxFrag<AF> hi, lo;
    split(a, hi, lo);
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(lo), acc, 4, 0, 0, (int)ws, 0, (int)as);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(hi), acc, 4, 0, 0, (int)ws, 0, (int)as);
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(a), acc, 4, AF == MX_E4M3 ? 0 : 4, 0,
                                                            (int)ws, 0, (int)as);
  }
}

// Few rows of a (16 at most): what counts is reading w once, from as many places at once as possible.  A workgroup of
// 8 waves takes 16 columns of the output and all of K; the waves take units of 256 columns of K in turn (whole cache
// lines of w) and add their sums through LDS in wave order.  Each wave has a ring of U units in LDS to itself, filled
// by DMA whose lanes read whole lines (operands loaded straight to registers, 16 bytes from each of 64 lines an
// instruction, took twice as long), so the waves need no barrier before the sums.  MR = 8 or 16 rows of a are held;
// rows beyond M repeat the last.
template <int AF, int MR, int U>
struct MxRows {
  static constexpr int NW = 8;
  static constexpr int RA = AF == MX_E4M3 ? 256 : 128, OA = 2048, OSC = OA + MR * RA, UNIT = OSC + 256;
  static constexpr int DA = MR * RA / 1024, D = 2 + DA + 1;   // DMA instructions of a unit: w, a, scales
  static constexpr int LDS = NW * U * UNIT;
  static_assert(LDS <= 160 * 1024 && NW * 1024 <= LDS, "LDS");
};

template <int AF, bool F32, int MR, int U>
__global__ void __launch_bounds__(512) mx_gemm_rows_kernel(MxGemmParams p) {
  using T = MxRows<AF, MR, U>;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16;
  const int kp = (int)mx_kp(p.K), sp = (int)mx_sp(p.K), nst = kp / 128, units = (nst + 1) / 2;
  const long pa = mx_row_bytes(p.K, AF), pw = kp / 2;
  const uint32_t lds0 = lds_offset(sm) + wave * U * T::UNIT;
  const uint8_t* mine = sm + wave * U * T::UNIT;

  // A DMA lane's row and chunk of 16 bytes; chunk c of a row lies at slot c ^ f(row), f = row / 2 mod 8 (rows of 128
  // bytes) or row (rows of 256): sixteen rows' chunk over all banks.
  constexpr int CA = T::RA / 16;
  uint32_t off_w[2], off_a[T::DA];
  int chunk_w[2], chunk_a[T::DA];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const int row = 8 * d + lane / 8;
    chunk_w[d] = lane % 8 ^ (row >> 1 & 7);
    off_w[d] = (uint32_t)(min(row, p.N - n0 - 1) * pw);
  }
#pragma unroll
  for (int d = 0; d < T::DA; ++d) {
    const int row = (64 / CA) * d + lane / CA;
    chunk_a[d] = lane % CA ^ (AF == MX_E4M3 ? row & 15 : row >> 1 & 7);
    off_a[d] = (uint32_t)(min(row, p.M - 1) * pa);
  }
  const uint8_t* src_w = p.w + (long)n0 * pw;
  // scale dwords of a unit: lanes 0..31 w's rows, then a's, each row's first step and then its second
  const uint8_t* ssrc = (lane < 32 ? p.ws + (long)min(n0 + lr, p.N - 1) * sp : p.as + (long)min(lr, p.M - 1) * sp) +
                        4 * (lane >> 4 & 1);
  auto fetch = [&](int unit, int buf) {
    const uint32_t to = lds0 + buf * T::UNIT;
    const bool half = 2 * unit + 1 >= nst;   // an odd last step: the unit's second half is its first again
#pragma unroll
    for (int d = 0; d < 2; ++d)
      dma16(src_w, off_w[d] + 128 * unit + 16 * (half ? chunk_w[d] & 3 : chunk_w[d]), to + 1024 * d);
#pragma unroll
    for (int d = 0; d < T::DA; ++d)
      dma16(p.a, off_a[d] + T::RA * unit + 16 * (half ? chunk_a[d] & (CA / 2 - 1) : chunk_a[d]), to + T::OA + 1024 * d);
    const uint8_t* at = ssrc + 8 * unit;
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(at), "{m0}"(to + T::OSC) : "memory");
  };

  const int mine_units = wave < units ? (units - wave + T::NW - 1) / T::NW : 0;
  f32x4 acc = {};
  const int ma = min(lr, MR - 1);
  if (mine_units) {
    // units past the last are the last again, into a buffer that is not read: the waits count the same loads throughout
    auto unit_of = [&](int i) { return wave + T::NW * min(i, mine_units - 1); };
#pragma unroll
    for (int i = 0; i < U; ++i) fetch(unit_of(i), i);
    int buf = 0;
#pragma unroll 1
    for (int i = 0; i < mine_units; ++i) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((U - 1) * T::D) : "memory");
      const uint8_t* u = mine + buf * T::UNIT;
      MxFrag<MX_E2M1> fw[2];
      MxFrag<AF> fa[2];
      uint32_t sw[2], sa[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        fw[j].q[0] = *reinterpret_cast<const u32x4*>(u + 128 * lr + 16 * ((4 * j + b) ^ (lr >> 1 & 7)));
        const uint8_t* row = u + T::OA + T::RA * ma;
        if (AF == MX_E4M3) {
          fa[j].q[0] = *reinterpret_cast<const u32x4*>(row + 16 * ((8 * j + b) ^ ma));
          fa[j].q[AF == MX_E4M3] = *reinterpret_cast<const u32x4*>(row + 16 * ((8 * j + 4 + b) ^ ma));
        } else {
          fa[j].q[0] = *reinterpret_cast<const u32x4*>(row + 16 * ((4 * j + b) ^ (ma >> 1 & 7)));
        }
        sw[j] = *reinterpret_cast<const uint32_t*>(u + T::OSC + 4 * (16 * j + lr)) >> (8 * b);
        sa[j] = *reinterpret_cast<const uint32_t*>(u + T::OSC + 128 + 4 * (16 * j + lr)) >> (8 * b);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // all of the unit is in registers
      fetch(unit_of(i + U), buf);
      buf = buf + 1 == U ? 0 : buf + 1;
      acc = mx_mfma16<AF, F32>(fw[0], fa[0], acc, sw[0], sa[0]);
      if (2 * unit_of(i) + 1 < nst) acc = mx_mfma16<AF, F32>(fw[1], fa[1], acc, sw[1], sa[1]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  __syncthreads();   // every ring is done with; their memory takes the sums
  f32x4* red = reinterpret_cast<f32x4*>(sm);
  red[64 * wave + lane] = acc;
  __syncthreads();
  // register r of lane (lr, b): row lr of a, column 4 b + r of w
  const int m = tid >> 4, n = tid & 15;
  if (m >= p.M || m >= 16 || n0 + n >= p.N) return;
  float v = 0.0f;
#pragma unroll
  for (int k = 0; k < T::NW; ++k) v += reinterpret_cast<const float*>(sm)[4 * (64 * k + 16 * (n / 4) + m) + n % 4];
  if (p.bias) v += bf16f(p.bias[n0 + n]);
  const long at = (long)m * p.ldy + n0 + n;
  if (F32) static_cast<float*>(p.y)[at] = v;
  else static_cast<uint16_t*>(p.y)[at] = (uint16_t)pack_bf16x2(v, 0.0f);
}

template <int AF, bool F32, int TM, int TN, int WM, int WN, int SPS, int NB>
hipError_t launch_tile(const MxGemmParams& p, hipStream_t st) {
  using T = MxTile<AF, F32, TM, TN, WM, WN, SPS, NB>;
  const long nbm = (p.M + T::BM - 1) / T::BM, nbn = (p.N + T::BN - 1) / T::BN;
  if (nbm * nbn > INT32_MAX) return hipErrorInvalidValue;
  mx_gemm_tile_kernel<AF, F32, TM, TN, WM, WN, SPS, NB>
      <<<(unsigned)(nbm * nbn), 64 * WM * WN, 0, st>>>(p, (int)nbm, (int)nbn, 4);
  return hipGetLastError();
}

template <int AF, bool F32, int MR, int U>
hipError_t launch_rows(const MxGemmParams& p, hipStream_t st) {
  mx_gemm_rows_kernel<AF, F32, MR, U><<<(unsigned)((p.N + 15) / 16), 512, 0, st>>>(p);
  return hipGetLastError();
}

template <int AF, bool F32>
hipError_t launch_kernel(int tile, const MxGemmParams& p, hipStream_t st) {
  constexpr bool E8 = AF == MX_E4M3;
  switch (tile) {
    case MX_ROWS:
      if constexpr (!E8)
        if (p.M > 8) return launch_rows<AF, F32, 16, 2>(p, st);
      return launch_rows<AF, F32, 8, E8 ? 2 : 3>(p, st);
    case 0: return launch_tile<AF, F32, 1, 1, 2, 2, E8 ? 2 : 4, E8 ? 4 : 3>(p, st);
    case 1: return launch_tile<AF, F32, E8 ? 1 : 2, E8 ? 2 : 1, 2, 2, E8 ? 2 : 4, E8 ? 4 : 3>(p, st);
    case 2: return launch_tile<AF, F32, 2, 2, 2, 2, E8 ? 2 : 4, 3>(p, st);
    // E4M3 with float32 output needs registers for the halves of its operands
    default: return launch_tile<AF, F32, E8 && F32 ? 2 : 4, 4, 2, 2, 2, E8 && !F32 ? 3 : 4>(p, st);
  }
}

// Block tiles: rows of a, of w, workgroups that share a CU, and microseconds per 1024 columns of K with n of them on a
// CU (us[n - 1]); a round takes 2 us besides.  As measured at K = 6144 (M x N and us of the tiles in order; E2M1: 77 x
// 6144 9.2 10.5 14.0 34, 256 x 6144 13.3 11.5 14.7 34, 256 x 16384 26.1 21.9 18.4 38, 4352 x 16384 - - 306 231; E4M3:
// 77 x 6144 9.9 12.6 18.9 30, 256 x 6144 17.4 15.0 20.5 30, 256 x 16384 34.5 28.6 24.9 35, 4352 x 16384 - - 375 330).
struct MxTileCost {
  int rows, cols, slots;
  float us[3];
};
const MxTileCost kTiles[2][MX_TILES] = {
    {{64, 64, 3, {1.2f, 1.9f, 2.9f}}, {128, 64, 2, {1.6f, 3.2f}}, {128, 128, 1, {2.75f}}, {256, 256, 1, {7.2f}}},
    {{64, 64, 3, {1.35f, 2.6f, 3.9f}}, {64, 128, 2, {2.1f, 4.4f}}, {128, 128, 2, {3.8f, 6.6f}}, {256, 256, 1, {10.3f}}}};

float tile_us(const MxTileCost& t, long tiles, int K) {
  const long whole = tiles / (256 * t.slots), rest = (tiles % (256 * t.slots) + 255) / 256;
  return whole * (2.0f + t.us[t.slots - 1] * (K / 1024.0f)) + (rest ? 2.0f + t.us[rest - 1] * (K / 1024.0f) : 0.0f);
}

long tiles_of(const MxTileCost& t, long M, long N) { return ((M + t.rows - 1) / t.rows) * ((N + t.cols - 1) / t.cols); }

struct MxChoice {
  int tile;
  float us;
  int large;   // rows that go to the large tiles ahead of a launch of smaller ones for the others, 0: one launch
};

// Up to 8 rows of a (16 of E2M1), unless 64 x 64 tiles fill the CUs, run the rows kernel (M = 1, K = 6144, E2M1 and
// E4M3: N = 1536 3.6 and 3.5 us, the tiles 8.1, 7.2; N = 6144 6.6 and 6.3, the tiles 8.8, 9.4; N = 12288 9.8 and 9.4,
// the tiles 9.5, 10.2; N = 16384 11.9 and 11.3, the tiles 10.7, 10.9); else the tile that takes least by its rounds.
// 9 to 16 rows of E4M3 would hold twice the bytes of a in every ring and gain at some sizes only (16 rows, this
// kernel and the tiles: N = 6144 with K = 1024 4.5 3.8, K = 6144 9.8 9.6, K = 16384 16.8 20.6; K = 6144 with N = 1536
// 4.7 7.3, N = 12288 14.4 10.6): they take the tiles.  As the last rows of a split the rows kernel counts 10 us (it
// takes 3.5 to 12.8 up to K = 16384).  A last round of large tiles that leaves most CUs idle costs nearly as much as
// a full one, so the rows behind the whole rounds go to smaller tiles where that is less: M = 4352, N = 16384, K =
// 6144 is 4 rounds and 64 tiles more, 241 us in one launch, 228 with the last 256 rows on 128 x 128 tiles (E4M3 333,
// 314); M = 3000, N = K = 6144 85, 67.
MxChoice choose(long M, long N, int K, int fmt) {
  const int e8 = fmt == MX_E4M3;
  if (M <= (e8 ? 8 : 16) && N < 64 * 256) return {MX_ROWS, 10.0f, 0};
  MxChoice best{0, tile_us(kTiles[e8][0], tiles_of(kTiles[e8][0], M, N), K), 0};
  for (int i = 1; i < MX_TILES; ++i) {
    const float us = tile_us(kTiles[e8][i], tiles_of(kTiles[e8][i], M, N), K);
    if (us < best.us) best = {i, us, 0};
  }
  const MxTileCost& t = kTiles[e8][MX_TILES - 1];
  const long nbn = (N + t.cols - 1) / t.cols, blocks = tiles_of(t, M, N) / 256 * 256 / nbn, rows = blocks * t.rows;
  if (blocks > 0 && rows < M) {
    const float us = tile_us(t, blocks * nbn, K) + choose(M - rows, N, K, fmt).us + 2.0f;
    if (us < 0.97f * best.us) best = {MX_TILES - 1, us, (int)rows};
  }
  return best;
}

template <int AF, bool F32>
hipError_t launch_any(const MxGemmParams& p, hipStream_t st) {
  const MxChoice c = choose(p.M, p.N, p.K, AF);
  if (c.large == 0) return launch_kernel<AF, F32>(c.tile, p, st);
  MxGemmParams q = p;
  q.M = c.large;
  if (hipError_t e = launch_kernel<AF, F32>(c.tile, q, st)) return e;
  q.M = p.M - c.large;
  q.a += c.large * mx_row_bytes(p.K, AF);
  q.as += c.large * mx_sp(p.K);
  q.y = static_cast<uint8_t*>(p.y) + c.large * p.ldy * (F32 ? 4 : 2);
  return launch_any<AF, F32>(q, st);
}

}  // namespace

int mx_gemm_tile(int M, int N, int K, int fmt, int& rows, int& cols, bool& split) {
  const MxChoice c = choose(M, N, K, fmt);
  split = c.large > 0;
  rows = c.tile == MX_ROWS ? (M <= 8 ? 8 : 16) : kTiles[fmt == MX_E4M3][c.tile].rows;
  cols = c.tile == MX_ROWS ? 16 : kTiles[fmt == MX_E4M3][c.tile].cols;
  return c.tile;
}

hipError_t launch_mx_gemm(const MxGemmParams& p, int fmt, bool out_f32, hipStream_t st) {
  if (fmt == MX_E4M3) return out_f32 ? launch_any<MX_E4M3, true>(p, st) : launch_any<MX_E4M3, false>(p, st);
  return out_f32 ? launch_any<MX_E2M1, true>(p, st) : launch_any<MX_E2M1, false>(p, st);
}

}  // namespace svdq
