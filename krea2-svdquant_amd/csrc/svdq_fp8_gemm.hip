// Product of an E4M3 activation a [M, kp] (a float32 scale for each row and 128 columns, [kp / 128, M]) with an E4M3 weight
// w [N, kp] (a float32 scale for each 128 x 128 block, [ceil(N / 128), kp / 128]):
//   y[m, n] = sum over blocks b of sa[b, m] sw[n / 128, b] (sum over the block's 128 k of a[m, k] w[n, k])  (+ bias[n])
// in float32, rounded once to bf16.
//
// v_mfma_f32_16x16x128 sums exactly one block: its result is scaled and added to the accumulator by one FMA per value
// (the scales are any float32, so the matrix instruction's own power-of-two scales cannot take them).  The weight is the
// first operand, so a lane holds one row m and four consecutive n: its scales are one value per row of tiles, times one per
// block that is the same for the whole wave.  Their product is a float32 too: blocks of which it is 2^128 and more are not finite, and
// of one below 2^-126 the part is off by up to 2^-150 x 128 x 448^2.  (The scales' powers of two as the instruction's own, and what
// they are between powers of two in the FMA, would keep the whole range: 4352 x 16384, K = 6144 391 us, so 385; 40 x 6144 10.0, 9.5.)
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

__device__ __forceinline__ void dma16_at(const void* at, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(at), "{m0}"(lds) : "memory");
}

template <class F, int... I>
__device__ __forceinline__ void for_each_index(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// Block tile BM x BN (BM = 16 TM WM rows of a, BN = 16 TN WN rows of w, a wave's 16 TN within one block of 128), WM x WN
// waves, a ring of NB stages of 128 columns in LDS filled by DMA.  Rows of 128 bytes lie in chunks of 16, chunk c at slot
// c ^ (row / 2 mod 8).
//
// A stage's products go by pairs of tiles of w, TM tiles of a within a pair, so that the operands of a have time to be
// replaced: those of the next stage are read behind their last use in the last pair, the operands of w a pair ahead.  Each product is
// followed by the scaling of the one two before it and by a memory instruction or two; a block of them would leave the
// matrix unit idle while their queues drain.  Ahead of the last pair everything of the stage has been read: there the wave
// waits for the next stage's bytes and for the other waves, and the buffer takes stage s + NB.
//
// 256 x 256 at 4096 x 16384, K = 6144: 345 us, 2390 TFLOP/s; the products with their FMAs alone reach 3500 from registers, at
// a clock that falls under them.
template <int TM, int TN, int WM, int WN, int NB>
struct Fp8Tile {
  static constexpr int NW = WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN;
  static constexpr int TA = BM / 8, TB = BN / 8;                            // DMA instructions of 1024 bytes
  static constexpr int DA = TA / NW, D = DA + TB / NW + 1;                  // per wave and stage, the last one of scales
  static constexpr int BUF = (TA + TB) * 1024, OS = NB * BUF, LDS = OS + NB * NW * 256;
  static constexpr int GROUPS = 160 * 1024 / LDS;                           // workgroups that a CU's LDS holds
  static constexpr int PITCH = 32 * TN + 16;                                // of 16 rows of the output in LDS
  static_assert(LDS <= 160 * 1024 && NW * 16 * PITCH <= LDS, "LDS");
  static_assert(TA % NW == 0 && TB % NW == 0 && 128 % (16 * TN) == 0 && TN % 4 == 0 && TM <= 4 && NB >= 2, "whole instructions");
  static_assert(NB * D <= 63, "vmcnt counts to 63");
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
  const int chunk = lane % 8 ^ (lane / 8 >> 1 & 3);   // row / 2 mod 8 of row 8 i + lane / 8: 4 (i & 1) more
  uint32_t off[T::D - 1];
#pragma unroll
  for (int d = 0; d < T::D - 1; ++d) {
    const bool a = d < T::DA;
    const int i = wave + T::NW * (a ? d : d - T::DA), row = 8 * i + lane / 8;
    off[d] = (uint32_t)((long)min(row, (a ? p.M - m0 : p.N - n0) - 1) * kp + 16 * (chunk ^ (i & 1 ? 4 : 0)));
  }
  const uint8_t *src_a = p.a + (long)m0 * kp, *src_w = p.w + (long)n0 * kp;
  const int mw = m0 + 16 * TM * wm, nw = n0 + 16 * TN * wn;
  const float* src_s = p.as + min(mw + min(lane, 16 * TM - 1), p.M - 1);
  int ahead = 0;
  // this wave's d-th instruction of the stage `ahead`; past the last one that again, so that the waits count the same
  // loads throughout
  auto fetch = [&](int buf, int d) {
    if (d == T::D - 1) {
      dma4_at(src_s, lds0 + T::OS + 256 * (buf * T::NW + wave));
      if (++ahead < nst) {
        src_a += 128;
        src_w += 128;
        src_s += p.lds;
      }
    } else {
      dma16(d < T::DA ? src_a : src_w, off[d],
            lds0 + buf * T::BUF + 1024 * (d < T::DA ? wave + T::NW * d : T::TA + wave + T::NW * (d - T::DA)));
    }
  };
  const float* wsrow = p.ws + (long)min(nw / 128, (p.N - 1) / 128) * nst;
  float wscales = wsrow[min(lane, nst - 1)];   // of stages s .. s + 63
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(wscales)::"memory");

  constexpr int P = TN / 2, S = 2 * TM, READS = 4 + 2 * TM;
  constexpr int D0 = T::D / 2;   // instructions issued in a last pair, the others in the first pair that follows
  Fp8Frag fa[TM], fw[2][2];
  f32x4 acc[TN][TM] = {}, v[4] = {};
  float sc[TM], sraw[TM], scl = 0.0f;
  const uint32_t turn = 16 * (b ^ (lr >> 1 & 7));
  const uint8_t *pa = nullptr, *pw = nullptr;   // this lane's chunk in its row of the first tiles
  const float* ps = nullptr;
  auto at_buffer = [&](int buf) {
    pa = sm + buf * T::BUF + (16 * TM * wm + lr) * 128 + turn;
    pw = sm + buf * T::BUF + T::TA * 1024 + (16 * TN * wn + lr) * 128 + turn;
    ps = reinterpret_cast<const float*>(sm + T::OS + 256 * (buf * T::NW + wave)) + lr;
  };
  const int other = 64 - 2 * (turn & 64);   // chunk c ^ 4
  auto read_w = [&](int pair, int i) {      // i-th of the four reads of a pair
    fw[pair & 1][i / 2].q[i % 2] = *reinterpret_cast<const u32x4*>(pw + 2048 * (2 * pair + i / 2) + (i % 2 ? other : 0));
  };
  auto read_a = [&](int i) { fa[i / 2].q[i % 2] = *reinterpret_cast<const u32x4*>(pa + 2048 * (i / 2) + (i % 2 ? other : 0)); };
  auto scaled = [&](int slot, float s) {    // the product of a slot into its accumulator
    const int pair = slot / S, j = slot % S;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[2 * pair + j % 2][j / 2][r] = __builtin_fmaf(v[slot & 3][r], s, acc[2 * pair + j % 2][j / 2][r]);
  };

#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int d = 0; d < (i == NB - 1 ? D0 : T::D); ++d) fetch(i, d);
  landed_and_met<(NB - 2) * T::D + D0>();
  at_buffer(0);
#pragma unroll
  for (int i = 0; i < 4; ++i) read_w(0, i);
#pragma unroll
  for (int i = 0; i < 2 * TM; ++i) read_a(i);
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    sraw[t] = ps[16 * t];
    sc[t] = sraw[t] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wscales), 0));
  }
  int cur = 0, last = NB - 1;   // the buffer of this stage, and the one that is being filled
#pragma unroll 1
  for (int s = 0; s < nst; ++s) {
    if ((s + 1) % 64 == 0) {   // waited for in here: a wait behind it would be for every stage's loads
      wscales = wsrow[min(s + 1 + lane, nst - 1)];
      asm volatile("s_waitcnt vmcnt(0)" : "+v"(wscales)::"memory");
    }
    const float sw = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wscales), (s + 1) & 63));
    const int nxt = cur + 1 == NB ? 0 : cur + 1;
    for_each_index([&](auto pp) {
      constexpr int pair = decltype(pp)::value;
      constexpr bool final = pair == P - 1;
      if (final) {
        landed_and_met<(NB - 2) * T::D>();
        at_buffer(nxt);
      }
      // the memory instructions of this pair, those of slot j behind its product
      constexpr int ND = final ? D0 : pair == 0 ? T::D - D0 : 0;
      constexpr int PER = (READS + S - 1) / S;
#pragma unroll
      for (int j = 0; j < S; ++j) {
        constexpr int slots = P * S;
        const int slot = pair * S + j;
        __builtin_amdgcn_s_setprio(1);   // a wave that has a product to issue goes first: 340 -> 336 us at 4096 x 16384 x 6144
        v[slot & 3] = fp8_mfma16(fw[pair & 1][j % 2], fa[j / 2]);
        __builtin_amdgcn_s_setprio(0);
        if (slot < 2) scaled(slots - 2 + slot, scl);
        else scaled(slot - 2, sc[(slot - 2) % S / 2]);
        if (final) {
          // four of w's, then a's behind their last use
#pragma unroll
          for (int i = 0; i < READS; ++i) {
            const int at_ = i < 4 ? i / PER : (i - 4) / 2 * 2 + 1 > i / PER ? (i - 4) / 2 * 2 + 1 : i / PER;
            if ((at_ < S ? at_ : S - 1) == j) {
              if (i < 4) read_w(0, i);   // pair P is even: the next stage's pair 0 goes to buffer 0
              else read_a(i - 4);
            }
          }
          if (j < TM) sraw[j] = ps[16 * j];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i * (S < 4 ? S : 4) / 4 == j) read_w(pair + 1, i);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
          if (d * S / (ND ? ND : 1) == j) fetch(final ? cur : last, final ? d : D0 + d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }, std::make_integer_sequence<int, P>{});
    scl = sc[TM - 1];
#pragma unroll
    for (int t = 0; t < TM; ++t) sc[t] = sraw[t] * sw;
    last = cur;
    cur = nxt;
  }
  scaled(P * S - 2, scl);
  scaled(P * S - 1, scl);
  // Register r of lane (lr, b): row lr of a, column 4 b + r of w.  16 rows at a time go through LDS, each wave in a part of
  // its own, and out as whole rows of its tile past the L2, whose lines the operands need.  Nothing of the DMA may be under way when
  // LDS is used again, here or by the next workgroup.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  uint8_t* stage_out = sm + wave * 16 * T::PITCH;
  constexpr int COLS = 16 * TN, LPR = COLS / 8;   // lanes a row
  const bool wide = p.ldy % 8 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
  f32x4 bias[TN];
#pragma unroll
  for (int x = 0; x < TN; ++x)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = nw + 16 * x + 4 * b + r;
      bias[x][r] = p.bias && n < p.N ? bf16f(p.bias[n]) : 0.0f;
    }
  const int cols = min(COLS, p.N - nw);
#pragma unroll
  for (int t = 0; t < TM; ++t) {
#pragma unroll
    for (int x = 0; x < TN; ++x) {
      const f32x4 y = acc[x][t] + bias[x];
      *reinterpret_cast<u32x2*>(stage_out + lr * T::PITCH + 32 * x + 8 * b) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own writes, read by its other lanes
    const int rows = min(16, p.M - (mw + 16 * t));
    uint16_t* out = p.y + (long)(mw + 16 * t) * p.ldy + nw;
    if (wide && cols % 8 == 0) {
#pragma unroll
      for (int k = 0; k < 16 * LPR / 64; ++k) {
        const int row = (64 * k + lane) / LPR, c = (64 * k + lane) % LPR;
        const u32x4 y = *reinterpret_cast<const u32x4*>(stage_out + row * T::PITCH + 16 * c);
        if (row < rows && 8 * c < cols) __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(out + (long)row * p.ldy + 8 * c));
      }
    } else {
#pragma unroll 4
      for (int k = 0; k < 16 * COLS / 64; ++k) {
        const int row = (64 * k + lane) / COLS, c = (64 * k + lane) % COLS;
        if (row < rows && c < cols) out[(long)row * p.ldy + c] = *reinterpret_cast<const uint16_t*>(stage_out + row * T::PITCH + 2 * c);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// Four columns of a row, with the bias.
__device__ __forceinline__ void fp8_store4(const Fp8GemmParams& p, long m, int n, f32x4 y) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (p.bias && n + r < p.N) y[r] += bf16f(p.bias[n + r]);
  uint16_t* out = p.y + m * p.ldy + n;
  const u32x2 o = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  if (n + 3 < p.N && p.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % 8 == 0) {
    *reinterpret_cast<u32x2*>(out) = o;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < p.N) out[r] = (uint16_t)(o[r / 2] >> 16 * (r % 2));
  }
}

// Adds 8 waves' sums of 16 rows and 16 columns in wave order; memory: 8 KB of LDS that the waves have done with.
__device__ __forceinline__ void fp8_rows_sum(const Fp8GemmParams& p, uint8_t* sm, const f32x4& acc, int n0) {
  const int tid = threadIdx.x;
  __syncthreads();   // every ring is done with; their memory takes the sums
  reinterpret_cast<f32x4*>(sm)[tid] = acc;
  __syncthreads();
  // register r of lane (lr, b): row lr of a, column 4 b + r of w
  const int m = tid >> 4, n = tid & 15;
  if (m >= p.M || m >= 16 || n0 + n >= p.N) return;
  float y = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) y += reinterpret_cast<const float*>(sm)[4 * (64 * k + 16 * (n / 4) + m) + n % 4];
  if (p.bias) y += bf16f(p.bias[n0 + n]);
  p.y[(long)m * p.ldy + n0 + n] = (uint16_t)pack_bf16x2(y, 0.0f);
}

// Few rows of a (16 at most): what counts is reading w once, from as many places at once as possible.  A workgroup of
// 8 waves takes 16 columns of the output and all of K; the waves take blocks of 128 columns of K in turn (whole cache
// lines of w) and add their sums through LDS in wave order.  Each wave has a ring of U blocks in LDS to itself, filled
// by DMA, so the waves need no barrier before the sums.  MR = 8 or 16 rows of a are held; rows beyond M repeat the last.
// HBM-bound: 1 x 6144, K = 6144 8.1 us a call (4.7 TB/s), 16 rows 9.1; N = 16384 18.4 (5.5 TB/s).
template <int MR, int U>
struct Fp8Rows {
  static constexpr int NW = 8, OA = 2048, OSC = OA + 128 * MR, UNIT = OSC + 256;
  static constexpr int DA = MR / 8, D = 2 + DA + 1;   // DMA instructions of a block: w, a, scales
  static constexpr int LDS = NW * U * UNIT;
  static_assert(LDS <= 80 * 1024 && NW * 1024 <= LDS, "two workgroups share a CU's LDS");
};

template <int MR, int U>
__global__ void __launch_bounds__(512) fp8_gemm_rows_kernel(Fp8GemmParams p) {
  using T = Fp8Rows<MR, U>;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, kp = (int)fp8_kp(p.K), nst = kp / 128;
  const uint32_t lds0 = lds_offset(sm) + wave * U * T::UNIT;
  const uint8_t* mine = sm + wave * U * T::UNIT;
  const int chunk = lane % 8 ^ (lane / 8 >> 1 & 3);   // as in the tiles
  uint32_t off_w[2], off_a[T::DA];
#pragma unroll
  for (int d = 0; d < 2; ++d) off_w[d] = (uint32_t)(min(8 * d + lane / 8, p.N - n0 - 1) * (long)kp + 16 * (chunk ^ 4 * d));
#pragma unroll
  for (int d = 0; d < T::DA; ++d) off_a[d] = (uint32_t)(min(8 * d + lane / 8, p.M - 1) * (long)kp + 16 * (chunk ^ 4 * d));
  const uint8_t* src_w = p.w + (long)n0 * kp;
  // scales of a block: lanes 0..15 the rows', lane 16 the weight's
  const float* ssrc = lane < 16 ? p.as + min(lane, p.M - 1) : p.ws + (long)(n0 / 128) * nst;
  const long sstep = lane < 16 ? p.lds : 1;
  auto fetch = [&](int block, int buf) {
    const uint32_t to = lds0 + buf * T::UNIT;
#pragma unroll
    for (int d = 0; d < 2; ++d) dma16(src_w, off_w[d] + 128 * block, to + 1024 * d);
#pragma unroll
    for (int d = 0; d < T::DA; ++d) dma16(p.a, off_a[d] + 128 * block, to + T::OA + 1024 * d);
    dma4_at(ssrc + sstep * block, to + T::OSC);
  };
  const int count = wave < nst ? (nst - wave + T::NW - 1) / T::NW : 0;
  f32x4 acc = {};
  const int ma = min(lr, MR - 1), o0 = 16 * (b ^ (lr >> 1 & 7)), oa = 16 * (b ^ (ma >> 1 & 7));
  if (count) {
    // blocks past the last are the last again, into a buffer that is not read: the waits count the same loads throughout
    auto block_of = [&](int i) { return wave + T::NW * min(i, count - 1); };
#pragma unroll
    for (int i = 0; i < U; ++i) fetch(block_of(i), i);
    int buf = 0;
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((U - 1) * T::D) : "memory");
      const uint8_t* u = mine + buf * T::UNIT;
      Fp8Frag fw, fa;
      fw.q[0] = *reinterpret_cast<const u32x4*>(u + 128 * lr + o0);
      fw.q[1] = *reinterpret_cast<const u32x4*>(u + 128 * lr + (o0 ^ 64));
      fa.q[0] = *reinterpret_cast<const u32x4*>(u + T::OA + 128 * ma + oa);
      fa.q[1] = *reinterpret_cast<const u32x4*>(u + T::OA + 128 * ma + (oa ^ 64));
      const float* sc = reinterpret_cast<const float*>(u + T::OSC);
      const float s = sc[lr] * sc[16];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // all of the block is in registers
      fetch(block_of(i + U), buf);
      buf = buf + 1 == U ? 0 : buf + 1;
      const f32x4 v = fp8_mfma16(fw, fa);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(v[r], s, acc[r]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  fp8_rows_sum(p, sm, acc, n0);
}

// Strips, for outputs of few tiles (16 TM rows a workgroup, 16 TN columns): as with few rows, NW waves take blocks of all of K
// in turn, each with a ring of two in LDS to itself, and add their sums in wave order.  A lone tile spends 0.27 us on a
// block of K, most of it waiting at one point or another for DMA, LDS, the matrix unit and the other waves; here NW such
// chains run side by side without a barrier.  77 x 6144, K = 6144: 11.6 us, as 64 x 64 tiles 16.5 (w alone takes 7.1 to read).
template <int TM, int TN, int NW>
struct Fp8Strip {
  static constexpr int OA = 2048 * TN, OSC = OA + 2048 * TM, UNIT = OSC + 512;   // w, a, scales of 16 TM rows and w's
  static constexpr int D = 2 * TN + 2 * TM + 2;                                // DMA instructions of a block
  static constexpr int LDS = 2 * NW * UNIT;
  static_assert(LDS <= 160 * 1024 && TM * TN * 1024 <= 2 * UNIT && 16 * TM <= 128 && 128 % (16 * TN) == 0, "LDS");
};

template <int TM, int TN, int NW>
__global__ void __launch_bounds__(64 * NW) fp8_gemm_strip_kernel(Fp8GemmParams p) {
  using T = Fp8Strip<TM, TN, NW>;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16 * TN, m0 = blockIdx.y * 16 * TM, kp = (int)fp8_kp(p.K), nst = kp / 128;
  const uint32_t lds0 = lds_offset(sm) + wave * 2 * T::UNIT;
  const uint8_t* mine = sm + wave * 2 * T::UNIT;
  const int chunk = lane % 8 ^ (lane / 8 >> 1 & 3);   // as in the tiles
  uint32_t off_w[2 * TN], off_a[2 * TM];
#pragma unroll
  for (int d = 0; d < 2 * TN; ++d)
    off_w[d] = (uint32_t)(min(8 * d + lane / 8, p.N - n0 - 1) * (long)kp + 16 * (chunk ^ 4 * (d & 1)));
#pragma unroll
  for (int d = 0; d < 2 * TM; ++d)
    off_a[d] = (uint32_t)(min(8 * d + lane / 8, p.M - m0 - 1) * (long)kp + 16 * (chunk ^ 4 * (d & 1)));
  const uint8_t *src_w = p.w + (long)n0 * kp, *src_a = p.a + (long)m0 * kp;
  // scales of a block: the rows', and behind the last of them the weight's
  auto scale_at = [&](int i) { return i < 16 * TM ? p.as + min(m0 + i, p.M - 1) : p.ws + (long)(n0 / 128) * nst; };
  const float *src_s = scale_at(lane), *src_t = scale_at(64 + lane);
  const long step_s = lane < 16 * TM ? p.lds : 1, step_t = 64 + lane < 16 * TM ? p.lds : 1;
  auto fetch = [&](int block, int buf) __attribute__((always_inline)) {
    const uint32_t to = lds0 + buf * T::UNIT;
#pragma unroll
    for (int d = 0; d < 2 * TN; ++d) dma16(src_w, off_w[d] + 128 * block, to + 1024 * d);
#pragma unroll
    for (int d = 0; d < 2 * TM; ++d) dma16(src_a, off_a[d] + 128 * block, to + T::OA + 1024 * d);
    dma4_at(src_s + step_s * block, to + T::OSC);
    dma4_at(src_t + step_t * block, to + T::OSC + 256);
  };
  const int count = wave < nst ? (nst - wave + NW - 1) / NW : 0;
  f32x4 acc[TN][TM] = {};
  const uint32_t o0 = 128 * lr + 16 * (b ^ (lr >> 1 & 7));
  if (count) {
    // blocks past the last are the last again, into a buffer that is not read: the waits count the same loads throughout
    auto block_of = [&](int i) { return wave + NW * min(i, count - 1); };
    fetch(block_of(0), 0);
    fetch(block_of(1), 1);
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::D) : "memory");
      const uint8_t* u = mine + (i & 1) * T::UNIT;
      Fp8Frag fw[TN], fa[TM];
      float s[TM];
#pragma unroll
      for (int x = 0; x < TN; ++x) {
        fw[x].q[0] = *reinterpret_cast<const u32x4*>(u + 2048 * x + o0);
        fw[x].q[1] = *reinterpret_cast<const u32x4*>(u + 2048 * x + (o0 ^ 64));
      }
      const float* sc = reinterpret_cast<const float*>(u + T::OSC);
      const float ws = sc[16 * TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        fa[t].q[0] = *reinterpret_cast<const u32x4*>(u + T::OA + 2048 * t + o0);
        fa[t].q[1] = *reinterpret_cast<const u32x4*>(u + T::OA + 2048 * t + (o0 ^ 64));
        s[t] = sc[16 * t + lr] * ws;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // all of the block is in registers
      __builtin_amdgcn_sched_barrier(0);
      fetch(block_of(i + 2), i & 1);
#pragma unroll
      for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int x = 0; x < TN; ++x) {
          const f32x4 v = fp8_mfma16(fw[x], fa[t]);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[x][t][r] = __builtin_fmaf(v[r], s[t], acc[x][t][r]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  __syncthreads();   // every ring is done with; their memory takes the sums
  f32x4* sums = reinterpret_cast<f32x4*>(sm);
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int x = 0; x < TN; ++x) sums[64 * (TM * TN * wave + TN * t + x) + lane] = acc[x][t];
  __syncthreads();
  // register r of lane (lr, b): row lr of a, column 4 b + r of w
#pragma unroll
  for (int q = wave; q < TM * TN; q += NW) {
    const int m = m0 + 16 * (q / TN) + lr, n = n0 + 16 * (q % TN) + 4 * b;
    f32x4 y = {};
#pragma unroll
    for (int k = 0; k < NW; ++k) y += sums[64 * (TM * TN * k + q) + lane];
    if (m < p.M) fp8_store4(p, m, n, y);
  }
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// The scale of a row's block that lanes l, l ^ 16, l ^ 32, l ^ 48 hold 32 bf16 values each of.
__device__ __forceinline__ float row4_scale(const u32x4 (&v)[4]) {
  u16x2 part[4] = {};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    part[j % 4] = __builtin_elementwise_max(part[j % 4], __builtin_bit_cast(u16x2, v[j / 4][j % 4] & 0x7FFF7FFFu));
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(part[0], part[1]), __builtin_elementwise_max(part[2], part[3]));
  uint32_t top = max((uint32_t)m[0], (uint32_t)m[1]);
  if (__any(top >= 0x7F80u)) {   // values that are not finite: they say nothing about the scale
    top = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t d = v[j / 4][j % 4];
      top = max(top, max(fp8_magnitude(bf16lo(d)), fp8_magnitude(bf16hi(d))) >> 16);
    }
  }
  uint32_t other = top;
  permlane16_swap(top, other);
  top = other = max(top, other);
  permlane32_swap(top, other);
  return fp8_scale(max(top, other) << 16);
}

// The same of up to four rows of a bf16 activation, encoded by every workgroup for itself: K % 128 = 0, rows of x on 16 bytes.
// A lane holds 32 of a block's 128 values of its row, and four lanes agree on the scale.  The conversion rounds as that of the
// quantising kernel, so the sums are the same.  A block is encoded while its part of w is on its way; that takes longer than the wait,
// but less than a launch: one row, K = 6144, N = 6144 9.3 us and (two launches) 10.2, N = 1536 5.4 and 8.0, N = 16384 19.8 and 20.6, four
// rows, N = 6144 9.5 and 10.4.  Built for eight rows, N = 16384 took 24.6 and in two launches 23.3, so more than four go the other way.
struct Fp8RowsOf {
  static constexpr int MR = 4, NW = 8, U = 3, OA = 2048, OSC = OA + 256 * MR, UNIT = OSC + 256;
  static constexpr int D = 2 + 1 + 1;   // DMA instructions of a block: w, x, the weight's scale
  static constexpr int LDS = NW * U * UNIT;
  static_assert(LDS <= 80 * 1024 && NW * 1024 <= LDS, "two workgroups share a CU's LDS");
};

__global__ void __launch_bounds__(512) fp8_linear_rows_kernel(Fp8GemmParams p, const uint16_t* __restrict__ x, long ldx) {
  using T = Fp8RowsOf;
  constexpr int U = T::U;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, kp = p.K, nst = kp / 128;
  const uint32_t lds0 = lds_offset(sm) + wave * U * T::UNIT;
  const uint8_t* mine = sm + wave * U * T::UNIT;
  const int chunk = lane % 8 ^ (lane / 8 >> 1 & 3);
  uint32_t off_w[2];
#pragma unroll
  for (int d = 0; d < 2; ++d) off_w[d] = (uint32_t)(min(8 * d + lane / 8, p.N - n0 - 1) * (long)kp + 16 * (chunk ^ 4 * d));
  const uint16_t* src_x = x + min(lane / 16, p.M - 1) * ldx + 8 * (lane % 16);
  const uint8_t* src_w = p.w + (long)n0 * kp;
  const float* src_s = p.ws + (long)(n0 / 128) * nst;
  auto fetch = [&](int block, int buf) __attribute__((always_inline)) {
    const uint32_t to = lds0 + buf * T::UNIT;
    dma16_at(src_x + 128 * block, to + T::OA);
#pragma unroll
    for (int d = 0; d < 2; ++d) dma16(src_w, off_w[d] + 128 * block, to + 1024 * d);
    dma4_at(src_s + block, to + T::OSC);
  };
  const int count = wave < nst ? (nst - wave + T::NW - 1) / T::NW : 0;
  f32x4 acc = {};
  const int o0 = 16 * (b ^ (lr >> 1 & 7)), ox = 256 * (lr % T::MR) + 32 * b;
  if (count) {
    auto block_of = [&](int i) { return wave + T::NW * min(i, count - 1); };
#pragma unroll
    for (int i = 0; i < U; ++i) fetch(block_of(i), i);
    int buf = 0;
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      const uint8_t* u = mine + buf * T::UNIT;
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((U - 1) * T::D + 3) : "memory");   // x is there, w not yet
      Fp8Frag fw, fa;
      u32x4 v[4];   // values 16 b .. 16 b + 15, 64 + 16 b .. 64 + 16 b + 15
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const u32x4*>(u + T::OA + ox + 128 * (j / 2) + 16 * (j % 2));
      const float s = row4_scale(v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        fa.q[j / 2][2 * (j % 2)] = fp8_encode_bf16x4(v[j][0], v[j][1], s);
        fa.q[j / 2][2 * (j % 2) + 1] = fp8_encode_bf16x4(v[j][2], v[j][3], s);
      }
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((U - 1) * T::D) : "memory");
      fw.q[0] = *reinterpret_cast<const u32x4*>(u + 128 * lr + o0);
      fw.q[1] = *reinterpret_cast<const u32x4*>(u + 128 * lr + (o0 ^ 64));
      const float ws = *reinterpret_cast<const float*>(u + T::OSC);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // all of the block is in registers
      fetch(block_of(i + U), buf);
      buf = buf + 1 == U ? 0 : buf + 1;
      const f32x4 y = fp8_mfma16(fw, fa);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(y[r], s * ws, acc[r]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  fp8_rows_sum(p, sm, acc, n0);
}

template <int TM, int TN, int WM, int WN, int NB>
hipError_t launch_tile(const Fp8GemmParams& p, hipStream_t st) {
  using T = Fp8Tile<TM, TN, WM, WN, NB>;
  const long nbm = (p.M + T::BM - 1) / T::BM, nbn = (p.N + T::BN - 1) / T::BN;
  fp8_gemm_tile_kernel<TM, TN, WM, WN, NB><<<(unsigned)(nbm * nbn), 64 * WM * WN, 0, st>>>(p, (int)nbm, (int)nbn, 4);
  return hipGetLastError();
}

template <int TM, int TN, int NW>
hipError_t launch_strip(const Fp8GemmParams& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.N + 16 * TN - 1) / (16 * TN)), (unsigned)((p.M + 16 * TM - 1) / (16 * TM)));
  fp8_gemm_strip_kernel<TM, TN, NW><<<grid, 64 * NW, 0, st>>>(p);
  return hipGetLastError();
}

// What a kernel's workgroups take: rows of a, of w, their threads, how many share a CU, and microseconds for a block of K with
// n of them on a CU (us[n - 1]); a launch takes 3.5 us besides, a further round 1, and w is read from memory at 5.2 TB/s at most.
// Measured (us, K = 6144; strips of 32 x 16, 32 x 32, 64 x 32, 48 x 64 and 64 x 64, then the tiles):
//     32 x  1536     6.2   7.5   8.6  10.4  12.4 |  16.0  21.2  40.0  38.2  59.6
//     77 x  1536     9.4   7.5   9.2  11.0  13.2 |  16.1  21.3  40.3  38.5  60.0
//     32 x  6144    12.1   9.3   9.3  11.0  13.1 |  16.5  21.4  40.6  38.6  59.9
//     64 x  6144    17.3  15.9  10.6  11.4  13.9 |  16.7  21.4  40.8  38.8  60.3
//     77 x  6144    25.4  21.3  17.0  11.6  13.6 |  16.5  21.5  40.9  38.8  60.3
//    128 x  6144    32.2  23.8  19.3  20.7  14.1 |  16.7  21.6  41.0  38.8  60.5
//    320 x  6144    76.6  59.1  37.6  32.7  26.6 |  23.4  22.4  40.3  39.2  61.5
//   1024 x  6144   240   167   107    94.2  76.8 |  62.4  52.9  47.9  42.2  61.7
//   2381 x  6144   567   388   253   200   188   | 149   125   103    95.9  80.6
struct Fp8Cost {
  int rows, cols, threads, slots;
  float us[3];
};
constexpr int FP8_STRIPS = 5, FP8_KERNELS = FP8_STRIPS + 5;
const Fp8Cost kCosts[FP8_KERNELS] = {
    {32, 16, 512, 1, {0.075f}}, {32, 32, 512, 1, {0.105f}}, {64, 32, 256, 1, {0.15f}}, {48, 64, 256, 1, {0.185f}},
    {64, 64, 256, 1, {0.235f}}, {64, 64, 256, 3, {0.27f, 0.42f, 0.64f}}, {64, 128, 256, 2, {0.38f, 0.62f}},
    {128, 128, 256, 2, {0.78f, 1.10f}}, {256, 128, 512, 1, {1.00f}}, {256, 256, 512, 1, {1.75f}}};
constexpr long FP8_THREADS = 1L << 32;   // a launch holds fewer

struct Fp8Choice {
  int kernel;
  float us;
};
Fp8Choice choose(long M, long N, int K) {
  const long blocks = fp8_kp(K) / 128;
  const float read = 3.5f + N * blocks * 128 / 5.2e6f;   // of w, from memory
  Fp8Choice best{0, INFINITY};
  for (int i = 0; i < FP8_KERNELS; ++i) {
    const Fp8Cost& t = kCosts[i];
    const long nbm = (M + t.rows - 1) / t.rows, nbn = (N + t.cols - 1) / t.cols, all = nbm * nbn;
    if ((i < FP8_STRIPS && nbm > 65535) || all * t.threads >= FP8_THREADS) continue;   // tiles of 64 x 64 always fit
    const long whole = all / (256 * t.slots), rest = (all % (256 * t.slots) + 255) / 256;
    float us = 2.5f + whole * (1.0f + blocks * t.us[t.slots - 1]) + (rest ? 1.0f + blocks * t.us[rest - 1] : 0.0f);
    if (us < read) us = 0.9f * read + 0.1f * us;   // where reading w takes longest, what takes least besides
    if (us < best.us) best = {i, us};
  }
  return best;
}

// Rows ahead of the last round of the largest tiles, where the others take less in a launch of their own than in a round that is
// nearly empty, else 0.  4352 x 16384, K = 6144: 382 us, in one launch 396 (4096 rows alone 342 to 347).
long head_rows(long M, long N, int K) {
  const Fp8Cost& t = kCosts[FP8_KERNELS - 1];
  const Fp8Choice all = choose(M, N, K);
  const long nbm = (M + t.rows - 1) / t.rows, nbn = (N + t.cols - 1) / t.cols;
  const long rows = nbm * nbn / 256 * 256 / nbn * t.rows;
  if (all.kernel != FP8_KERNELS - 1 || rows <= 0 || rows >= M) return 0;
  return choose(rows, N, K).us + choose(M - rows, N, K).us < all.us ? rows : 0;
}

hipError_t launch_kernel(int kernel, const Fp8GemmParams& p, hipStream_t st) {
  switch (kernel) {
    case 0: return launch_strip<2, 1, 8>(p, st);
    case 1: return launch_strip<2, 2, 8>(p, st);
    case 2: return launch_strip<4, 2, 4>(p, st);
    case 3: return launch_strip<3, 4, 4>(p, st);
    case 4: return launch_strip<4, 4, 4>(p, st);
    case 5: return launch_tile<1, 4, 4, 1, 3>(p, st);
    case 6: return launch_tile<2, 4, 2, 2, 3>(p, st);
    case 7: return launch_tile<4, 4, 2, 2, 2>(p, st);
    case 8: return launch_tile<4, 4, 4, 2, 3>(p, st);
    default: return launch_tile<4, 8, 4, 2, 2>(p, st);
  }
}

}  // namespace

// 16 columns a workgroup of 512 threads: wider outputs than a launch holds go to the other kernels
static bool few_rows(int M, int N) { return M <= 16 && (N + 15L) / 16 * 512 < FP8_THREADS; }

int fp8_gemm_kernel(int M, int N, int K, int& rows, int& cols, int& head) {
  head = 0;
  if (few_rows(M, N)) {
    rows = 16;
    cols = 16;
    return FP8_ROWS_KERNEL;
  }
  head = (int)head_rows(M, N, K);
  const int kernel = choose(M - head, N, K).kernel;
  rows = kCosts[kernel].rows;
  cols = kCosts[kernel].cols;
  return kernel < FP8_STRIPS ? FP8_STRIP_KERNEL : FP8_TILE_KERNEL;
}

hipError_t launch_fp8_gemm(const Fp8GemmParams& p, hipStream_t st) {
  if (few_rows(p.M, p.N)) {
    if (p.M > 8) fp8_gemm_rows_kernel<16, 2><<<(unsigned)((p.N + 15) / 16), 512, 0, st>>>(p);
    else fp8_gemm_rows_kernel<8, 3><<<(unsigned)((p.N + 15) / 16), 512, 0, st>>>(p);
    return hipGetLastError();
  }
  const long rows = head_rows(p.M, p.N, p.K);
  if (!rows) return launch_kernel(choose(p.M, p.N, p.K).kernel, p, st);
  Fp8GemmParams head = p, rest = p;
  head.M = (int)rows;
  rest.M -= head.M;
  rest.a += rows * fp8_kp(p.K);
  rest.as += rows;
  rest.y += rows * p.ldy;
  if (hipError_t e = launch_kernel(FP8_KERNELS - 1, head, st); e != hipSuccess) return e;
  return launch_kernel(choose(rest.M, p.N, p.K).kernel, rest, st);
}

long fp8_linear_workspace_bytes(int M, int K) {
  const long kp = fp8_kp(K);
  return M * kp + M * (kp / 32);   // codes, scales
}

hipError_t launch_fp8_linear(Fp8GemmParams p, const uint16_t* x, long ldx, void* workspace, hipStream_t st) {
  if (p.M <= Fp8RowsOf::MR && few_rows(p.M, p.N) && p.K % 128 == 0 && ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0) {
    fp8_linear_rows_kernel<<<(unsigned)((p.N + 15) / 16), 512, 0, st>>>(p, x, ldx);
    return hipGetLastError();
  }
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + p.M * fp8_kp(p.K));
  p.a = codes;
  p.as = scales;
  if (hipError_t e = launch_fp8_quantize(x, ldx, p.M, p.K, codes, scales, st); e != hipSuccess) return e;
  return launch_fp8_gemm(p, st);
}

}  // namespace svdq
