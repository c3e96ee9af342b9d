// The 8-bit cache of keys and values, and attention over it.
//
// Pages hold 64 tokens of every key / value head: keys as [64, D], values transposed as [D, 64], so that both enter the
// matrix instructions as they lie, and a float32 scale each for a page and head.  A sequence is a row of the page table and
// its length; the new tokens of all sequences lie behind one another in the rows of k, v and q, sequence b's from
// offsets[b].
//
// Everything that comes from device memory is held to its range before it is used as an index: offsets to the rows there
// are, lengths to the table's width, pages to the cache (others hold nothing, and nothing is written to them).
//
// append:  a page's scale is that of its new tokens (svdq_fp8.h), or the larger (in magnitude) of that and the one it has where
//          it holds tokens already; those are then rounded again under the new scale.
// attend:  o = sum over visible j of softmax_j(scale q . k_j) v_j,  j < length, and with a causal mask, for the i-th of n new
//          tokens, j <= length - n + i; 0 where nothing is visible.
#include <type_traits>

#include "svdq_fp8.h"
#include "svdq_kernels.h"

namespace svdq {
namespace {

constexpr int PAGE = 64;

__device__ __forceinline__ u32x4 ld16(const void* p) { return *reinterpret_cast<const u32x4*>(p); }

// The first row of sequence b; sequence B stands for the rows behind the last one.
__device__ __forceinline__ int first_row(const Kv8Cache& c, int b) {
  return b <= 0 ? 0 : b > c.B ? c.N : min(max(c.offsets[b], 0), c.N);
}

// Work is dealt out in units of `unit` rows, numbered so that sequence b's begin at rows_before / unit + extra b: a number
// that needs no sum over the sequences before, at least the ceiling of its rows over the unit further on (plus extra - 1).
// Finds the sequence of a number; lanes look at 64 sequences at a time.
__device__ __forceinline__ long first_unit(const Kv8Cache& c, int b, int mult, int unit, int extra) {
  return (long)first_row(c, b) * mult / unit + (long)extra * b;
}
struct Kv8Sequence {
  int b, row0, n, len;   // sequence, its first row and new tokens, tokens held
  long unit0;            // its first unit
  int share;             // SHARE: a `run`-th of all units' pages, rounded up
};
template <bool SHARE = false>
__device__ __forceinline__ Kv8Sequence find_sequence(const Kv8Cache& c, long number, int mult, int unit, int extra, int run = 0) {
  const int lane = threadIdx.x & 63;
  Kv8Sequence s;
  s.share = 0;
  if (c.B < 63) {   // a lane each: one latency for all of it
    const int row = first_row(c, lane), len = c.lengths[min(lane, c.B - 1)];
    s.b = __popcll(__ballot(lane > 0 && lane <= c.B && (long)row * mult / unit + (long)extra * lane <= number));
    s.row0 = __builtin_amdgcn_readlane(row, s.b);
    s.n = __builtin_amdgcn_readlane(row, s.b + 1) - s.row0;
    s.len = __builtin_amdgcn_readlane(len, s.b);
    if (SHARE) {
      const int n = __shfl_down(row, 1, 64) - row, pages = (min(max(len, 0), c.W * PAGE) + PAGE - 1) / PAGE;
      float work = lane < c.B && n > 0 ? (float)pages * (float)(((long)n * mult + unit - 1) / unit) : 0.0f;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) work += __shfl_xor(work, o, 64);
      s.share = (int)fminf(ceilf(work / (float)run), 1e6f);
    }
  } else {
    int before = 0;
    for (int b0 = 1; b0 <= c.B; b0 += 64)
      before += __popcll(__ballot(b0 + lane <= c.B && first_unit(c, b0 + lane, mult, unit, extra) <= number));
    s.b = __builtin_amdgcn_readfirstlane(before);
    s.row0 = first_row(c, s.b);
    s.n = first_row(c, s.b + 1) - s.row0;
    s.len = c.lengths[min(s.b, c.B - 1)];
  }
  s.n = max(s.n, 0);
  s.len = s.b == c.B ? 0 : min(max(s.len, 0), c.W * PAGE);
  s.unit0 = (long)s.row0 * mult / unit + (long)extra * s.b;
  return s;
}

// ---- append -------------------------------------------------------------------------------------

// q = x rounded to float32 and the sign of x - q: a float32 that rounds to fewer bits as x does (the last bit tells that
// something was cut off).
__device__ __forceinline__ float sticky(float q, float rest) {
  if (rest == 0.0f || q == 0.0f) return q;
  const uint32_t b = __float_as_uint(q);
  return __uint_as_float(((rest < 0.0f) != (q < 0.0f) ? b - 1 : b) | 1u);
}

// One workgroup for a page and head that new tokens go to.  Keys and values of its tokens are held in registers (16 bytes
// of a token a thread and round) while their largest magnitudes are found.  A chain of reads (offsets and lengths, table and
// tokens) bounds it: a token of each of 32 sequences 5.3 us, three prompts of up to 1101 tokens 10.8 (21 MB).
template <int D>
__global__ void __launch_bounds__(256) kv8_append_kernel(Kv8Cache c, const uint16_t* __restrict__ k, long ldk,
                                                         const uint16_t* __restrict__ v, long ldv) {
  constexpr int CH = D / 8, ROUNDS = PAGE * CH / 256;   // chunks of 8 channels of a token
  __shared__ uint32_t tops[2][4];
  constexpr int PITCH = PAGE + 4;   // bytes of a channel: one word over, which spreads the lanes over the banks
  __shared__ __attribute__((aligned(16))) uint8_t turn[D * PITCH];
  const int tid = threadIdx.x, head = blockIdx.x % c.Hkv;
  const long number = blockIdx.x / c.Hkv;
  const Kv8Sequence q = find_sequence(c, number, 1, PAGE, 2);
  if (q.b >= c.B || q.n == 0 || number < q.unit0) return;   // before its first: offsets that do not ascend
  const int b = q.b, row0 = q.row0, n = q.n;
  const long start = q.len, page = start / PAGE + (number - q.unit0);
  if (page >= c.W || page * PAGE >= start + n) return;
  const int id = c.table[(long)b * c.W + page];
  const int lo = (int)max(start - page * PAGE, 0L), hi = (int)min(start + n - page * PAGE, (long)PAGE);
  const long base = row0 + page * PAGE - start;   // row of the page's slot 0

  u32x4 x[2][ROUNDS];   // on their way while the page is looked up
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int slot = ROUNDS * (tid / CH) + i, ch = tid % CH;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      x[w][i] = u32x4{};
      if (slot >= lo && slot < hi) x[w][i] = ld16((w ? v + (base + slot) * ldv : k + (base + slot) * ldk) + head * D + 8 * ch);
    }
  }
  if (id < 0 || id >= c.P) return;
  const long at = (long)id * c.Hkv + head;
  uint8_t *kc = c.kc + at * PAGE * D, *vc = c.vc + at * PAGE * D;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i)
#pragma unroll
      for (int d = 0; d < 4; ++d)
        top[w] = max(top[w], max(fp8_magnitude(bf16lo(x[w][i][d])), fp8_magnitude(bf16hi(x[w][i][d]))));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top[w] = max(top[w], (uint32_t)__shfl_xor((int)top[w], o, 64));
    if ((tid & 63) == 0) tops[w][tid >> 6] = top[w];
  }
  const float had[2] = {c.scales[2 * at], c.scales[2 * at + 1]};
  __syncthreads();
  float s[2], again[2];   // the page's scales, and what its older codes are multiplied by
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    s[w] = fp8_scale(max(max(tops[w][0], tops[w][1]), max(tops[w][2], tops[w][3])));
    again[w] = 1.0f;
    if (lo > 0) {
      if (fabsf(had[w]) >= s[w]) s[w] = had[w];
      else again[w] = had[w] / s[w];
    }
  }
  if (tid < 2) c.scales[2 * at + tid] = tid ? s[1] : s[0];
  auto encode = [](u32x4 r, float s) {
    if (s < 0.0f || __float_as_uint(s) & 0x7FFFFFu) {   // a scale of the caller's, no power of two: the conversion takes only those
      auto over = [&](float v) {
        const float q = v / s;
        const float rest = __builtin_fmaf(-q, s, v);   // |s| is at least what the new tokens need
        return sticky(q, s < 0.0f ? -rest : rest);
      };
      return u32x2{fp8_encode4(over(bf16lo(r[0])), over(bf16hi(r[0])), over(bf16lo(r[1])), over(bf16hi(r[1])), 1.0f),
                   fp8_encode4(over(bf16lo(r[2])), over(bf16hi(r[2])), over(bf16lo(r[3])), over(bf16hi(r[3])), 1.0f)};
    }
    return u32x2{fp8_encode4(bf16lo(r[0]), bf16hi(r[0]), bf16lo(r[1]), bf16hi(r[1]), s),
                 fp8_encode4(bf16lo(r[2]), bf16hi(r[2]), bf16lo(r[3]), bf16hi(r[3]), s)};
  };
  auto scaled = [](uint32_t x, float f) {   // four older codes
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
    auto times = [&](float v) { return sticky(v * f, __builtin_fmaf(v, f, -(v * f))); };
    return fp8_encode4(times(a[0]), times(a[1]), times(b[0]), times(b[1]), 1.0f);
  };
  const bool whole = lo == 0 && hi == PAGE;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int slot = ROUNDS * (tid / CH) + i, ch = tid % CH;
    u32x2* kd = reinterpret_cast<u32x2*>(kc + slot * D + 8 * ch);
    if (slot >= lo && slot < hi) {
      *kd = encode(x[0][i], s[0]);
      if (!whole) {
        const u32x2 o = encode(x[1][i], s[1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) vc[(8 * ch + e) * PAGE + slot] = (uint8_t)(o[e / 4] >> (8 * (e % 4)));
      }
    } else if (slot < lo && again[0] != 1.0f) {
      const u32x2 old = *kd;
      *kd = u32x2{scaled(old[0], again[0]), scaled(old[1], again[0])};
    }
  }
  if (whole) {   // values through LDS: a thread holds ROUNDS tokens of 8 channels, a line of the page is 64 of one
    const int ch = tid % CH;
    u32x2 o[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) o[i] = encode(x[1][i], s[1]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) w |= (o[i][e / 4] >> 8 * (e % 4) & 0xFFu) << 8 * i;
      uint8_t* to = turn + (8 * ch + e) * PITCH + ROUNDS * (tid / CH);
      if (ROUNDS == 4) *reinterpret_cast<uint32_t*>(to) = w;
      else *reinterpret_cast<uint16_t*>(to) = (uint16_t)w;
    }
    __syncthreads();
    for (int i = tid; i < D * PAGE / 16; i += 256) {
      const uint32_t* from = reinterpret_cast<const uint32_t*>(turn + i / 4 * PITCH + 16 * (i % 4));
      *reinterpret_cast<u32x4*>(vc + 16 * i) = u32x4{from[0], from[1], from[2], from[3]};
    }
  } else if (lo > 0 && again[1] != 1.0f) {
    // whole words of older values; in the last one the new tokens' bytes, which other threads write, are not touched
    for (int i = tid; i < D * (lo / 4); i += 256) {
      uint32_t* w = reinterpret_cast<uint32_t*>(vc + i / (lo / 4) * PAGE) + i % (lo / 4);
      *w = scaled(*w, again[1]);
    }
    for (int i = tid; i < D * (lo % 4); i += 256) {
      uint8_t* q = vc + i / (lo % 4) * PAGE + lo / 4 * 4 + i % (lo % 4);
      *q = (uint8_t)scaled(*q, again[1]);
    }
  }
}

// ---- attention -----------------------------------------------------------------------------------
// The query heads of a key / value head lie beside the tokens as rows of one matrix: row r of a sequence is token r / G, head
// G hk + r % G.  A tile of rows reads each page once.

struct Kv8Args {
  Kv8Cache c;
  const uint16_t* q;
  long ldq;
  uint16_t* o;
  int H, G, causal;
  int splits;       // of a tile along the keys
  int run;          // many rows: pieces of a head's tiles that are to be about as long; 0: every tile has `splits`
  int numbers;      // of tiles, those of no tile among them
  int whole;        // many rows: an XCD's tiles that are not split
  float scale_log2;
  float* part_o;    // [tile, split, rows, D]
  float* part_ml;   // [tile, split, rows, 2]: maximum (log2 units), sum
};

struct Kv8Tile {
  int b, row0, n, rows, r0, len;   // sequence, its first row of q and tokens, its rows of heads, the tile's first, tokens held
  int share;
};
template <int R>
__device__ __forceinline__ bool kv8_tile(const Kv8Args& p, long number, Kv8Tile& t) {
  const Kv8Sequence q = R > 16 && p.run ? find_sequence<(R > 16)>(p.c, number, p.G, R, 1, p.run) : find_sequence(p.c, number, p.G, R, 1);
  t.b = q.b;
  t.row0 = q.row0;
  t.n = q.n;
  t.len = q.len;
  t.rows = q.n * p.G;
  t.share = q.share;
  const long r0 = (number - q.unit0) * R;
  t.r0 = (int)r0;
  return r0 >= 0 && r0 < t.rows;   // below 0: offsets that do not ascend
}
// keys that the row's token sees
__device__ __forceinline__ int kv8_visible(const Kv8Args& p, const Kv8Tile& t, int row) {
  return p.causal ? max(t.len - t.n + row / p.G + 1, 0) : t.len;
}

// Many rows: workgroups go round the 8 XCDs, each with an L2 of its own.  With g the largest power of two, 8 at most, that
// divides the key / value heads, XCD x takes heads x mod g, x mod g + g, ... one after another, and every (8 / g)-th of their
// tiles: an L2 holds the pages of a head or two at a time.  The last tiles, which see most under a causal mask, go first.
// An XCD's first `whole` tiles run in one piece, the others in `splits` along the keys.
__host__ __device__ inline int kv8_shared(int Hkv) { return Hkv % 8 == 0 ? 8 : Hkv % 4 == 0 ? 4 : Hkv % 2 == 0 ? 2 : 1; }
__host__ __device__ inline long kv8_each(long numbers, int Hkv) {   // an XCD's tiles of a head
  const int per = 8 / kv8_shared(Hkv);
  return (numbers + per - 1) / per;
}
__device__ __forceinline__ bool kv8_tile_of(const Kv8Args& p, uint32_t x, uint32_t j, int& number, int& hk) {
  const uint32_t g = kv8_shared(p.c.Hkv), per = 8 / g, each = (uint32_t)kv8_each(p.numbers, p.c.Hkv), head = j / each;
  const uint32_t s = (j - head * each) * per + x / g;
  hk = x % g + g * head;
  number = p.numbers - 1 - s;
  return s < (uint32_t)p.numbers && head < p.c.Hkv / g;
}
// the tile of a workgroup, its piece and where that goes (-1: a whole tile)
__device__ __forceinline__ bool kv8_piece(const Kv8Args& p, int& number, int& hk, int& split, int& piece) {
  const uint32_t x = blockIdx.x % 8, j = blockIdx.x / 8;
  if (j < (uint32_t)p.whole) {
    split = 0;
    piece = -1;
    return kv8_tile_of(p, x, j, number, hk);
  }
  uint32_t k;
  if (p.run) {
    // every tile's first piece, then their second, ...: those that a tile does not have come last.  Between others the dispatcher
    // deals these out to few of the CUs (6 sequences of 900 to 9000 keys 192 us, so 168).
    const uint32_t tail = kv8_each(p.numbers, p.c.Hkv) * (p.c.Hkv / kv8_shared(p.c.Hkv)) - p.whole;
    split = (j - p.whole) / tail;
    k = (j - p.whole) - split * tail;
  } else {
    k = (j - p.whole) / p.splits;
    split = (j - p.whole) - k * p.splits;
  }
  piece = (k * 8 + x) * p.splits + split;
  return kv8_tile_of(p, x, p.whole + k, number, hk);
}

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Masked keys have probability 0, but 0 times a code that is not a number is not.  In pages of which rows see different parts
// such codes are taken out of the values, and the rows that do see them get them from a product of their own: of ones where
// the codes are and ones where the row sees the key.
__device__ __forceinline__ uint32_t fp8x4_nan(uint32_t x) {   // 0x80 in the bytes that are not a number
  return ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t bytes_of(uint32_t high) {   // 0xFF where a byte's top bit is set, other bits being clear
  return (high << 1) - (high >> 7);
}
// ones (bf16) for the low four, then the high four of eight bits
__device__ __forceinline__ u32x4 ones_of(uint32_t bits) {
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (bits >> 2 * e & 1 ? 0x3F80u : 0u) | (bits >> 2 * e & 2 ? 0x3F800000u : 0u);
  return o;
}
// the bits of eight keys from key `from` that lie below `end`
__device__ __forceinline__ uint32_t bits_below(int from, int end) {
  const int n = end - from;
  return n >= 8 ? 0xFFu : n <= 0 ? 0u : (1u << n) - 1u;
}
// four bits of bytes that hold 0x80 or 0
__device__ __forceinline__ uint32_t bits_of(uint32_t high) { return high * 0x00204081u >> 28; }

// bytes of 16 keys from key `from` that lie below `end`
__device__ __forceinline__ u32x4 keys_below(u32x4 x, int from, int end) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int n = end - from - 4 * d;
    x[d] = n >= 4 ? x[d] : n <= 0 ? 0u : x[d] & ((1u << (8 * n)) - 1u);
  }
  return x;
}
// Pages of a piece of a tile that is split: an even part, or, for pieces of a batch that are about as long, no less than t.share.
__device__ __forceinline__ int kv8_per(const Kv8Args& p, const Kv8Tile& t, int pages) {
  return max(max((pages + p.splits - 1) / p.splits, t.share), 1);   // of none: one that is empty
}

// The offset of a softmax's exponent follows the maximum only where that is more than 2^KV8_LAZY above it, so the output is
// hardly ever rescaled; probabilities up to 2^KV8_LAZY are as exact as those below 1.
constexpr float KV8_LAZY = 8.0f;
// score x factor - offset in one FMA is exact, the offset (a rounded product) is not: scores (log2 units) of 2^20 and more are
// multiplied and rounded by themselves, so that the largest is at its offset however large they are.
constexpr float KV8_LARGE = 0x1p20f;
constexpr int KV8_SPLITS = 128;   // at most

__device__ __forceinline__ float other_half_max(float v) {   // over lanes l and l ^ 32
  uint32_t a = __float_as_uint(v), b = a;
  permlane32_swap(a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}

// Few rows: 16 of them a workgroup, whose four waves take the split's pages in turn, each with a softmax of its own; they are
// joined in LDS at the end.  HBM-bound: 131072 tokens of 12 heads of 128 in 64 us, 6.3 TB/s, and 4.6 for the join.  Each wave has a page in LDS to itself, filled by DMA while it computes on the one before, which is
// in registers by then; the waves need no barrier before the end.
// A lane reads 16 channels of the key in its row of K, and 16 keys of one channel of V:
//   S^T = K Q^T: row 4 g + i of tile t stands for key 16 g + 4 t + i, so lane group g gets the probabilities of the 16 keys that
//   it reads values of; O^T += V^T P^T takes them as they are, tiles 2 u and 2 u + 1 in step u.
// Chunks of 16 bytes lie at slots that spread sixteen lanes' reads over the 64 banks: chunk c of key row r at
// c ^ (2 (r / 16) + r / 2 mod 2) (rows of 128 bytes; of 64: c ^ (r / 16)), of channel row r of V at c ^ (r / 4 mod 4).
template <bool NT>
__device__ __forceinline__ void dma16_page(const void* base, uint32_t off, uint32_t lds) {
  if (NT) asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
  else dma16(base, off, lds);
}

// A page's scale that is not finite makes all of its keys (values) NaN.
constexpr uint32_t FP8_NAN4 = 0x7F7F7F7Fu;
__device__ __forceinline__ float finite_or_nan(float f) { return fabsf(f) < INFINITY ? f : __builtin_nanf(""); }

template <int D>
struct Kv8Few {
  static constexpr int R = 16, PITCH = D + 4, HALF = PAGE * D, RING = 2 * HALF, DMA = 2 * HALF / 1024;
  static_assert(8 * RING <= 160 * 1024 && 4 * R * PITCH * 4 + 4 * R * 8 <= 4 * RING, "LDS");
  __device__ static int key_turn(int row) { return D == 128 ? row >> 4 << 1 | (row >> 1 & 1) : row >> 4; }
  // an instruction moves 1024 bytes of a page as they lie, chunks exchanged within their rows
  template <bool NT>
  __device__ static void fetch(const uint8_t* kc, const uint8_t* vc, uint32_t koff, uint32_t voff, uint32_t lds) {
#pragma unroll
    for (int d = 0; d < DMA / 2; ++d)   // its first key row is d * 1024 / D: what that adds to the turn
      dma16_page<NT>(kc + 1024 * d, koff ^ 16 * key_turn(d * (1024 / D)), lds + 1024 * d);
#pragma unroll
    for (int d = 0; d < DMA / 2; ++d) dma16_page<NT>(vc + 1024 * d, voff, lds + HALF + 1024 * d);
  }
};

template <int D>
__global__ void __launch_bounds__(256, 2) kv8_rows_kernel(Kv8Args p) {
  using T = Kv8Few<D>;
  constexpr int R = T::R, SP = D / 64, DT = D / 16, KC = D / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t sm[4 * T::RING];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // heads one after another: a page's heads lie side by side, and the card reads them together from all of its memory (a
  // head to an XCD reads parts of it: 131072 tokens 94 us, so 69)
  const uint32_t hk = blockIdx.x % p.c.Hkv, rest = blockIdx.x / p.c.Hkv, split = rest % p.splits, number = rest / p.splits;
  Kv8Tile t;
  if (!kv8_tile<R>(p, number, t)) return;
  const int row = min(t.r0 + lr, t.rows - 1);
  const int vis = kv8_visible(p, t, row);
  const int vmin = kv8_visible(p, t, t.r0), vmax = kv8_visible(p, t, min(t.r0 + R, t.rows) - 1);
  const int pages = (vmax + PAGE - 1) / PAGE, per = (pages + p.splits - 1) / p.splits;
  const int p0 = (int)split * per, p1 = min(p0 + per, pages);

  u32x4 qf[2 * SP];
  const uint16_t* qr = p.q + (long)(t.row0 + row / p.G) * p.ldq + (hk * p.G + row % p.G) * D + 16 * g;
#pragma unroll
  for (int s = 0; s < 2 * SP; ++s) qf[s] = ld16(qr + 64 * (s / 2) + 8 * (s % 2));

  f32x4 O[DT] = {};
  float m = -INFINITY, l = 0.0f;
  const int count = p0 + wave < p1 ? (p1 - p0 - wave + 3) / 4 : 0;   // this wave's pages: p0 + wave + 4 i
  if (count) {
    const uint32_t lds0 = lds_offset(sm) + wave * T::RING;
    const uint32_t koff = (lane / KC) * D + 16 * (lane % KC ^ (D == 128 ? lane / KC >> 1 & 1 : 0));
    const uint32_t voff = (lane / 4) * PAGE + 16 * (lane % 4 ^ (lane / 16 & 3));
    const int* table = p.c.table + (long)t.b * p.c.W;
    int id = 0;
    float ks = 0.0f, vs = 0.0f;
    auto look_up = [&](int i0) {   // lane i: page i0 + i of this wave; a page that is not there holds nothing
      const int i = i0 + lane;
      id = i < count ? table[p0 + wave + 4 * i] : -1;
      if (id < 0 || id >= p.c.P) id = -1;
      asm volatile("" : "+v"(id)::"memory");   // ahead of the DMA, which the compiler does not count
    };
    auto look_scales_up = [&] {
      const long at = (long)max(id, 0) * p.c.Hkv + hk;
      ks = finite_or_nan(p.c.scales[2 * at] * p.scale_log2);
      vs = p.c.scales[2 * at + 1];
      asm volatile("s_waitcnt vmcnt(0)" : "+v"(ks), "+v"(vs)::"memory");
    };
    look_up(0);
    int first = 0;   // the page that lane 0 holds
    // past the caches where no other tile reads the page (131072 tokens 77 us, so 69)
    const bool once = t.rows <= R;
    auto fetch = [&](int i) {   // page i of this wave, past the last one that again
      const int pid = max(__builtin_amdgcn_readlane(id, max(min(i, count - 1) - first, 0)), 0);
      const long at = (long)pid * p.c.Hkv + hk;
      const uint8_t *kc = p.c.kc + at * T::HALF, *vc = p.c.vc + at * T::HALF;
      if (once) T::template fetch<true>(kc, vc, koff, voff, lds0);
      else T::template fetch<false>(kc, vc, koff, voff, lds0);
    };
    fetch(0);
    look_scales_up();
    auto rescale = [&](float top) {
      const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) O[d] *= alpha;
    };
    auto rows_max = [](float v) {   // over the four lanes of a row
      v = fmaxf(v, __shfl_xor(v, 16, 64));
      return other_half_max(v);
    };
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      const int pg = p0 + wave + 4 * i;
      const bool have = __builtin_amdgcn_readlane(id, i - first) >= 0;
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), i - first));
      float pv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), i - first));
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      const uint8_t *sk = sm + wave * T::RING, *sv = sk + T::HALF;
      u32x4 kq[4][SP], vq[DT];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 16 * (lr >> 2) + 4 * k + (lr & 3);
#pragma unroll
        for (int s = 0; s < SP; ++s) kq[k][s] = ld16(sk + r * D + 16 * ((4 * s + g) ^ T::key_turn(r)));
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) vq[d] = ld16(sv + (16 * d + lr) * PAGE + 16 * (g ^ (lr >> 2)));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // all of the page is in registers
      __builtin_amdgcn_sched_barrier(0);
      if (i + 1 - first >= 64) {   // its next page is not among those looked up
        first = i + 1;
        look_up(first);
        look_scales_up();
      }
      fetch(i + 1);
      if (!have) continue;
      f32x4 S[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        S[k] = f32x4{};
#pragma unroll
        for (int s = 0; s < SP; ++s) {
          S[k] = mfma_bf16_16x16x32(fp8_to_bf16x8(kq[k][s][0], kq[k][s][1]), qf[2 * s], S[k]);
          S[k] = mfma_bf16_16x16x32(fp8_to_bf16x8(kq[k][s][2], kq[k][s][3]), qf[2 * s + 1], S[k]);
        }
      }
      u32x4 pf[2];
      if (pg * PAGE + PAGE <= vmin && f >= 0.0f && pv > 0x1p-60f && pv < 0x1p60f) {
        const float lv = __builtin_amdgcn_logf(pv);   // log2
        float hi = S[0][0];
#pragma unroll
        for (int k = 0; k < 16; ++k) hi = fmaxf(hi, S[k / 4][k % 4]);
        const float top = rows_max(hi * f);
        if (__any(top > m + KV8_LAZY)) rescale(top);
        const float base = m == -INFINITY ? 0.0f : m, off = base - lv;
        if (__any(!(fabsf(top) < KV8_LARGE))) {
#pragma clang fp contract(off)
#pragma unroll
          for (int k = 0; k < 16; ++k) S[k / 4][k % 4] = S[k / 4][k % 4] * f - base + lv;
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) S[k / 4][k % 4] = __builtin_fmaf(S[k / 4][k % 4], f, -off);
        }
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          const float a = __builtin_amdgcn_exp2f(S[k / 4][k % 4]), b = __builtin_amdgcn_exp2f(S[k / 4][k % 4 + 1]);
          const uint32_t w = pack_bf16x2(a, b);
          pf[k / 8][k % 8 / 2] = w;
          sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3F803F80u), sum, false);
        }
        l = __builtin_fmaf(sum, 1.0f / pv, l);
      } else {   // masks, values that are not numbers behind them, any scales
        const int key0 = pg * PAGE + 16 * g;
        float hi = -INFINITY;
        if (!(fabsf(pv) < INFINITY)) {   // values that are not numbers, which the masks below take out
          pv = 1.0f;
#pragma unroll
          for (int d = 0; d < DT; ++d) vq[d] = u32x4{} | FP8_NAN4;
        }
        {
#pragma clang fp contract(off)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            S[k / 4][k % 4] = key0 + k >= vis ? -INFINITY : S[k / 4][k % 4] * f;
            hi = fmaxf(hi, S[k / 4][k % 4]);
          }
        }
        const float top = rows_max(hi);
        if (__any(top > m + KV8_LAZY)) rescale(top);
        const float off = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          const float a = __builtin_amdgcn_exp2f(S[k / 4][k % 4] - off), b = __builtin_amdgcn_exp2f(S[k / 4][k % 4 + 1] - off);
          l += a + b;
          pf[k / 8][k % 8 / 2] = pack_bf16x2(a * pv, b * pv);
        }
        uint32_t odd = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          vq[d] = keys_below(vq[d], key0, vmax);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= fp8x4_nan(vq[d][e]);
        }
        if (__any(odd != 0)) {
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            f32x4 hit = {};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t lo = fp8x4_nan(vq[d][2 * u]), hi4 = fp8x4_nan(vq[d][2 * u + 1]);
              hit = mfma_bf16_16x16x32(ones_of(bits_of(lo) | bits_of(hi4) << 4), ones_of(bits_below(key0 + 8 * u, vis)), hit);
              vq[d][2 * u] &= ~bytes_of(lo);
              vq[d][2 * u + 1] &= ~bytes_of(hi4);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) O[d][r] = hit[r] > 0.0f ? __builtin_nanf("") : O[d][r];
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);   // the values are not converted ahead of the softmax: there are no registers for them
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < 2; ++u) O[d] = mfma_bf16_16x16x32(fp8_to_bf16x8(vq[d][2 * u], vq[d][2 * u + 1]), pf[u], O[d]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();   // every ring is done with; their memory takes the waves' sums
  float* so = reinterpret_cast<float*>(sm);
  float* sml = so + 4 * R * T::PITCH;
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(so + (wave * R + lr) * T::PITCH + 16 * d + 4 * g) = O[d];
  if (g == 0) {
    sml[2 * (wave * R + lr)] = m;
    sml[2 * (wave * R + lr) + 1] = l;
  }
  __syncthreads();
  // 16 threads a row
  const int r = tid >> 4, c0 = (tid & 15) * (D / 16);
  float mm = -INFINITY, ll = 0.0f, o[D / 16] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[2 * (w * R + r)]);
  const float base = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(sml[2 * (w * R + r)] - base);
    ll += f * sml[2 * (w * R + r) + 1];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] += f * so[(w * R + r) * T::PITCH + c0 + i];
  }
  if (t.r0 + r >= t.rows) return;
  if (p.splits == 1) {
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    uint16_t* out = p.o + ((long)(t.row0 + (t.r0 + r) / p.G) * p.H + hk * p.G + (t.r0 + r) % p.G) * D + c0;
#pragma unroll
    for (int i = 0; i < D / 16; i += 2)
      *reinterpret_cast<uint32_t*>(out + i) = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
    return;
  }
  const long at = (((long)number * p.c.Hkv + hk) * p.splits + split) * R + r;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) p.part_o[at * D + c0 + i] = o[i];
  if ((tid & 15) == 0) {
    p.part_ml[2 * at] = mm;
    p.part_ml[2 * at + 1] = ll;
  }
}

// Joins the splits of the rows of a tile of R, 8 / GROUPS of them a workgroup: half a wave finds the weights of a row's splits;
// then 32 lanes take a row's columns, and GROUPS such groups every GROUPS-th split.
template <int D, int R, int GROUPS>
__global__ void __launch_bounds__(256) kv8_join_kernel(Kv8Args p) {
  constexpr int C = D / 32, ROWS = 8 / GROUPS;   // columns of a lane, rows of a workgroup
  __shared__ float weight[ROWS][KV8_SPLITS], total[ROWS];
  __shared__ __attribute__((aligned(16))) float part[GROUPS][ROWS][D];
  const int tid = threadIdx.x, hl = tid & 31, hw = tid >> 5;
  const uint32_t tile = blockIdx.x / (R / ROWS);
  const int r0 = ROWS * (blockIdx.x % (R / ROWS));
  int number = tile / p.c.Hkv, hk = tile % p.c.Hkv;
  if (R > 16 && !kv8_tile_of(p, tile % 8, p.whole + tile / 8, number, hk)) return;
  Kv8Tile t;
  if (!kv8_tile<R>(p, number, t)) return;
  if (t.r0 + r0 >= t.rows) return;
  const long first = (long)tile * p.splits * R + r0;
  int splits = p.splits;
  if (R > 16) {   // those that the tile has: the others have written nothing
    const int pages = (kv8_visible(p, t, min(t.r0 + R, t.rows) - 1) + PAGE - 1) / PAGE, per = kv8_per(p, t, pages);
    splits = max((pages + per - 1) / per, 1);
  }
  if (hw < ROWS) {
    float m[KV8_SPLITS / 32], l[KV8_SPLITS / 32], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < KV8_SPLITS / 32; ++i) {
      const int s = 32 * i + hl;
      const long at = first + hw + (long)min(s, splits - 1) * R;
      m[i] = s < splits ? p.part_ml[2 * at] : -INFINITY;
      l[i] = s < splits ? p.part_ml[2 * at + 1] : 0.0f;
      top = fmaxf(top, m[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < KV8_SPLITS / 32; ++i) {
      const float f = __builtin_amdgcn_exp2f(m[i] - base);
      weight[hw][32 * i + hl] = f;
      sum += f * l[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (hl == 0) total[hw] = sum;
  }
  __syncthreads();
  const int r = hw % ROWS, g = hw / ROWS;
  float o[C] = {};
#pragma unroll 4
  for (int s = g; s < splits; s += GROUPS) {
    const float f = weight[r][s];
    const float* from = p.part_o + (first + r + (long)s * R) * D + C * hl;
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] += f * from[i];
  }
  if (GROUPS > 1) {
#pragma unroll
    for (int i = 0; i < C; ++i) part[g][r][C * hl + i] = o[i];
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int k = 1; k < GROUPS; ++k)
#pragma unroll
      for (int i = 0; i < C; ++i) o[i] += part[k][r][C * hl + i];
  }
  const int row = t.r0 + r0 + r;
  if (row >= t.rows) return;
  const float inv = total[r] == 0.0f ? 0.0f : 1.0f / total[r];
  uint32_t* out = reinterpret_cast<uint32_t*>(p.o + ((long)(t.row0 + row / p.G) * p.H + hk * p.G + row % p.G) * D + C * hl);
#pragma unroll
  for (int i = 0; i < C / 2; ++i) out[i] = pack_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
}

// Many rows: 32 a wave, 128 a workgroup; pages go through LDS, as bf16, for its four waves.  Two workgroups share a CU, so that
// one's softmax runs under the other's products.  A lane holds one row's scores of half of the keys.  Row
// 16 s + 8 a + 4 h + i of K in LDS is key 16 s + 8 h + 4 a + i of the page (bits 2 and 3 exchanged), so that the probabilities
// leave the softmax in the values' order.
//
// The scale of the keys is part of the exponent's factor, that of the values (vs) of its offset:
// exp2(f s - (m - log2 vs)) = vs p, which is what the product needs; the row's sum takes the rounded values over vs, two in an
// instruction.  The offset is a row's maximum over the first page and stays, so the output is touched by the matrix unit
// alone; later probabilities may exceed 1, which float32 and bf16 hold as exactly.  Where a sum passes 2^64, anything is
// not finite, an offset is large, or a page of which rows see different parts holds values that are no numbers, the tile is done
// again with an offset that follows the maximum.
// Scales that are no ordinary positive numbers are dealt with as the pages come in: a factor below 0 turns the keys' signs, other
// scales of values are multiplied into them, those that are not finite make the codes NaN.  Pages that are not there count as -infinity.
//
// Bound by the softmax and the conversions beside the products: 4352 tokens of 48 heads of 128 over 4608, 483 us, 1020 TFLOP/s
// (causal, over themselves 268); heads of 64, 4 x 2048 causal 98 us (700 TFLOP/s), 8192 all visible 919 TFLOP/s.
//
// Rows in LDS are not padded: chunks of 16 bytes lie at slots exchanged by the row, c ^ (row mod 16) in rows of 256 bytes, c ^
// (row / 2 mod 8) in rows of 128, which spreads sixteen lanes' reads of a chunk, and sixteen lanes' writes of two chunks each, over the 64
// banks.
template <int D>
struct Kv8Many {
  static constexpr int R = 128, CH = PAGE * D / 16 / 256, DB = D / 32, KS = D / 16, KB = PAGE * D * 2;   // bytes of a buffer
  __device__ static int key_turn(int row) { return D == 128 ? row & 15 : row >> 1 & 7; }
  __device__ static int value_turn(int row) { return row >> 1 & 7; }
};

struct Kv8Scale {
  float f, lv, inv, at;   // the exponent's factor, log2 of the values' scale and its reciprocal, 0 or (no page) -infinity
};

template <int D>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) kv8_many_kernel(Kv8Args p) {   // of heads of 64 three share a CU
  using T = Kv8Many<D>;
  constexpr int DB = T::DB, KS = T::KS, KB = T::KB;
  __shared__ __attribute__((aligned(1024))) uint8_t sk[2 * KB], sv[2 * KB];
  __shared__ uint16_t odd_keys[D][4];   // bits of the codes that are not numbers, of a page that some row sees a part of
  __shared__ int odd_any[4];            // whether a wave found any
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int number, hk, split, piece;
  if (!kv8_piece(p, number, hk, split, piece)) return;
  Kv8Tile t;
  if (!kv8_tile<T::R>(p, number, t)) return;
  const int vmin = kv8_visible(p, t, t.r0), vmax = kv8_visible(p, t, min(t.r0 + T::R, t.rows) - 1);
  const int pages = (vmax + PAGE - 1) / PAGE, per = piece < 0 ? pages : kv8_per(p, t, pages);
  const int p0 = split * per, p1 = min(p0 + per, pages), pe = vmin / PAGE;   // pages from pe on: some row sees a part of them
  if (split && p0 >= pages) return;   // a piece that the tile does not have

  const int row = min(t.r0 + 32 * wave + lr, t.rows - 1), vis = kv8_visible(p, t, row);
  u32x4 qf[KS];
  const uint16_t* qr = p.q + (long)(t.row0 + row / p.G) * p.ldq + (hk * p.G + row % p.G) * D + 8 * h;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = ld16(qr + 16 * s);

  // Pages, their scales and what follows from those are looked up 64 at a time, one a lane.
  const int* table = p.c.table + (long)t.b * p.c.W;
  int ids = -1, first = p0;   // the page that lane 0 holds
  float kss = 0.0f, vss = 0.0f, lvs = 0.0f, invs = 1.0f;
  uint64_t odd_scales = 0;    // pages that are not there or whose scales are no ordinary numbers
  auto ordinary = [](float vs) { return vs > 0x1p-60f && vs < 0x1p60f; };
  auto look_up = [&](int from) __attribute__((always_inline)) {
    first = from;
    ids = from + lane < p1 ? table[from + lane] : -1;
    if (ids < 0 || ids >= p.c.P) ids = -1;
  };
  auto look_scales_up = [&]() __attribute__((always_inline)) {
    const long at = (long)max(ids, 0) * p.c.Hkv + hk;
    kss = p.c.scales[2 * at] * p.scale_log2;
    vss = p.c.scales[2 * at + 1];
    lvs = ordinary(vss) ? __builtin_amdgcn_logf(vss) : 0.0f;   // log2
    invs = ordinary(vss) ? 1.0f / vss : 1.0f;
    odd_scales = __ballot(ids < 0 || !ordinary(vss) || !(kss > 0.0f && kss < INFINITY));
  };
  auto lane_of = [](float v, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)); };
  u32x4 kr[T::CH], vr[T::CH];
  auto load = [&](int pg) __attribute__((always_inline)) {
    const int id = max(__builtin_amdgcn_readlane(ids, pg - first), 0);
    const long at = ((long)id * p.c.Hkv + hk) * PAGE * D;
    const __amdgpu_buffer_rsrc_t k = __builtin_amdgcn_make_buffer_rsrc(p.c.kc + at, (short)0, PAGE * D, 0x00020000);
    const __amdgpu_buffer_rsrc_t v = __builtin_amdgcn_make_buffer_rsrc(p.c.vc + at, (short)0, PAGE * D, 0x00020000);
#pragma unroll
    for (int i = 0; i < T::CH; ++i) {
      kr[i] = __builtin_amdgcn_raw_buffer_load_b128(k, 16 * tid + 4096 * i, 0, 0);
      vr[i] = __builtin_amdgcn_raw_buffer_load_b128(v, 16 * tid + 4096 * i, 0, 0);
    }
  };
  auto scale_in = [&](int pg) __attribute__((always_inline)) {
    const int i = pg - first;
    Kv8Scale s{lane_of(kss, i), lane_of(lvs, i), lane_of(invs, i), 0.0f};
    if (odd_scales >> i & 1) {
      // a factor of 0 is the smallest there is: times -infinity that is no NaN
      s.f = s.f == 0.0f ? 0x1p-126f : fabsf(s.f) < INFINITY ? fabsf(s.f) : 1.0f;
      if (__builtin_amdgcn_readlane(ids, i) < 0) s = {0x1p-126f, -INFINITY, 1.0f, -INFINITY};
    }
    return s;
  };
  // The tile is to be done again: offsets that are too low for a later score, nothing there of the first page, values that
  // are no numbers behind a mask.
  bool again = false;
  auto store = [&](int pg, int buf) __attribute__((always_inline)) {
    const int i0 = pg - first;
    const bool odd = odd_scales >> i0 & 1, here = __builtin_amdgcn_readlane(ids, i0) >= 0;
    float vs = odd && here ? lane_of(vss, i0) : 1.0f;
    if (odd) {
      const float ks = lane_of(kss, i0);
      const uint32_t turn = here && ks < 0.0f ? 0x80808080u : 0u, keep = here ? ~0u : 0u;
      const uint32_t kn = here && !(fabsf(ks) < INFINITY) ? FP8_NAN4 : 0u, vn = fabsf(vs) < INFINITY ? 0u : FP8_NAN4;
#pragma unroll
      for (int i = 0; i < T::CH; ++i) {
        kr[i] = ((kr[i] & keep) ^ turn) | kn;
        vr[i] = (vr[i] & keep) | vn;
      }
      if (vn) vs = 1.0f;
    }
    if (pg >= pe) {
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < T::CH; ++i) {
        const int c = tid + 256 * i;
        vr[i] = keys_below(vr[i], pg * PAGE + 16 * (c % 4), vmax);
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t high = fp8x4_nan(vr[i][e]);
          bits |= bits_of(high) << 4 * e;
          vr[i][e] &= ~bytes_of(high);
        }
        odd_keys[c / 4][c % 4] = (uint16_t)bits;
        any |= bits;
      }
      const int found = __any(any != 0);
      if (lane == 0) odd_any[wave] = found;
      again |= found != 0;
    }
#pragma unroll
    for (int i = 0; i < T::CH; ++i) {
      const int c = tid + 256 * i, key = c / KS, kd = c % KS, d = c / 4, j = c % 4;
      const int kro = (key & ~12) | (key & 4) << 1 | (key & 8) >> 1;   // key's row: bits 2 and 3 exchanged
      uint8_t* kt = sk + buf * KB + kro * 2 * D + 16 * (2 * kd ^ T::key_turn(kro));
      uint8_t* vt = sv + buf * KB + d * 2 * PAGE + 16 * (2 * j ^ T::value_turn(d));
      const int ko = T::key_turn(kro) & 1 ? -16 : 16, vo = T::value_turn(d) & 1 ? -16 : 16;   // to chunk c ^ 1
      *reinterpret_cast<u32x4*>(kt) = fp8_to_bf16x8(kr[i][0], kr[i][1]);
      *reinterpret_cast<u32x4*>(kt + ko) = fp8_to_bf16x8(kr[i][2], kr[i][3]);
      u32x4 lo = fp8_to_bf16x8(vr[i][0], vr[i][1]), hi = fp8_to_bf16x8(vr[i][2], vr[i][3]);
      if (odd && !ordinary(vs)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = pack_bf16x2(bf16lo(lo[e]) * vs, bf16hi(lo[e]) * vs);
          hi[e] = pack_bf16x2(bf16lo(hi[e]) * vs, bf16hi(hi[e]) * vs);
        }
      }
      *reinterpret_cast<u32x4*>(vt) = lo;
      *reinterpret_cast<u32x4*>(vt + vo) = hi;
    }
  };

  f32x16 O[DB], S[2];
  u32x4 pf[2][2];
  float m, l;   // the exponent's offset (log2 units), this lane's part of the sum
  // This lane's chunk 2 g + h of its row of K, 2 s + h of its row of V: 32 g or 32 s exchanged into the address of the first.
  const uint32_t kl = lr * 2 * D + 16 * (h ^ T::key_turn(lr)), vl = lr * 2 * PAGE + 16 * (h ^ T::value_turn(lr));
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < DB; ++db) O[db] = f32x16{};
    m = -INFINITY;
    l = 0.0f;
  };
  auto scores = [&](int buf) __attribute__((always_inline)) {
    S[0] = S[1] = f32x16{};
#pragma unroll
    for (int g = 0; g < KS; ++g)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) S[hf] = mfma_bf16_32x32x16(ld16(sk + (kl ^ 32 * g) + buf * KB + hf * 64 * D), qf[g], S[hf]);
  };
  auto masked = [&](int pg) __attribute__((always_inline)) {   // register 8 s + 4 a + i: key 16 s + 4 a + i of the lane's
    const int key0 = pg * PAGE + 8 * h;
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (key0 + 16 * (r / 8) + r % 8 >= vis) S[r / 16][r % 16] = -INFINITY;
  };
  auto top_of = [&](const Kv8Scale& w) __attribute__((always_inline)) {   // the row's largest score
    float hi = S[0][0];
#pragma unroll
    for (int r = 1; r < 32; ++r) hi = fmaxf(hi, S[r / 16][r % 16]);
    return other_half_max(__builtin_fmaf(hi, w.f, w.at));
  };
  auto softmax = [&](const Kv8Scale& w, auto large) __attribute__((always_inline)) {   // large: scores of any size (KV8_LARGE)
    const float base = m == -INFINITY ? 0.0f : m, off = base - w.lv;
    auto power = [&](float score) __attribute__((always_inline)) {
#pragma clang fp contract(off)
      if (large) {
        const float rounded = score * w.f;
        return __builtin_amdgcn_exp2f(rounded - base + w.lv);
      }
      return __builtin_amdgcn_exp2f(__builtin_fmaf(score, w.f, -off));
    };
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < 32; r += 2) {
      const int hf = r / 16, q = r % 16;
      const uint32_t x = pack_bf16x2(power(S[hf][q]), power(S[hf][q + 1]));
      pf[hf][q / 8][q % 8 / 2] = x;
      sum[hf] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), __builtin_bit_cast(bf16x2, 0x3F803F80u), sum[hf], false);
    }
    l = __builtin_fmaf(sum[0] + sum[1], w.inv, l);
  };
  auto values = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int db = 0; db < DB; ++db)
        O[db] = mfma_bf16_32x32x16(ld16(sv + (vl ^ 32 * s) + buf * KB + db * 64 * PAGE), pf[s / 2][s % 2], O[db]);
  };
  clear();
  if (p0 < p1) {
    look_up(p0);
    load(p0);
    look_scales_up();
    store(p0, 0);
    Kv8Scale now = scale_in(p0);
    again |= __builtin_amdgcn_readlane(ids, 0) < 0;
    __syncthreads();
    auto stage = [&](int pg, int buf) __attribute__((always_inline)) {
      const int next = min(pg + 1, p1 - 1);
      if (next - first >= 64) {
        look_up(next);
        look_scales_up();
      }
      load(next);
      scores(buf);
      if (pg >= pe) masked(pg);
      if (pg == p0) m = top_of(now);
      softmax(now, std::false_type{});
      values(buf);
      store(next, buf ^ 1);
      now = scale_in(next);
      __syncthreads();
    };
    for (int pg = p0; pg < p1; pg += 2) {
      stage(pg, 0);
      if (pg + 1 < p1) stage(pg + 1, 1);
    }
  }
  again |= !(l <= 0x1p64f);   // infinities and NaN among them
  again |= vis > p0 * PAGE && p0 < p1 && !(fabsf(m) < KV8_LARGE);   // -infinity too: of keys that are seen, it tells nothing of the others
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) again |= !(fabsf(O[db][r]) < INFINITY);
  if (__syncthreads_or(again)) {
    clear();
    for (int pg = p0; pg < p1; ++pg) {
      if ((pg - p0) % 64 == 0) {
        look_up(pg);
        look_scales_up();
      }
      load(pg);
      __syncthreads();
      store(pg, 0);
      const Kv8Scale w = scale_in(pg);
      __syncthreads();
      scores(0);
      if (pg >= pe) {
        masked(pg);
        // rows that see a key whose value is not a number
        if (odd_any[0] | odd_any[1] | odd_any[2] | odd_any[3]) {
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            f32x16 hit = {};
#pragma unroll
            for (int s = 0; s < 4; ++s)
              hit = mfma_bf16_32x32x16(ones_of(odd_keys[32 * db + lr][s] >> 8 * h & 0xFFu),
                                       ones_of(bits_below(pg * PAGE + 16 * s + 8 * h, vis)), hit);
#pragma unroll
            for (int r = 0; r < 16; ++r) O[db][r] = hit[r] > 0.0f ? __builtin_nanf("") : O[db][r];
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      const float mn = fmaxf(m, top_of(w)), alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) O[db] *= alpha;
      softmax(w, std::true_type{});
      values(0);
    }
  }
  l += __shfl_xor(l, 32, 64);
  const int r = t.r0 + 32 * wave + lr;
  if (r >= t.rows) return;
  if (piece < 0) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* out = p.o + ((long)(t.row0 + r / p.G) * p.H + hk * p.G + r % p.G) * D + 4 * h;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<u32x2*>(out + 32 * db + 8 * q) = u32x2{pack_bf16x2(O[db][4 * q] * inv, O[db][4 * q + 1] * inv),
                                                                 pack_bf16x2(O[db][4 * q + 2] * inv, O[db][4 * q + 3] * inv)};
    return;
  }
  const long at = (long)piece * T::R + r - t.r0;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(p.part_o + at * D + 32 * db + 8 * q + 4 * h) =
          f32x4{O[db][4 * q], O[db][4 * q + 1], O[db][4 * q + 2], O[db][4 * q + 3]};
  if (h == 0) {
    p.part_ml[2 * at] = m;
    p.part_ml[2 * at + 1] = l;
  }
}

struct Kv8Plan {
  bool many;
  int rows;     // of a tile
  int numbers;  // of tiles, those of no tile among them
  int splits;   // pieces of a tile along the keys
  int run;      // Kv8Args::run
  int whole;    // many rows: an XCD's tiles that are not split
  long pieces;  // partial results
};

long kv8_all(const Kv8Plan& pl, int Hkv) { return kv8_each(pl.numbers, Hkv) * (Hkv / kv8_shared(Hkv)); }   // an XCD's tiles

// Sequences are as long as the table is wide at most, and shorter ones split into shorter pieces, a page or none each where the table
// is much wider (32 tokens over 2000 keys each: a table of 33 pages 36 us, of 129 or 2049 49).
Kv8Plan kv8_plan(const Kv8Cache& c, int H, bool causal) {
  const long G = H / c.Hkv, rows = c.N * G;
  Kv8Plan pl{};
  // A page that is read for 16 rows takes the few-rows kernel's 16 x 16 products through all of it again for the next 16; the
  // other kernel reads it once for 128 rows, but a workgroup of it that is not full takes as long as a full one.  Rows
  // (of heads) a sequence at most, ragged up to 4096 keys, 12 heads of 128, few / many rows kernel: 8 x 128 30 / 46 us, 8 x 256
  // 47 / 53, 32 x 64 75 / 102; 1 x 308 of 65536 (two and a half tiles) 340 / 210.
  // One kernel serves all of a batch, by its rows in the mean: a prompt among single tokens takes longer than the two apart (2000
  // tokens over 6096 and 31 over 4096 500 us, 286 and 65 apart; 4352 and 31 356, 260 and 65).
  pl.many = rows > 256L * c.B;
  pl.rows = pl.many ? 128 : 16;
  pl.numbers = (int)(rows / pl.rows + c.B + 1);
  if (!pl.many) {
    const long busy = ((rows + 15) / 16 > c.B ? (rows + 15) / 16 : c.B) * c.Hkv;
    // One workgroup a CU reads fastest where there are no more (131072 tokens, 12 heads, in 252 pieces 69 us, 312 84, 504 72).
    // Up to 512 tiles in two pieces each fill the last round better (32 sequences of up to 8192 tokens, 12 heads: 88 us, in
    // one piece 99), longer tables alone (64 of up to 2048, 4 heads of 64, in one piece 16, two 19.5).
    const long want = busy <= 256 ? 256 / busy : busy <= 512 ? 2 : 1, most = c.W / (busy <= 256 ? 16 : 64);
    pl.splits = (int)(want > KV8_SPLITS ? KV8_SPLITS : want);
    if (pl.splits > most) pl.splits = (int)most;
    if (pl.splits < 1) pl.splits = 1;
    pl.pieces = pl.splits == 1 ? 0 : (long)pl.numbers * c.Hkv * pl.splits;
    return pl;
  }
  // 64 workgroups run on an XCD at a time
  const long tiles = (rows + 127) / 128 > c.B ? (rows + 127) / 128 : c.B;   // as many as there can be, all about equal
  const long each = kv8_each(tiles, c.Hkv) * (c.Hkv / kv8_shared(c.Hkv)), all = kv8_all(pl, c.Hkv);
  const long rounds = each / 64, rest = each % 64, most = c.W / 4;
  pl.whole = (int)all;
  pl.splits = 1;
  if (rest && (rounds == 0 || !causal)) {
    long want = 64 / rest;
    // Tiles that take more than half of the places are not split evenly, and the longest would run alone at the end: there a
    // batch's longer sequences are cut into up to three pieces, about as long as a place's share of all (6 sequences of 900 to
    // 9000 keys, 12 heads of 128: 251 us, so 168; 4 of 940 to 6000, 4 heads of 64, 117 and 86).  With fewer tiles it brings
    // nothing, as two workgroups of a CU get done 1.2 times as much as one (three chunks over 5000 keys and less 42 us, so 53).
    if (rounds == 0 && want == 1 && c.B > 1 && c.B < 63) {   // a lane for each sequence
      want = 3;
      pl.run = (int)(512 / c.Hkv > 1 ? 512 / c.Hkv : 1);
    }
    pl.splits = (int)(want > (rounds ? 8 : KV8_SPLITS) ? (rounds ? 8 : KV8_SPLITS) : want);
    if (pl.splits > most) pl.splits = (int)most;
    if (pl.splits > 1) pl.whole = (int)(rounds == 0 ? 0 : all - rest);
    else pl.splits = 1;
  }
  pl.pieces = 8 * (all - pl.whole) * pl.splits;
  return pl;
}

template <int D>
hipError_t launch_attention(const Kv8Args& a, const Kv8Plan& pl, hipStream_t st) {
  if (pl.many) {
    const int all = (int)kv8_all(pl, a.c.Hkv);
    kv8_many_kernel<D><<<(unsigned)(8 * (pl.whole + (all - pl.whole) * pl.splits)), 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || pl.pieces == 0) return e;
    kv8_join_kernel<D, 128, 1><<<(unsigned)(8 * (all - pl.whole) * 16), 256, 0, st>>>(a);
  } else {
    const unsigned tiles = (unsigned)(pl.numbers * a.c.Hkv);
    kv8_rows_kernel<D><<<tiles * pl.splits, 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || pl.pieces == 0) return e;
    kv8_join_kernel<D, 16, 4><<<tiles * 8, 256, 0, st>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_append(const Kv8Cache& c, const uint16_t* k, long ldk, const uint16_t* v, long ldv,
                             hipStream_t st) {
  const unsigned grid = (unsigned)((c.N / PAGE + 2L * c.B) * c.Hkv);
  if (c.D == 128) kv8_append_kernel<128><<<grid, 256, 0, st>>>(c, k, ldk, v, ldv);
  else kv8_append_kernel<64><<<grid, 256, 0, st>>>(c, k, ldk, v, ldv);
  return hipGetLastError();
}

long kv8_attention_workspace_bytes(const Kv8Cache& c, int H, int causal) {
  const Kv8Plan pl = kv8_plan(c, H, causal);
  return pl.pieces * pl.rows * (c.D + 2) * 4;
}

int kv8_attention_kernel(const Kv8Cache& c, int H, int causal, int& splits, int& whole, int& tiles) {
  const Kv8Plan pl = kv8_plan(c, H, causal);
  splits = pl.splits;
  whole = pl.whole;
  tiles = pl.many ? (int)kv8_all(pl, c.Hkv) : pl.numbers;
  return !pl.many ? KV8_FEW : pl.splits > 1 && pl.run ? KV8_MANY_RAGGED : KV8_MANY;
}

hipError_t launch_kv8_attention(const Kv8Cache& c, const Kv8Attention& a, void* workspace, hipStream_t st) {
  const Kv8Plan pl = kv8_plan(c, a.H, a.causal);
  float* part = static_cast<float*>(workspace);
  const Kv8Args args{c, a.q, a.ldq, a.o, a.H, a.H / c.Hkv, a.causal, pl.splits, pl.splits > 1 ? pl.run : 0, pl.numbers, pl.whole,
                     a.scale * 1.4426950408889634f, part, part + pl.pieces * pl.rows * c.D};
  return c.D == 128 ? launch_attention<128>(args, pl, st) : launch_attention<64>(args, pl, st);
}

}  // namespace svdq
