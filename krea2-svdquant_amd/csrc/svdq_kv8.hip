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
// append:  a page's scale is that of its new tokens (svdq_fp8.h), or the larger of that and the one it has where it holds
//          tokens already; those are then rounded again under the new scale.
// attend:  o = sum over visible j of softmax_j(scale q . k_j) v_j,  j < length, and with a causal mask, for the i-th of n new
//          tokens, j <= length - n + i; 0 where nothing is visible.
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
__device__ __forceinline__ int find_sequence(const Kv8Cache& c, long number, int mult, int unit, int extra) {
  int before = 0;
  for (int b0 = 1; b0 <= c.B; b0 += 64) {
    const int b = b0 + (threadIdx.x & 63);
    before += __popcll(__ballot(b <= c.B && first_unit(c, b, mult, unit, extra) <= number));
  }
  return __builtin_amdgcn_readfirstlane(before);
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
// of a token a thread and round) while their largest magnitudes are found.
template <int D>
__global__ void __launch_bounds__(256) kv8_append_kernel(Kv8Cache c, const uint16_t* __restrict__ k, long ldk,
                                                         const uint16_t* __restrict__ v, long ldv) {
  constexpr int CH = D / 8, ROUNDS = PAGE * CH / 256;   // chunks of 8 channels of a token
  __shared__ uint32_t tops[2][4];
  __shared__ __attribute__((aligned(16))) uint8_t turn[D * PAGE];
  const int tid = threadIdx.x, head = blockIdx.x % c.Hkv;
  const long number = blockIdx.x / c.Hkv;
  const int b = find_sequence(c, number, 1, PAGE, 2);
  if (b >= c.B) return;
  const int row0 = first_row(c, b), n = first_row(c, b + 1) - row0;
  if (n <= 0) return;
  const long start = min(max(c.lengths[b], 0), c.W * PAGE);
  const long page = start / PAGE + (number - first_unit(c, b, 1, PAGE, 2));
  if (page >= c.W || page * PAGE >= start + n) return;
  const int id = c.table[(long)b * c.W + page];
  if (id < 0 || id >= c.P) return;
  const int lo = (int)max(start - page * PAGE, 0L), hi = (int)min(start + n - page * PAGE, (long)PAGE);
  const long base = row0 + page * PAGE - start;   // row of the page's slot 0
  const long at = (long)id * c.Hkv + head;
  uint8_t *kc = c.kc + at * PAGE * D, *vc = c.vc + at * PAGE * D;

  u32x4 x[2][ROUNDS];
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int slot = (tid + 256 * i) / CH, ch = (tid + 256 * i) % CH;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      x[w][i] = u32x4{};
      if (slot >= lo && slot < hi) x[w][i] = ld16((w ? v + (base + slot) * ldv : k + (base + slot) * ldk) + head * D + 8 * ch);
    }
  }
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
  __syncthreads();
  float s[2], again[2];   // the page's scales, and what its older codes are multiplied by
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    s[w] = fp8_scale(max(max(tops[w][0], tops[w][1]), max(tops[w][2], tops[w][3])));
    again[w] = 1.0f;
    if (lo > 0) {
      const float before = c.scales[2 * at + w];
      if (before >= s[w]) {
        s[w] = before;
      } else {
        again[w] = before / s[w];
      }
    }
  }
  __syncthreads();   // the scales have been read
  if (tid < 2) c.scales[2 * at + tid] = tid ? s[1] : s[0];
  auto encode = [](u32x4 r, float s) {
    if (__float_as_uint(s) & 0x7FFFFFu) {   // a scale of the caller's, no power of two: the conversion takes only those
      auto over = [&](float v) {
        const float q = v / s;
        return sticky(q, __builtin_fmaf(-q, s, v));   // s > 0: it is at least what the new tokens need
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
    const int slot = (tid + 256 * i) / CH, ch = (tid + 256 * i) % CH;
    u32x2* kd = reinterpret_cast<u32x2*>(kc + slot * D + 8 * ch);
    if (slot >= lo && slot < hi) {
      *kd = encode(x[0][i], s[0]);
      const u32x2 o = encode(x[1][i], s[1]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint8_t q = (uint8_t)(o[e / 4] >> (8 * (e % 4)));
        if (whole) turn[(8 * ch + e) * PAGE + (slot ^ (ch % 16 * 4))] = q;   // spread over the banks
        else vc[(8 * ch + e) * PAGE + slot] = q;
      }
    } else if (slot < lo && again[0] != 1.0f) {
      const u32x2 old = *kd;
      *kd = u32x2{scaled(old[0], again[0]), scaled(old[1], again[0])};
    }
  }
  if (whole) {
    __syncthreads();
    for (int i = tid; i < D * PAGE / 16; i += 256) {
      const int d = i / 4, key = 16 * (i % 4), f = d / 8 % 16 * 4;
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = *reinterpret_cast<const uint32_t*>(turn + d * PAGE + ((key + 4 * e) ^ f));
      *reinterpret_cast<u32x4*>(vc + d * PAGE + key) = o;
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
  int H, G, causal, splits;
  float scale_log2;
  float* part_o;    // [tile, split, rows, D]
  float* part_ml;   // [tile, split, rows, 2]: maximum (log2 units), sum
};

struct Kv8Tile {
  int b, row0, n, rows, r0, len;   // sequence, its first row of q and tokens, its rows of heads, the tile's first, tokens held
};
template <int R>
__device__ __forceinline__ bool kv8_tile(const Kv8Args& p, long number, Kv8Tile& t) {
  t.b = find_sequence(p.c, number, p.G, R, 1);
  t.row0 = first_row(p.c, t.b);
  t.n = max(first_row(p.c, t.b + 1) - t.row0, 0);
  t.rows = t.n * p.G;
  const long r0 = (number - first_unit(p.c, t.b, p.G, R, 1)) * R;
  if (r0 >= t.rows) return false;
  t.r0 = (int)r0;
  t.len = t.b == p.c.B ? 0 : min(max(p.c.lengths[t.b], 0), p.c.W * PAGE);
  return true;
}
// keys that the row's token sees
__device__ __forceinline__ int kv8_visible(const Kv8Args& p, const Kv8Tile& t, int row) {
  return p.causal ? max(t.len - t.n + row / p.G + 1, 0) : t.len;
}

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Masked keys have probability 0, but 0 times a code that is not a number is not: where masked keys may hold such codes,
// they are taken out of the values, and the rows that do see them get them from a product of their own.
__device__ __forceinline__ uint32_t bf16x2_nan(uint32_t x) {   // 0xFFFF in the halves that are not a number
  const uint32_t lo = (x & 0x7FFFu) > 0x7F80u ? 0xFFFFu : 0u, hi = (x & 0x7FFF0000u) > 0x7F800000u ? 0xFFFF0000u : 0u;
  return lo | hi;
}
__device__ __forceinline__ u32x4 bf16x8_nan(u32x4 x) {
  return u32x4{bf16x2_nan(x[0]), bf16x2_nan(x[1]), bf16x2_nan(x[2]), bf16x2_nan(x[3])};
}
// bytes of 16 keys from key `from` that lie below `end`
__device__ __forceinline__ u32x4 keys_below(u32x4 x, int from, int end) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int n = end - from - 4 * d;
    x[d] = n >= 4 ? x[d] : n <= 0 ? 0u : x[d] & ((1u << (8 * n)) - 1u);
  }
  return x;
}

// Few rows: 16 of them a workgroup, whose four waves take the split's pages in turn, each with a softmax of its own; they are
// joined in LDS at the end.  Pages go from memory straight into the operands of the matrix instructions: a lane's 16 bytes of
// keys are 16 channels of the key in its row of K, its 16 bytes of values 16 keys of one channel.
//   S^T = K Q^T: row 4 g + i of tile t stands for key 16 g + 4 t + i, so lane group g gets the probabilities of the 16 keys that
//   it holds values of; O^T += V^T P^T takes them as they are, tiles 2 u and 2 u + 1 in step u.
template <int D>
__global__ void __launch_bounds__(256) kv8_rows_kernel(Kv8Args p) {
  constexpr int R = 16, SP = D / 64, DT = D / 16, PITCH = D + 4;
  __shared__ __attribute__((aligned(16))) float so[4][R * PITCH];
  __shared__ float sml[4][R][2];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = blockIdx.x % p.splits;
  const int tile = blockIdx.x / p.splits, hk = tile % p.c.Hkv;
  Kv8Tile t;
  if (!kv8_tile<R>(p, tile / p.c.Hkv, t)) return;
  const int row = min(t.r0 + lr, t.rows - 1);
  const int vis = kv8_visible(p, t, row);
  const int vmin = kv8_visible(p, t, t.r0), vmax = kv8_visible(p, t, min(t.r0 + R, t.rows) - 1);
  const int pages = (vmax + PAGE - 1) / PAGE, per = (pages + p.splits - 1) / p.splits;
  const int p0 = split * per, p1 = min(p0 + per, pages);

  u32x4 qf[2 * SP];
  const uint16_t* qr = p.q + (long)(t.row0 + row / p.G) * p.ldq + (hk * p.G + row % p.G) * D + 16 * g;
#pragma unroll
  for (int s = 0; s < 2 * SP; ++s) qf[s] = ld16(qr + 64 * (s / 2) + 8 * (s % 2));

  f32x4 O[DT] = {};
  float m = -INFINITY, l = 0.0f;
  const int* table = p.c.table + (long)t.b * p.c.W;
  for (int pg = p0 + wave; pg < p1; pg += 4) {
    const int id = table[pg];
    if (id < 0 || id >= p.c.P) continue;
    const long at = (long)id * p.c.Hkv + hk;
    const uint8_t *kc = p.c.kc + at * PAGE * D + (16 * (lr >> 2) + (lr & 3)) * D + 16 * g, *vc = p.c.vc + at * PAGE * D + lr * PAGE + 16 * g;
    const float ks = p.c.scales[2 * at] * p.scale_log2, vs = p.c.scales[2 * at + 1];
    u32x4 kq[4][SP], vq[DT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int s = 0; s < SP; ++s) kq[i][s] = ld16(kc + 4 * i * D + 64 * s);
#pragma unroll
    for (int d = 0; d < DT; ++d) vq[d] = ld16(vc + 16 * d * PAGE);
    f32x4 S[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      S[i] = f32x4{};
#pragma unroll
      for (int s = 0; s < SP; ++s) {
        S[i] = mfma_bf16_16x16x32(fp8_to_bf16x8(kq[i][s][0], kq[i][s][1]), qf[2 * s], S[i]);
        S[i] = mfma_bf16_16x16x32(fp8_to_bf16x8(kq[i][s][2], kq[i][s][3]), qf[2 * s + 1], S[i]);
      }
    }
    const int key0 = pg * PAGE + 16 * g;
    const bool edge = pg * PAGE + PAGE > vmin;   // some row does not see all of the page
    if (edge) {
#pragma unroll
      for (int d = 0; d < DT; ++d) vq[d] = keys_below(vq[d], key0, vmax);
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        S[i][r] = edge && key0 + 4 * i + r >= vis ? -INFINITY : S[i][r] * ks;
        top = fmaxf(top, S[i][r]);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    m = mn;
    l *= alpha;
    u32x4 pf[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        S[i][r] = __builtin_amdgcn_exp2f(S[i][r] - base);
        l += S[i][r];
      }
      pf[i / 2][2 * (i % 2)] = pack_bf16x2(S[i][0] * vs, S[i][1] * vs);
      pf[i / 2][2 * (i % 2) + 1] = pack_bf16x2(S[i][2] * vs, S[i][3] * vs);
    }
    uint32_t odd = 0;   // codes that are not a number, in a page of which rows see different parts
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int r = 0; r < 4; ++r) O[d][r] *= alpha;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 vf = fp8_to_bf16x8(vq[d][2 * u], vq[d][2 * u + 1]);
        if (edge) {
          const u32x4 bad = bf16x8_nan(vf);
          vf &= ~bad;
          odd |= bad[0] | bad[1] | bad[2] | bad[3];
        }
        O[d] = mfma_bf16_16x16x32(vf, pf[u], O[d]);
      }
    }
    if (edge && __any(odd != 0)) {
      u32x4 seen[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          seen[u][e] = (key0 + 8 * u + 2 * e < vis ? 0x3F80u : 0u) | (key0 + 8 * u + 2 * e + 1 < vis ? 0x3F800000u : 0u);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f32x4 hit = {};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u32x4 bad = bf16x8_nan(fp8_to_bf16x8(vq[d][2 * u], vq[d][2 * u + 1])) & 0x3F803F80u;
          hit = mfma_bf16_16x16x32(bad, seen[u], hit);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) O[d][r] = hit[r] > 0.0f ? __builtin_nanf("") : O[d][r];
      }
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&so[wave][lr * PITCH + 16 * d + 4 * g]) = O[d];
  if (g == 0) {
    sml[wave][lr][0] = m;
    sml[wave][lr][1] = l;
  }
  __syncthreads();
  // 16 threads a row
  const int r = tid >> 4, c0 = (tid & 15) * (D / 16);
  float mm = -INFINITY, ll = 0.0f, o[D / 16] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[w][r][0]);
  const float base = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(sml[w][r][0] - base);
    ll += f * sml[w][r][1];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] += f * so[w][r * PITCH + c0 + i];
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
  const long at = (long)blockIdx.x * R + r;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) p.part_o[at * D + c0 + i] = o[i];
  if ((tid & 15) == 0) {
    p.part_ml[2 * at] = mm;
    p.part_ml[2 * at + 1] = ll;
  }
}

// Joins the splits of 16 rows of a tile of R.
template <int D, int R>
__global__ void __launch_bounds__(256) kv8_join_kernel(Kv8Args p) {
  const int tile = blockIdx.x / (R / 16), part = blockIdx.x % (R / 16), hk = tile % p.c.Hkv;
  Kv8Tile t;
  if (!kv8_tile<R>(p, tile / p.c.Hkv, t)) return;
  const int r = 16 * part + (threadIdx.x >> 4), c0 = (threadIdx.x & 15) * (D / 16);
  if (t.r0 + r >= t.rows) return;
  const long first = (long)tile * p.splits * R + r;
  float mm = -INFINITY, ll = 0.0f, o[D / 16] = {};
  for (int s = 0; s < p.splits; ++s) mm = fmaxf(mm, p.part_ml[2 * (first + (long)s * R)]);
  const float base = mm == -INFINITY ? 0.0f : mm;
  for (int s = 0; s < p.splits; ++s) {
    const long at = first + (long)s * R;
    const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * at] - base);
    ll += f * p.part_ml[2 * at + 1];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] += f * p.part_o[at * D + c0 + i];
  }
  const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
  uint16_t* out = p.o + ((long)(t.row0 + (t.r0 + r) / p.G) * p.H + hk * p.G + (t.r0 + r) % p.G) * D + c0;
#pragma unroll
  for (int i = 0; i < D / 16; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
}

// Many rows: 32 a wave, 128 a workgroup; pages go through LDS, as bf16, for its four waves.  A lane holds one row's scores of half of
// the keys.  Row 16 s + 8 a + 4 h + i of K in LDS order is key 16 s + 8 h + 4 a + i of the page (bits 2 and 3 exchanged), so that the
// probabilities leave the softmax in the values' order.
template <int D>
struct Kv8Many {
  static constexpr int R = 128, KP = 2 * D + 16, VP = 2 * PAGE + 16, CH = PAGE * D / 16 / 256;
};

template <int D>
__global__ void __launch_bounds__(256, 2) kv8_many_kernel(Kv8Args p) {
  using T = Kv8Many<D>;
  __shared__ __attribute__((aligned(16))) uint8_t sk[2][PAGE * T::KP];
  __shared__ __attribute__((aligned(16))) uint8_t sv[2][D * T::VP];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = blockIdx.x % p.splits;
  const int tile = blockIdx.x / p.splits, hk = tile % p.c.Hkv;
  Kv8Tile t;
  if (!kv8_tile<T::R>(p, tile / p.c.Hkv, t)) return;
  const int row = min(t.r0 + 32 * wave + lr, t.rows - 1);
  const int vis = kv8_visible(p, t, row);
  const int vmin = kv8_visible(p, t, t.r0), vmax = kv8_visible(p, t, min(t.r0 + T::R, t.rows) - 1);
  const int pages = (vmax + PAGE - 1) / PAGE, per = (pages + p.splits - 1) / p.splits;
  const int p0 = split * per, p1 = min(p0 + per, pages);

  u32x4 qf[D / 16];
  const uint16_t* qr = p.q + (long)(t.row0 + row / p.G) * p.ldq + (hk * p.G + row % p.G) * D + 8 * h;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qf[s] = ld16(qr + 16 * s);

  const int* table = p.c.table + (long)t.b * p.c.W;
  u32x4 kr[T::CH], vr[T::CH];
  float ks_next = 0.0f, vs_next = 0.0f;
  bool have_next = false;
  auto load = [&](int pg) {
    const int id = table[pg];
    have_next = id >= 0 && id < p.c.P;
    const long at = (long)(have_next ? id : 0) * p.c.Hkv + hk;
    ks_next = p.c.scales[2 * at] * p.scale_log2;
    vs_next = p.c.scales[2 * at + 1];
#pragma unroll
    for (int i = 0; i < T::CH; ++i) {
      kr[i] = ld16(p.c.kc + at * PAGE * D + 16 * (tid + 256 * i));
      vr[i] = ld16(p.c.vc + at * PAGE * D + 16 * (tid + 256 * i));
    }
  };
  auto store = [&](int pg, int buf) {
#pragma unroll
    for (int i = 0; i < T::CH; ++i) {
      const int c = tid + 256 * i, key = c / (D / 16), kd = c % (D / 16), d = c / 4, vk = 16 * (c % 4);
      // key's row: bits 2 and 3 exchanged
      const int kro = (key & ~12) | (key & 4) << 1 | (key & 8) >> 1;
      *reinterpret_cast<u32x4*>(&sk[buf][kro * T::KP + 32 * kd]) = fp8_to_bf16x8(kr[i][0], kr[i][1]);
      *reinterpret_cast<u32x4*>(&sk[buf][kro * T::KP + 32 * kd + 16]) = fp8_to_bf16x8(kr[i][2], kr[i][3]);
      const u32x4 x = pg * PAGE + PAGE > vmax ? keys_below(vr[i], pg * PAGE + vk, vmax) : vr[i];
      *reinterpret_cast<u32x4*>(&sv[buf][d * T::VP + 2 * vk]) = fp8_to_bf16x8(x[0], x[1]);
      *reinterpret_cast<u32x4*>(&sv[buf][d * T::VP + 2 * vk + 16]) = fp8_to_bf16x8(x[2], x[3]);
    }
  };

  f32x16 O[D / 32] = {};
  float m = -INFINITY, l = 0.0f;
  if (p0 < p1) {
    load(p0);
    store(p0, 0);
  }
  float ks = ks_next, vs = vs_next;
  bool have = have_next;
  __syncthreads();
  for (int pg = p0; pg < p1; ++pg) {
    const int buf = (pg - p0) & 1;
    if (pg + 1 < p1) load(pg + 1);
    const bool edge = pg * PAGE + PAGE > vmin || !have;
    const int sees = have ? vis : 0;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      f32x16 S = {};
      const uint8_t* ka = &sk[buf][(32 * hf + lr) * T::KP + 16 * h];
#pragma unroll
      for (int s = 0; s < D / 16; ++s) S = mfma_bf16_32x32x16(ld16(ka + 32 * s), qf[s], S);
      const int key0 = pg * PAGE + 32 * hf + 8 * h;   // register 8 s + 4 a + i: key 16 s + 4 a + i further
      float top = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        S[r] = edge && key0 + 16 * (r / 8) + r % 8 >= sees ? -INFINITY : S[r] * ks;
        top = fmaxf(top, S[r]);
      }
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      m = mn;
      l *= alpha;
      u32x4 pf[2];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float a = __builtin_amdgcn_exp2f(S[r] - base), b = __builtin_amdgcn_exp2f(S[r + 1] - base);
        l += a + b;
        pf[r / 8][r % 8 / 2] = pack_bf16x2(a * vs, b * vs);
      }
      if (!have) pf[0] = pf[1] = u32x4{};   // 0 times a scale that is not there
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
#pragma unroll
        for (int r = 0; r < 16; ++r) O[db][r] *= alpha;
        const uint8_t* va = &sv[buf][(32 * db + lr) * T::VP + 16 * h + 64 * hf];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          u32x4 vf = ld16(va + 32 * s);
          if (edge) {
            const u32x4 bad = bf16x8_nan(vf);
            vf &= ~bad;
            if (have && __any((bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
              u32x4 seen;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                seen[e] = (key0 + 16 * s + 2 * e < vis ? 0x3F80u : 0u) | (key0 + 16 * s + 2 * e + 1 < vis ? 0x3F800000u : 0u);
              const f32x16 hit = mfma_bf16_32x32x16(bad & 0x3F803F80u, seen, f32x16{});
#pragma unroll
              for (int r = 0; r < 16; ++r) O[db][r] = hit[r] > 0.0f ? __builtin_nanf("") : O[db][r];
            }
          }
          O[db] = mfma_bf16_32x32x16(vf, pf[s], O[db]);
        }
      }
    }
    if (pg + 1 < p1) store(pg + 1, buf ^ 1);
    ks = ks_next;
    vs = vs_next;
    have = have_next;
    __syncthreads();
  }
  l += __shfl_xor(l, 32, 64);
  if (t.r0 + 32 * wave + lr >= t.rows) return;
  if (p.splits == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* out = p.o + ((long)(t.row0 + row / p.G) * p.H + hk * p.G + row % p.G) * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<u32x2*>(out + 32 * db + 8 * q) = u32x2{pack_bf16x2(O[db][4 * q] * inv, O[db][4 * q + 1] * inv),
                                                                 pack_bf16x2(O[db][4 * q + 2] * inv, O[db][4 * q + 3] * inv)};
    return;
  }
  const long at = (long)blockIdx.x * T::R + 32 * wave + lr;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
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
  int rows;      // of a tile
  long tiles;    // numbers of tiles times key / value heads, those of no tile among them
  int splits;
};

// Up to 16 rows a sequence on average take the kernel for few rows.  Splits: until the card is full, two pages a wave at least.
Kv8Plan kv8_plan(const Kv8Cache& c, int H) {
  const long G = H / c.Hkv, rows = c.N * G;
  Kv8Plan pl;
  pl.many = rows > 32L * c.B;
  pl.rows = pl.many ? 128 : 16;
  pl.tiles = (rows / pl.rows + c.B + 1) * c.Hkv;
  const long busy = ((rows + pl.rows - 1) / pl.rows > c.B ? (rows + pl.rows - 1) / pl.rows : c.B) * c.Hkv;
  const long want = (pl.many ? 512 : 1024) / (busy > 0 ? busy : 1), most = pl.many ? c.W / 4 : c.W / 8;
  pl.splits = (int)(want < 1 ? 1 : want > 128 ? 128 : want);
  if (pl.splits > most) pl.splits = most < 1 ? 1 : (int)most;
  while (pl.splits > 1 && pl.tiles * pl.splits > (long)(UINT32_MAX / 256)) pl.splits /= 2;   // more than a launch holds
  return pl;
}

template <int D>
hipError_t launch_attention(const Kv8Args& a, const Kv8Plan& pl, hipStream_t st) {
  const unsigned grid = (unsigned)(pl.tiles * pl.splits);
  if (pl.many) kv8_many_kernel<D><<<grid, 256, 0, st>>>(a);
  else kv8_rows_kernel<D><<<grid, 256, 0, st>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || pl.splits == 1) return e;
  if (pl.many) kv8_join_kernel<D, 128><<<(unsigned)(pl.tiles * 8), 256, 0, st>>>(a);
  else kv8_join_kernel<D, 16><<<(unsigned)pl.tiles, 256, 0, st>>>(a);
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

long kv8_attention_workspace_bytes(const Kv8Cache& c, int H) {
  const Kv8Plan pl = kv8_plan(c, H);
  return pl.splits == 1 ? 0 : pl.tiles * pl.splits * pl.rows * (c.D + 2) * 4;
}

hipError_t launch_kv8_attention(const Kv8Cache& c, const Kv8Attention& a, void* workspace, hipStream_t st) {
  const Kv8Plan pl = kv8_plan(c, a.H);
  float* part = static_cast<float*>(workspace);
  const Kv8Args args{c, a.q, a.ldq, a.o, a.H, a.H / c.Hkv, a.causal, pl.splits, a.scale * 1.4426950408889634f,
                     part, part + pl.tiles * pl.splits * pl.rows * c.D};
  return c.D == 128 ? launch_attention<128>(args, pl, st) : launch_attention<64>(args, pl, st);
}

}  // namespace svdq
