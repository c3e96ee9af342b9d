// bf16 activations into E4M3 codes with a float32 scale for each 128 columns of a row:
//   s = the smallest power of two >= 2^-126 with max |v| <= 448 s,   q = E4M3(v / s), ties to even
// Rows of kp = K rounded up to 128 codes (zeros beyond K); scales are [kp / 128, M], so that the rows of a tile of the product
// lie side by side.  HBM-bound: one read, one write of half the bytes; 77 x 6144 2.6 us, 4352 x 6144 15.5 (5.2 TB/s).
#include "svdq_fp8.h"
#include "svdq_kernels.h"

namespace svdq {
namespace {

// the largest over the 16 lanes of a row of the wave
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true));   // row_ror:8
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xF, 0xF, true));
}

// A wave takes 512 columns of a row: 8 a lane, 16 lanes a block.  VEC: rows start on 16 bytes and K % 8 == 0.
template <bool VEC>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const uint16_t* __restrict__ x, long ldx, long units, int M,
                                                           int K, uint8_t* __restrict__ codes,
                                                           float* __restrict__ scales) {
  const int kp = (int)fp8_kp(K), per_row = (kp + 511) / 512, lane = threadIdx.x & 63;
  const long unit = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= units) return;
  const long row = unit / per_row;
  const int c = 512 * (int)(unit - row * per_row) + 8 * lane;
  const uint16_t* src = x + row * ldx + c;
  float v[8];
  if (VEC) {
    const u32x4 r = c < K ? *reinterpret_cast<const u32x4*>(src) : u32x4{};
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      v[2 * d] = bf16lo(r[d]);
      v[2 * d + 1] = bf16hi(r[d]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? bf16f(src[i]) : 0.0f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, fp8_magnitude(v[i]));
  const float s = fp8_scale(row16_max(top));
  if (c >= kp) return;
  const u32x2 o = {fp8_encode4(v[0], v[1], v[2], v[3], s), fp8_encode4(v[4], v[5], v[6], v[7], s)};
  *reinterpret_cast<u32x2*>(codes + row * kp + c) = o;
  if (lane % 16 == 0) scales[(long)(c / 128) * M + row] = s;
}

}  // namespace

hipError_t launch_fp8_quantize(const uint16_t* x, long ldx, int M, int K, uint8_t* codes, float* scales,
                               hipStream_t st) {
  const long units = (long)M * ((fp8_kp(K) + 511) / 512);
  const unsigned grid = (unsigned)((units + 3) / 4);
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && ldx % 8 == 0 && K % 8 == 0)
    fp8_quantize_kernel<true><<<grid, 256, 0, st>>>(x, ldx, units, M, K, codes, scales);
  else
    fp8_quantize_kernel<false><<<grid, 256, 0, st>>>(x, ldx, units, M, K, codes, scales);
  return hipGetLastError();
}

}  // namespace svdq
