// Device helpers that the attention kernels over the 8-bit cache share.
#pragma once

#include "attention_tiles.h"
#include "fp8.h"

namespace nvamd {

// s = K . q for 16 rows of codes (128 dims) and 16 columns of a query: lane (row or column n, gq) gives dims 16 gq .. +15
// and 64 + 16 gq .. +15 of either, the scale byte of its row, and that of block gq of its column.
__device__ __forceinline__ f32x4 mfma_fp8_fp8(const u32x4 (&k)[2], u32 k_scale, i32x8 q, u32 q_scale, f32x4 c) {
  const i32x8 codes = {(int)k[0][0], (int)k[0][1], (int)k[0][2], (int)k[0][3],
                       (int)k[1][0], (int)k[1][1], (int)k[1][2], (int)k[1][3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes, q, c, 0, 0, 0, (int)k_scale, 0, (int)q_scale);
}
__device__ __forceinline__ void score(f32x4 &s, const u32x4 (&k)[2], u32 k_scale, i32x8 q_hi, i32x8 q_lo, u32 q_scale) {
  s = mfma_fp8_fp8(k, k_scale, q_hi, q_scale, f32x4{0.f, 0.f, 0.f, 0.f});
  s = mfma_fp8_fp8(k, k_scale, q_lo, q_scale, s);
}

// Keeps a dim's first n tokens (any n) of a tile.
__device__ __forceinline__ void keep_tokens(u32x4 &codes, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i) codes[i] = keep_bytes(codes[i], n - 4 * i);
}
// The operand of V^T for 8 tokens of a dim: words i and i + 1 of its codes.
template <int I>
__device__ __forceinline__ u32x4 expand8(u32x4 codes, float scale) {
  return u32x4{fp8_pair<false>(codes[I], scale), fp8_pair<true>(codes[I], scale), fp8_pair<false>(codes[I + 1], scale),
               fp8_pair<true>(codes[I + 1], scale)};
}
__device__ __forceinline__ u32x4 expand8(u32x2 codes, float scale) {
  return u32x4{fp8_pair<false>(codes[0], scale), fp8_pair<true>(codes[0], scale), fp8_pair<false>(codes[1], scale),
               fp8_pair<true>(codes[1], scale)};
}
// o += V^T P^T for 16 dims and the 64 tokens of a wave's step: lane (n, gq) has the codes of dim n, the 16 tokens of tile
// gq, and that tile's scale.
__device__ __forceinline__ void add_values(f32x4 &o, u32x4 codes, float scale, const u32x4 (&p)[2]) {
  o = mfma16(expand8<0>(codes, scale), p[0], o);
  o = mfma16(expand8<2>(codes, scale), p[1], o);
}

}  // namespace nvamd
