// Device helpers that the attention kernels over the 4-bit cache share.
#pragma once

#include "attention_tiles.h"
#include "fp4.h"

namespace nvamd {

// S += K . q for 16 rows of codes (128 dims) and 16 columns of e4m3, each block of 32 dims under its scale byte.  Lane
// (row or column n, gq) gives block gq of its row, dims 16 gq .. +15 and 64 + 16 gq .. +15 of its column, and the
// scales of block gq of either, the row's in byte B of a word (checked on gfx950).
template <int B>
__device__ __forceinline__ f32x4 mfma_fp4_fp8(u32x4 k, u32 k_scales, i32x8 q, u32 q_scale, f32x4 c) {
  const i32x8 codes = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes, q, c, 4, 0, B, (int)k_scales, 0, (int)q_scale);
}

template <int B>
__device__ __forceinline__ void score(f32x4 &s, u32x4 k, u32 k_scales, i32x8 q_hi, i32x8 q_lo, u32 q_scale) {
  s = mfma_fp4_fp8<B>(k, k_scales, q_hi, q_scale, f32x4{0.f, 0.f, 0.f, 0.f});
  s = mfma_fp4_fp8<B>(k, k_scales, q_lo, q_scale, s);
}

// Byte B of a word of scales as a float scale: one instruction (the compiler takes two for bytes 0..2).
template <int B>
__device__ __forceinline__ float scale_of(u32 word) {
  float r;
  if constexpr (B == 0)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0"
        : "=v"(r)
        : "v"(23), "v"(word));
  else if constexpr (B == 1)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1"
        : "=v"(r)
        : "v"(23), "v"(word));
  else if constexpr (B == 2)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2"
        : "=v"(r)
        : "v"(23), "v"(word));
  else
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3"
        : "=v"(r)
        : "v"(23), "v"(word));
  return r;
}

// The operands of V^T for 4 tokens (a word of codes) of a dim pair: bf16 pairs of tokens, of the first and of the
// second dim.
__device__ __forceinline__ void expand4(u32 codes, u32 scales, u32 &a01, u32 &a23, u32 &b01, u32 &b23) {
  const u32 v0 = fp4_pair<0>(codes, scale_of<0>(scales)), v1 = fp4_pair<1>(codes, scale_of<1>(scales));
  const u32 v2 = fp4_pair<2>(codes, scale_of<2>(scales)), v3 = fp4_pair<3>(codes, scale_of<3>(scales));
  a01 = pair_lo(v0, v1);
  a23 = pair_lo(v2, v3);
  b01 = pair_hi(v0, v1);
  b23 = pair_hi(v2, v3);
}

// o[2q], o[2q + 1] += V^T P^T for dims 32q .. 32q+31 and the 64 tokens of a wave's step (lane (n, gq): codes of dims
// 32q + n and 32q + 16 + n of the 16 tokens of tile gq, v_scales the scales of block n / 4, tokens 4 (n % 4) .. +3 of
// that tile).
template <int Q>
__device__ __forceinline__ void add_values(f32x4 (&o)[8], const u32x4 (&codes)[4], u32 v_scales, const u32x4 (&p)[2]) {
  const u32 sc[4] = {dpp_u32<kRowBcast + 4 * Q>(v_scales), dpp_u32<kRowBcast + 4 * Q + 1>(v_scales),
                     dpp_u32<kRowBcast + 4 * Q + 2>(v_scales), dpp_u32<kRowBcast + 4 * Q + 3>(v_scales)};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32 a[4], b[4];
    expand4(codes[Q][2 * h], sc[2 * h], a[0], a[1], b[0], b[1]);
    expand4(codes[Q][2 * h + 1], sc[2 * h + 1], a[2], a[3], b[2], b[3]);
    o[2 * Q] = mfma16(u32x4{a[0], a[1], a[2], a[3]}, p[h], o[2 * Q]);
    o[2 * Q + 1] = mfma16(u32x4{b[0], b[1], b[2], b[3]}, p[h], o[2 * Q + 1]);
  }
}

}  // namespace nvamd
