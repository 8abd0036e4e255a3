// Device helpers that the attention kernels over the 4-bit cache share.
#pragma once

#include "fp4.h"

namespace nvamd {

constexpr float kNoScore = -3e38f;   // reference of an empty softmax: finite, so that it needs no guard in exponents
constexpr float kRescaleLog2 = 8.f;  // the reference moves when a score exceeds it by 2^8
constexpr u32 kBf16PairOne = 0x3F803F80u;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0,
                                                 0, 0);
}

// max / sum over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_over_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_xor32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_over_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum_xor32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// S += K . q for 16 rows of codes (128 dims) and 16 columns of e4m3, each block of 32 dims under its scale byte.  Lane
// (row or column n, gq) gives block gq of its row, dims 16 gq .. +15 and 64 + 16 gq .. +15 of its column, and the
// scales of block gq of either, the row's in byte B of a word (checked on gfx950).
template <int B>
__device__ __forceinline__ f32x4 mfma_fp4_fp8(u32x4 k, u32 k_scales, i32x8 q, u32 q_scale, f32x4 c) {
  const i32x8 codes = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(codes, q, c, 4, 0, B, (int)k_scales, 0, (int)q_scale);
}

// A block of 32 bf16 query values as hi + lo in e4m3 under 2^-s, s from its largest value, which lands in [128, 256).
// hi keeps 4 of the 8 significant bits and lo the rest: the sum is the value itself down to 2^-9 of the block's
// largest, and off by at most 2^-17 of the largest below.
struct QueryScale {
  float up;  // 2^s
  u32 byte;  // of 2^-s; 255, which makes every score NaN, for a block with an infinity or a NaN
};
__device__ __forceinline__ QueryScale query_scale(u32 top) {  // top: the largest value's bf16 bits, sign cleared
  const int e = min(max((int)(top >> 7), 20), 254);  // its biased exponent
  return {__uint_as_float((u32)(127 + 134 - e) << 23), top >= 0x7f80u ? 255u : (u32)(e - 7)};
}
__device__ __forceinline__ u32 largest(u32x4 x) {
  u32 top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const u32 w = x[e];
    top = max(top, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
  }
  return top;
}
// 4 values (two words of pairs) to a word of hi and one of lo.
__device__ __forceinline__ void split4(u32 w0, u32 w1, float up, int &hi, int &lo) {
  const float a = bf16_lo(w0) * up, b = bf16_hi(w0) * up, c = bf16_lo(w1) * up, d = bf16_hi(w1) * up;
  int h = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  h = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, h, true);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a - __builtin_amdgcn_cvt_f32_fp8(h, 0),
                                          b - __builtin_amdgcn_cvt_f32_fp8(h, 1), 0, false);
  hi = h;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(c - __builtin_amdgcn_cvt_f32_fp8(h, 2),
                                       d - __builtin_amdgcn_cvt_f32_fp8(h, 3), r, true);
}
// A lane's 32 values, in the order of the operand: 16 of one block, then 16 of another.
__device__ __forceinline__ void split32(const u32x4 (&x)[4], float up0, float up1, i32x8 &hi, i32x8 &lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int h, l;
      split4(x[j][2 * i], x[j][2 * i + 1], j < 2 ? up0 : up1, h, l);
      hi[2 * j + i] = h;
      lo[2 * j + i] = l;
    }
}

// The operand of mfma_fp4_fp8 from a row's dims 16 gq .. +15 and 64 + 16 gq .. +15; returns its scale byte.
__device__ __forceinline__ u32 query_operand(const u32x4 (&x)[4], int gq, i32x8 &hi, i32x8 &lo) {
  // Lanes gq and gq ^ 1 hold the halves of blocks gq / 2 and 2 + gq / 2.
  auto over_pair = [](u32 v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((u32)r[0], (u32)r[1]);
  };
  const QueryScale s0 = query_scale(over_pair(max(largest(x[0]), largest(x[1]))));
  const QueryScale s1 = query_scale(over_pair(max(largest(x[2]), largest(x[3]))));
  split32(x, s0.up, s1.up, hi, lo);
  // Lane gq gives block gq's: lanes 0 and 3 hold theirs, 1 and 2 take them from gq ^ 2.
  const u32 mine = gq < 2 ? s0.byte : s1.byte, give = gq < 2 ? s1.byte : s0.byte;
  const auto r = __builtin_amdgcn_permlane32_swap(give, give, false, false);
  return gq == 0 || gq == 3 ? mine : gq == 1 ? (u32)r[1] : (u32)r[0];
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

// Lanes of the banks in MASK (4 lanes each, of 16) take src moved by the DPP control, the others keep `old`.
template <int CTRL, int MASK>
__device__ __forceinline__ float dpp_into(float old, float src) {
  return __uint_as_float((u32)__builtin_amdgcn_update_dpp((int)__float_as_uint(old), (int)__float_as_uint(src), CTRL, 0xF,
                                                          MASK, false));
}
template <int CTRL>
__device__ __forceinline__ u32 dpp_u32(u32 v) {
  return (u32)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
constexpr int kRowShl4 = 0x104, kRowShl8 = 0x108, kRowShl12 = 0x10C;  // lane n <- lane n + 4, 8, 12 of its 16
constexpr int kRowShr4 = 0x114, kRowShr8 = 0x118, kRowShr12 = 0x11C;  // lane n <- lane n - 4, 8, 12
constexpr int kRowRor4 = 0x124;
constexpr int kRowBcast = 0x150;  // + n: every lane <- lane n of its 16

// Codes are read once: past the caches' normal keeping.
__device__ __forceinline__ u32x4 load16(const u8 *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
}

// Keeps the first n bytes (any n) of a word.
__device__ __forceinline__ u32 keep_bytes(u32 v, int n) {
  return n >= 4 ? v : n <= 0 ? 0u : v & ((1u << (8 * n)) - 1u);
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
