// Device helpers that the attention kernels over quantised caches share: products and exchanges over the 16 lanes of a
// tile, and the query as two e4m3 numbers per value.
#pragma once

#include "common.h"

namespace nvamd {

using u8 = uint8_t;

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

// The operand of a product of 16 x 16 x 128 from a row's dims 16 gq .. +15 and 64 + 16 gq .. +15; returns its scale byte.
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

}  // namespace nvamd
