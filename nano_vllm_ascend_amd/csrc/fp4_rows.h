// A head vector in rows of the 4-bit cache: quantising, storing, and the norm and rotation before it, by 8 lanes; lane
// c holds dims 8c .. 8c + 7 and 64 + 8c .. 64 + 8c + 7.
#pragma once

#include "fp4.h"

namespace nvamd {

// max over the 4 lanes of an aligned quad, of non-negative integers
__device__ __forceinline__ u32 quad_max(u32 v) {
  v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, kDppQuadXor1, 0xF, 0xF, true));
  v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, kDppQuadXor2, 0xF, 0xF, true));
  return v;
}
__device__ __forceinline__ u32 quad_xor2(u32 v) {
  return (u32)__builtin_amdgcn_mov_dpp((int)v, kDppQuadXor2, 0xF, 0xF, true);
}

// Scale byte and codes of a lane's 8 values of a block that a quad shares.
__device__ __forceinline__ u32 quantise8(u32x4 x, u32 &scale) {
  u32 m = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = max(m, max(x[e] & 0x7fffu, (x[e] >> 16) & 0x7fffu));
  scale = fp4_scale_byte(quad_max(m));
  return scale == kFp4Nan ? 0u : fp4_codes(x, fp4_scale(scale));
}

struct Fp4Row {
  int64_t tile;  // 16-token tile of the row's page and head
  int t;         // token of the tile
};

__device__ __forceinline__ Fp4Row row_at(int64_t slot, int head, int num_kv_heads, int bs_log2) {
  const int64_t block = slot >> bs_log2;
  const int token = (int)(slot & ((1 << bs_log2) - 1));
  return {fp4_tile(block, token, head, num_kv_heads, bs_log2), token & 15};
}

// lo / hi: dims 8c.. and 64 + 8c.. of the row, c = lane of the 8.
__device__ __forceinline__ void store_key(const Fp4Cache &cache, const Fp4Row &r, int c, u32x4 lo, u32x4 hi) {
  u32 s_lo, s_hi;
  const u32 w_lo = quantise8(lo, s_lo), w_hi = quantise8(hi, s_hi);
  u32 *row = reinterpret_cast<u32 *>(cache.k_codes + r.tile * kFp4TileBytes + r.t * kFp4RowBytes);
  row[c] = w_lo;
  row[8 + c] = w_hi;
  if ((c & 3) == 0) {
    u8 *s = cache.k_scales + r.tile * kFp4TileScales;
    s[fp4_key_scale_at(r.t, c >> 2)] = (u8)s_lo;
    s[fp4_key_scale_at(r.t, 2 + (c >> 2))] = (u8)s_hi;
  }
}

// A byte of the values holds dims 32q + r and 32q + 16 + r: the two lanes of a quad that differ in bit 1 hold the two
// halves of a block, and exchange so that the one builds the bytes of the low block, the other those of the high one.
// The bytes go to `tile` in LDS, [64 bytes of a row][8 tokens], at token `tok`.
__device__ __forceinline__ void value_bytes(const Fp4Cache &cache, const Fp4Row &r, bool live, int c, int tok, u32x4 lo,
                                            u32x4 hi, u8 *tile) {
  u32 s_lo, s_hi;
  const u32 w_lo = quantise8(lo, s_lo), w_hi = quantise8(hi, s_hi);
  const u32 o_lo = quad_xor2(w_lo), o_hi = quad_xor2(w_hi);
  const bool second = (c & 2) != 0;
  const u32 first16 = second ? o_hi : w_lo, last16 = second ? w_hi : o_lo;
  // bytes j of even and of odd nibbles: (low nibble of the first half, low nibble of the second)
  const u32 even = (first16 & 0x0f0f0f0fu) | ((last16 & 0x0f0f0f0fu) << 4);
  const u32 odd = ((first16 >> 4) & 0x0f0f0f0fu) | (last16 & 0xf0f0f0f0u);
  const int q = (second ? 2 : 0) + (c >> 2);
  u8 *p = tile + (16 * q + 8 * (c & 1)) * 8 + tok;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    p[(2 * j) * 8] = (u8)(even >> (8 * j));
    p[(2 * j + 1) * 8] = (u8)(odd >> (8 * j));
  }
  if (live && (c & 3) == 0) {
    u8 *s = cache.v_scales + r.tile * kFp4TileScales;
    s[fp4_value_scale_at(r.t, c >> 2)] = (u8)s_lo;
    s[fp4_value_scale_at(r.t, 2 + (c >> 2))] = (u8)s_hi;
  }
}

// A wave's own LDS writes before its own reads: LDS serves a wave in order, so only the compiler has to keep it.
__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

__device__ __forceinline__ double dpp_add(double v, int lo, int hi) {
  return v + __builtin_bit_cast(double, ((uint64_t)(u32)hi << 32) | (u32)lo);
}
template <int CTRL>
__device__ __forceinline__ double dpp_sum(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return dpp_add(v, __builtin_amdgcn_mov_dpp((int)(u32)b, CTRL, 0xF, 0xF, true),
                 __builtin_amdgcn_mov_dpp((int)(u32)(b >> 32), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ double dpp_sum8(double v) {
  return dpp_sum<kDppHalfMirror>(dpp_sum<kDppQuadXor2>(dpp_sum<kDppQuadXor1>(v)));
}

// A 32-bit value that rounds to bf16 as x does.  A plain cast rounds too, and may land on a border of bf16 that x is
// only close to; here all but the top 20 bits of the fraction are cut off, and the last of these is set if any of the
// rest was.  (From 2^-129 on; below that the cast rounds at 2^-149, 2^-16 of bf16's step there.)
__device__ __forceinline__ float bf16_bound(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint64_t top = (uint64_t)((u32)(b >> 32) | ((u32)b != 0u ? 1u : 0u)) << 32;
  return (float)__builtin_bit_cast(double, top);
}

// A lane's part of a row's sum of squares.
__device__ __forceinline__ double sum_squares(u32x4 lo, u32x4 hi) {
  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double x0 = bf16_lo(lo[e]), x1 = bf16_hi(lo[e]), x2 = bf16_lo(hi[e]), x3 = bf16_hi(hi[e]);
    ss += x0 * x0;
    ss += x1 * x1;
    ss += x2 * x2;
    ss += x3 * x3;
  }
  return ss;
}
__device__ __forceinline__ double norm_factor(double squares, double eps) {
  return rsqrt(squares * (1.0 / kHeadDim) + eps);
}

// y = x * rsqrt(mean(x^2) + eps) * w, then the rotation out[d] = y[d] cos[d] - y[d+64] sin[d], out[d+64] = y[d+64]
// cos[d] + y[d] sin[d], in 64 bits with one rounding to bf16 at the end.  A 4-bit code's step is a
// third to a half of the value, so a key that 32-bit arithmetic puts on the other side of a rounding border is that far
// off; in 64 bits the code is that of the exact value.  x w is exact in 64 bits (in 32 its bits would fit, its exponent not
// always), and the reciprocal root comes last: one multiplication for each result.
__device__ __forceinline__ void norm_rope_f64(u32x4 &lo, u32x4 &hi, const u32x4 w_lo, const u32x4 w_hi,
                                              const float (&cs)[8], const float (&sn)[8], double rstd) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float r_lo[2], r_hi[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double x_lo = i ? bf16_hi(lo[e]) : bf16_lo(lo[e]), x_hi = i ? bf16_hi(hi[e]) : bf16_lo(hi[e]);
      const double y_lo = x_lo * (i ? bf16_hi(w_lo[e]) : bf16_lo(w_lo[e]));
      const double y_hi = x_hi * (i ? bf16_hi(w_hi[e]) : bf16_lo(w_hi[e]));
      const double c = cs[2 * e + i], s = sn[2 * e + i];
      r_lo[i] = bf16_bound((y_lo * c - y_hi * s) * rstd);
      r_hi[i] = bf16_bound((y_hi * c + y_lo * s) * rstd);
    }
    lo[e] = pack_bf16x2(r_lo[0], r_lo[1]);
    hi[e] = pack_bf16x2(r_hi[0], r_hi[1]);
  }
}

}  // namespace nvamd
