// A head vector in rows of the 4-bit cache: quantising, storing, and the norm and rotation before it, by 8 lanes; lane
// c holds dims 8c .. 8c + 7 and 64 + 8c .. 64 + 8c + 7.
#pragma once

#include "fp4.h"
#include "norm_rope64.h"

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

}  // namespace nvamd
