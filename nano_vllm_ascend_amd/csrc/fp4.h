// The 4-bit KV cache's number format and page layout (nvamd.h, "KV cache held in 4 bits"), shared by the
// kernels that write and read it.
#pragma once

#include "common.h"

namespace nvamd {

using u8 = uint8_t;

constexpr int kFp4Block = 32;              // dims that share a scale
constexpr int kFp4RowBytes = kHeadDim / 2;  // codes of a head vector
constexpr int kFp4Scales = kHeadDim / kFp4Block;
constexpr int kFp4Tile = 16;                // tokens of a tile: the unit that a page's bytes are ordered in
constexpr int kFp4TileBytes = kFp4Tile * kFp4RowBytes;
constexpr int kFp4TileScales = kFp4Tile * kFp4Scales;
constexpr u32 kFp4Nan = 255;                // scale byte of a block that holds an infinity or a NaN

// Scale byte of a block whose largest |x| has the bf16 bits `amax` (sign cleared): the least e with
// max <= 7 * 2^e is the maximum's own exponent - 2, or one more where its fraction is past 1.75 = 7 / 4.  Within [2,
// 252], so that every value and its product with the largest code are normal, finite bf16 numbers.
__device__ __forceinline__ u32 fp4_scale_byte(u32 amax) {
  const int e = (int)(amax >> 7) - 2 + ((amax & 0x7f) > 0x60 ? 1 : 0);
  return amax >= 0x7f80u ? kFp4Nan : (u32)min(max(e, 2), 252);
}
__device__ __forceinline__ float fp4_scale(u32 byte) { return __uint_as_float(byte << 23); }

// The codes of 8 bf16 values at a scale (element 0 in the low nibble): v_cvt_scalef32_pk_fp4_bf16 rounds to nearest,
// ties to the even code, and saturates at 6 (checked on gfx950 over every bf16 value).
template <int B>
__device__ __forceinline__ u32 fp4_put_pair(u32 codes, u32 pair, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2v, pair), scale, B);
}
__device__ __forceinline__ u32 fp4_codes(u32x4 x, float scale) {
  u32 r = fp4_put_pair<0>(0u, x[0], scale);
  r = fp4_put_pair<1>(r, x[1], scale);
  r = fp4_put_pair<2>(r, x[2], scale);
  return fp4_put_pair<3>(r, x[3], scale);
}

// The two bf16 values of byte B of `codes` (low nibble first), exact: a code has two significant bits.  A scale of byte
// 255 gives NaN for every code, and one of byte 0 2^-127 (checked on gfx950 over all bytes and scales).
template <int B>
__device__ __forceinline__ u32 fp4_pair(u32 codes, float scale) {
  return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}
// All 8 values of a word of codes.
__device__ __forceinline__ u32x4 fp4_values(u32 codes, float scale) {
  return u32x4{fp4_pair<0>(codes, scale), fp4_pair<1>(codes, scale), fp4_pair<2>(codes, scale),
               fp4_pair<3>(codes, scale)};
}

// Index of the 16-token tile that holds a token of a page: tiles of a page's head follow one another.
__device__ __forceinline__ int64_t fp4_tile(int64_t block, int token, int head, int num_kv_heads, int bs_log2) {
  return (((block * num_kv_heads + head) << bs_log2) + token) >> 4;
}
// Byte of block q's scale of token t inside a tile's scales.
__device__ __forceinline__ int fp4_key_scale_at(int t, int q) { return (t & 3) * 16 + q * 4 + (t >> 2); }
__device__ __forceinline__ int fp4_value_scale_at(int t, int q) { return q * 16 + t; }

// One layer's pages.
struct Fp4Cache {
  u8 *k_codes;
  u8 *k_scales;
  u8 *v_codes;
  u8 *v_scales;
};

inline bool fp4_cache_ok(const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales) {
  return k_codes && k_scales && v_codes && v_scales && aligned16(k_codes) && aligned16(k_scales) &&
         aligned16(v_codes) && aligned16(v_scales);
}

}  // namespace nvamd
