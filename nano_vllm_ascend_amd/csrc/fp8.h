// The 8-bit KV cache's number format and page layout (nvamd.h, "KV cache held in 8 bits"), shared by the kernels that
// write and read it.
#pragma once

#include "common.h"

namespace nvamd {

using u8 = uint8_t;

constexpr int kFp8Tile = 16;  // tokens that share a scale: the unit that a page's bytes are ordered in
constexpr int kFp8TileBytes = kFp8Tile * kHeadDim;

// Scale byte of values whose largest |x| has the bf16 bits `amax` (sign cleared, finite): the least e with max <= 448 *
// 2^e = 1.75 * 2^(e + 8) is the maximum's own exponent - 8, or one more where its fraction is past 1.75.  Within [10,
// 246], so that every value is a normal, finite bf16 number (the largest maxima then saturate: clamp_to_codes).
constexpr int kFp8LeastScale = 10, kFp8MostScale = 246;
__device__ __forceinline__ u32 fp8_scale_byte(u32 amax) {
  const int e = (int)(amax >> 7) - 8 + ((amax & 0x7f) > 0x60 ? 1 : 0);
  return (u32)min(max(e, kFp8LeastScale), kFp8MostScale);
}
__device__ __forceinline__ float fp8_scale(u32 byte) { return __uint_as_float(byte << 23); }

typedef short s16x2 __attribute__((ext_vector_type(2)));
// The codes of a bf16 pair at a scale, in the low or high half of a word: v_cvt_scalef32_pk_fp8_bf16 rounds to nearest,
// ties to the even code, and gives the code 127 with the sign, NaN, for an infinity, a NaN and all that rounds past 448
// (checked on gfx950 over every bf16 value).
template <bool HIGH>
__device__ __forceinline__ u32 fp8_put_pair(u32 codes, u32 pair, float scale) {
  return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(s16x2, codes),
                                                                           __builtin_bit_cast(bf16x2v, pair), scale, HIGH));
}
// The two bf16 values of a half of a word, exact: a code has four significant bits.
template <bool HIGH>
__device__ __forceinline__ u32 fp8_pair(u32 codes, float scale) {
  return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

// Index of the 16-token tile that holds a token of a page: tiles of a page's head follow one another.
__device__ __forceinline__ int64_t fp8_tile(int64_t block, int token, int head, int num_kv_heads, int bs_log2) {
  return (((block * num_kv_heads + head) << bs_log2) + token) >> 4;
}
// Byte of dim d of token t of a tile.
__device__ __forceinline__ int fp8_key_at(int t, int d) { return (d >> 6) * (kFp8TileBytes / 2) + t * 64 + (d & 63); }
__device__ __forceinline__ int fp8_value_at(int t, int d) { return d * kFp8Tile + t; }

// One layer's pages.
struct Fp8Cache {
  u8 *k_codes;
  u8 *k_scales;
  u8 *v_codes;
  u8 *v_scales;
};

inline bool fp8_cache_ok(const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales) {
  return k_codes && k_scales && v_codes && v_scales && aligned16(k_codes) && aligned16(v_codes);
}

}  // namespace nvamd
