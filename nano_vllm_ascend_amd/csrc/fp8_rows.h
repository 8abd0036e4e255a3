// Rows that go into tiles of the 8-bit cache: a wave writes tokens o .. o + n - 1 of one head's tile.
//
// Their largest finite |x| gives a scale.  Rows that begin a tile (o = 0) set it; others raise the tile's to theirs if
// that is larger, and the codes of the other 16 - n tokens are then rounded to the new scale.  (The step from one power
// of two to another moves a code's exponent; only what falls below 2^-6 of the scale loses bits.)  So a tile is filled
// from its first token on, in any number of calls, and holds the same values but for those bits.
#pragma once

#include "fp8.h"

namespace nvamd {

__device__ __forceinline__ u32 wave_max_u32(u32 v) {
  v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, kDppQuadXor1, 0xF, 0xF, true));
  v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, kDppQuadXor2, 0xF, 0xF, true));
  v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, kDppHalfMirror, 0xF, 0xF, true));
  v = max(v, (u32)__builtin_amdgcn_mov_dpp((int)v, kDppMirror, 0xF, 0xF, true));
  const u32 a = (u32)__builtin_amdgcn_readlane((int)v, 0), b = (u32)__builtin_amdgcn_readlane((int)v, 16);
  const u32 c = (u32)__builtin_amdgcn_readlane((int)v, 32), d = (u32)__builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}

// The largest |x| of N words of bf16 pairs over the wave, as bits; infinities and NaNs do not count.
template <int N>
__device__ __forceinline__ u32 largest_finite(const u32 (&x)[N]) {
  u32 top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
  top = wave_max_u32(top);
  if (__builtin_expect(top >= 0x7f80u, 0)) {
    top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u32 a = x[i] & 0x7fffu, b = (x[i] >> 16) & 0x7fffu;
      top = max(top, max(a >= 0x7f80u ? 0u : a, b >= 0x7f80u ? 0u : b));
    }
    top = wave_max_u32(top);
  }
  return top;
}

// Maxima past 448 * 2^119 saturate there (the conversion would make them NaN).
__device__ __forceinline__ u32 clamp_half(u32 x) {
  const u32 a = x & 0x7fffu;
  return a > 0x7f60u && a < 0x7f80u ? (x & 0x8000u) | 0x7f60u : x;
}
template <int N>
__device__ __forceinline__ void clamp_to_codes(u32 (&x)[N], u32 byte) {
  if (__builtin_expect(byte != (u32)kFp8MostScale, 1)) return;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = clamp_half(x[i] & 0xffffu) | clamp_half(x[i] >> 16) << 16;
}

// Codes under a scale, under another that is 2^up times as large.
__device__ __forceinline__ u32 raise_codes(u32 codes, float up) {
  u32 r = fp8_put_pair<false>(0u, fp8_pair<false>(codes, 1.f), up);
  return fp8_put_pair<true>(r, fp8_pair<true>(codes, 1.f), up);
}
__device__ __forceinline__ float raise_factor(u32 from, u32 to) {  // 2^(to - from), or as much as makes every code 0
  return __uint_as_float((127u + min(to - from, 100u)) << 23);
}

// Keys.  Lane (tok, c), 8 lanes a token: x[p] holds token 8 p + tok, dims 8c .. 8c + 7, then 64 + 8c .. (zeros where that
// is none of the tokens written).  `held`: the tile's scale byte, where o > 0.
__device__ __forceinline__ void store_keys(const Fp8Cache &cache, int64_t tile, int o, int n, u32 held, int tok, int c,
                                           u32 (&x)[16]) {
  u32 byte = fp8_scale_byte(largest_finite(x));
  if (o > 0) byte = max(byte, held);
  clamp_to_codes(x, byte);
  const float scale = fp8_scale(byte);
  u8 *base = cache.k_codes + tile * kFp8TileBytes + 8 * c;
  const bool raise = o > 0 && byte != held;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int t = 8 * p + tok;
    u32x2 *lo = reinterpret_cast<u32x2 *>(base + fp8_key_at(t, 0)), *hi = reinterpret_cast<u32x2 *>(base + fp8_key_at(t, 64));
    if (t >= o && t < o + n) {
      u32 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = fp8_put_pair<true>(fp8_put_pair<false>(0u, x[8 * p + 2 * i], scale), x[8 * p + 2 * i + 1], scale);
      *lo = u32x2{w[0], w[1]};
      *hi = u32x2{w[2], w[3]};
    } else if (raise) {
      const float up = raise_factor(held, byte);
      const u32x2 a = *lo, b = *hi;
      *lo = u32x2{raise_codes(a[0], up), raise_codes(a[1], up)};
      *hi = u32x2{raise_codes(b[0], up), raise_codes(b[1], up)};
    }
  }
  if (tok == 0 && c == 0 && (o == 0 || raise)) cache.k_scales[tile] = (u8)byte;
}

// Values.  Lane l: x[t] holds dims 2l, 2l + 1 of token t (zeros where that is none of the tokens written); old: the 32
// bytes of its two dims that the tile holds, where o > 0.  Tokens behind rows that begin a tile become zeros.
__device__ __forceinline__ void store_values(const Fp8Cache &cache, int64_t tile, int o, int n, u32 held,
                                             u32x4 (&old)[2], int lane, u32 (&x)[16]) {
  u32 byte = fp8_scale_byte(largest_finite(x));
  if (o > 0) byte = max(byte, held);
  clamp_to_codes(x, byte);
  const float scale = fp8_scale(byte);
  const bool raise = o > 0 && byte != held;
  u32x4 *dst = reinterpret_cast<u32x4 *>(cache.v_codes + tile * kFp8TileBytes + 2 * lane * kFp8Tile);
  if (raise) {
    const float up = raise_factor(held, byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      old[0][i] = raise_codes(old[0][i], up);
      old[1][i] = raise_codes(old[1][i], up);
    }
  }
  // bytes of the tokens written, as masks of the four words
  const u32 tokens = ((1u << n) - 1u) << o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 a = fp8_put_pair<true>(fp8_put_pair<false>(0u, x[4 * i], scale), x[4 * i + 1], scale);
    const u32 b = fp8_put_pair<true>(fp8_put_pair<false>(0u, x[4 * i + 2], scale), x[4 * i + 3], scale);
    const u32 bits = tokens >> (4 * i) & 15u;
    const u32 mask = ((bits & 1u) | (bits & 2u) << 7 | (bits & 4u) << 14 | (bits & 8u) << 21) * 0xffu;
    old[0][i] = (old[0][i] & ~mask) | (__builtin_amdgcn_perm(b, a, 0x06040200u) & mask);
    old[1][i] = (old[1][i] & ~mask) | (__builtin_amdgcn_perm(b, a, 0x07050301u) & mask);
  }
  dst[0] = old[0];
  dst[1] = old[1];
  if (lane == 0 && (o == 0 || raise)) cache.v_scales[tile] = (u8)byte;
}

}  // namespace nvamd
