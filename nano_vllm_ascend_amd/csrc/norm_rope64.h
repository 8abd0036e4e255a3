// Per-head RMSNorm and rotate-half RoPE in 64 bits, for keys that are quantised afterwards; 8 lanes a row, lane c holds
// dims 8c .. 8c + 7 and 64 + 8c .. 64 + 8c + 7.
#pragma once

#include "common.h"

namespace nvamd {

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
// cos[d] + y[d] sin[d], in 64 bits with one rounding to bf16 at the end.  A code's step is a third to a half of the value
// in 4 bits (an eighth in 8), so a key that 32-bit arithmetic puts on the other side of a rounding border is that far off;
// in 64 bits the code is that of the exact value.  x w is exact in 64 bits (in 32 its bits would fit, its exponent not
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
