// The 4-bit paged KV cache: writing rows, reading rows back, and the per-head QK-RMSNorm + RoPE that
// writes them in the same pass (the 4-bit counterparts of kv_store.hip).
//
// Every kernel gives an aligned group of 8 lanes one head vector: lane c holds dims 8c..8c+7 and 64+8c..64+8c+7, so
// a block of 32 dims is the low (or high) half of 4 consecutive lanes, its maximum two DPP steps away, and RoPE
// needs no lane exchange.
#include "fp4.h"

namespace nvamd {
namespace {

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

// A byte of the values holds dims 32q + r and 32q + 16 + r: the two lanes of a quad that differ in bit 1 hold the two halves
// of a block, and exchange so that the one builds the bytes of the low block, the other those of the high one.
__device__ __forceinline__ void store_value(const Fp4Cache &cache, const Fp4Row &r, int c, u32x4 lo, u32x4 hi) {
  u32 s_lo, s_hi;
  const u32 w_lo = quantise8(lo, s_lo), w_hi = quantise8(hi, s_hi);
  const u32 o_lo = quad_xor2(w_lo), o_hi = quad_xor2(w_hi);
  const bool second = (c & 2) != 0;
  const u32 first16 = second ? o_hi : w_lo, last16 = second ? w_hi : o_lo;
  const int q = (second ? 2 : 0) + (c >> 2);
  u8 *p = cache.v_codes + r.tile * kFp4TileBytes + (16 * q + 8 * (c & 1)) * kFp4Tile + r.t;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    p[j * kFp4Tile] = (u8)(((first16 >> (4 * j)) & 15) | (((last16 >> (4 * j)) & 15) << 4));
  if ((c & 3) == 0) {
    u8 *s = cache.v_scales + r.tile * kFp4TileScales;
    s[fp4_value_scale_at(r.t, c >> 2)] = (u8)s_lo;
    s[fp4_value_scale_at(r.t, 2 + (c >> 2))] = (u8)s_hi;
  }
}

struct WriteArgs {
  const u16 *k;
  int64_t k_stride;
  const u16 *v;
  int64_t v_stride;
  Fp4Cache cache;
  const int64_t *slots;
  int64_t num_slots;
  int num_tokens;
  int num_kv_heads;
  int bs_log2;
  u32 *err;
};

// Vectors of a token: its key heads, then its value heads.
__global__ void __launch_bounds__(256)
kv_write_fp4_kernel(WriteArgs a) {
  const int vecs = 2 * a.num_kv_heads;
  const int64_t gv = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  if (gv >= (int64_t)a.num_tokens * vecs) return;  // whole 8-lane groups leave together
  const int t = (int)(gv / vecs);
  const int vec = (int)(gv % vecs);
  const int c = threadIdx.x & 7;
  const int64_t slot = a.slots[t];
  if (slot >= a.num_slots || slot < -1) {
    if (vec == 0 && c == 0) flag_index_error(a.err, NVAMD_ERR_SLOT);
    return;
  }
  if (slot < 0) return;  // -1: a padding row
  const bool is_k = vec < a.num_kv_heads;
  const int h = is_k ? vec : vec - a.num_kv_heads;
  const u16 *src = (is_k ? a.k + t * a.k_stride : a.v + t * a.v_stride) + h * kHeadDim + 8 * c;
  const u32x4 lo = ld16(src), hi = ld16(src + 64);
  const Fp4Row r = row_at(slot, h, a.num_kv_heads, a.bs_log2);
  if (is_k)
    store_key(a.cache, r, c, lo, hi);
  else
    store_value(a.cache, r, c, lo, hi);
}

struct ReadArgs {
  u16 *k;
  int64_t k_stride;
  u16 *v;
  int64_t v_stride;
  Fp4Cache cache;
  const int64_t *slots;
  int64_t num_slots;
  int num_tokens;
  int num_kv_heads;
  int bs_log2;
  u32 *err;
};

// As the write, the other way round; a row without a slot, or with one outside the cache, is zeros.
__global__ void __launch_bounds__(256)
kv_read_fp4_kernel(ReadArgs a) {
  const int vecs = 2 * a.num_kv_heads;
  const int64_t gv = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  if (gv >= (int64_t)a.num_tokens * vecs) return;
  const int t = (int)(gv / vecs);
  const int vec = (int)(gv % vecs);
  const int c = threadIdx.x & 7;
  const int64_t slot = a.slots[t];
  const bool bad = slot >= a.num_slots || slot < -1;
  if (bad && vec == 0 && c == 0) flag_index_error(a.err, NVAMD_ERR_SLOT);
  const bool live = !bad && slot >= 0;
  const bool is_k = vec < a.num_kv_heads;
  const int h = is_k ? vec : vec - a.num_kv_heads;
  const Fp4Row r = row_at(live ? slot : 0, h, a.num_kv_heads, a.bs_log2);
  const u32x4 zero = {0u, 0u, 0u, 0u};
  if (is_k) {
    u32x4 lo = zero, hi = zero;
    if (live) {
      const u32 *row = reinterpret_cast<const u32 *>(a.cache.k_codes + r.tile * kFp4TileBytes + r.t * kFp4RowBytes);
      const u8 *s = a.cache.k_scales + r.tile * kFp4TileScales;
      lo = fp4_values(row[c], fp4_scale(s[fp4_key_scale_at(r.t, c >> 2)]));
      hi = fp4_values(row[8 + c], fp4_scale(s[fp4_key_scale_at(r.t, 2 + (c >> 2))]));
    }
    u16 *dst = a.k + t * a.k_stride + h * kHeadDim + 8 * c;
    st16(dst, lo);
    st16(dst + 64, hi);
  } else {
    // lane c: bytes 8(c % 2) .. +7 of block c / 2, dims 8(c % 2) + j of the block's first and of its second half
    u32x4 first = zero, last = zero;
    if (live) {
      const u8 *p = a.cache.v_codes + r.tile * kFp4TileBytes + (16 * (c >> 1) + 8 * (c & 1)) * kFp4Tile + r.t;
      const float scale = fp4_scale(a.cache.v_scales[r.tile * kFp4TileScales + fp4_value_scale_at(r.t, c >> 1)]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32 x = fp4_pair<0>(p[2 * j * kFp4Tile], scale), y = fp4_pair<0>(p[(2 * j + 1) * kFp4Tile], scale);
        first[j] = pair_lo(x, y);
        last[j] = pair_hi(x, y);
      }
    }
    u16 *dst = a.v + t * a.v_stride + h * kHeadDim + 32 * (c >> 1) + 8 * (c & 1);
    st16(dst, first);
    st16(dst + 16, last);
  }
}

struct NormRopeFp4Args {
  u16 *q_out;
  int64_t q_out_stride;
  u16 *k_out;  // or null
  int64_t k_out_stride;
  const u16 *q;
  int64_t q_stride;
  const u16 *q_w;
  const u16 *k_w;
  const int64_t *positions;
  const float *cos_sin;
  int max_positions;
  int num_heads;
  float eps;
  WriteArgs w;
};

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

// y = x * rsqrt(mean(x^2) + eps) * w, then the rotation out[d] = y[d] cos[d] - y[d+64] sin[d], out[d+64] = y[d+64]
// cos[d] + y[d] sin[d], in 64 bits with one rounding to bf16 at the end.  A 4-bit code's step is a
// third to a half of the value, so a key that 32-bit arithmetic puts on the other side of a rounding border is that far off;
// in 64 bits the code is that of the exact value.  The fp64 units keep up with the stream.
__device__ __forceinline__ void norm_rope_f64(u32x4 &lo, u32x4 &hi, const u32x4 w_lo, const u32x4 w_hi,
                                              const float *table_row, int c, float eps) {
  double x[16];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = bf16_lo(lo[e]);
    x[2 * e + 1] = bf16_hi(lo[e]);
    x[8 + 2 * e] = bf16_lo(hi[e]);
    x[8 + 2 * e + 1] = bf16_hi(hi[e]);
  }
  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
  const double rstd = rsqrt(dpp_sum8(ss) * (1.0 / kHeadDim) + (double)eps);
  const f32x4 c0 = *reinterpret_cast<const f32x4 *>(table_row + 8 * c);
  const f32x4 c1 = *reinterpret_cast<const f32x4 *>(table_row + 8 * c + 4);
  const f32x4 s0 = *reinterpret_cast<const f32x4 *>(table_row + 64 + 8 * c);
  const f32x4 s1 = *reinterpret_cast<const f32x4 *>(table_row + 64 + 8 * c + 4);
  float r_lo[8], r_hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const u32 wl = w_lo[e >> 1], wh = w_hi[e >> 1];
    const double y_lo = x[e] * rstd * (double)((e & 1) ? bf16_hi(wl) : bf16_lo(wl));
    const double y_hi = x[8 + e] * rstd * (double)((e & 1) ? bf16_hi(wh) : bf16_lo(wh));
    const double cs = e < 4 ? c0[e & 3] : c1[e & 3], sn = e < 4 ? s0[e & 3] : s1[e & 3];
    r_lo[e] = (float)(y_lo * cs - y_hi * sn);
    r_hi[e] = (float)(y_hi * cs + y_lo * sn);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    lo[e] = pack_bf16x2(r_lo[2 * e], r_lo[2 * e + 1]);
    hi[e] = pack_bf16x2(r_hi[2 * e], r_hi[2 * e + 1]);
  }
}

// Vectors of a token: its query heads, its key heads, its value heads.
__global__ void __launch_bounds__(256)
qk_norm_rope_fp4_kernel(NormRopeFp4Args a) {
  const int hkv = a.w.num_kv_heads;
  const int vecs = a.num_heads + 2 * hkv;
  const int64_t gv = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  if (gv >= (int64_t)a.w.num_tokens * vecs) return;
  const int t = (int)(gv / vecs);
  const int vec = (int)(gv % vecs);
  const int c = threadIdx.x & 7;
  int64_t slot = a.w.slots[t];
  if (slot >= a.w.num_slots || slot < -1) {
    if (vec == 0 && c == 0) flag_index_error(a.w.err, NVAMD_ERR_SLOT);
    slot = -1;
  }
  if (vec >= a.num_heads + hkv) {
    if (slot < 0) return;
    const int h = vec - a.num_heads - hkv;
    const u16 *src = a.w.v + t * a.w.v_stride + h * kHeadDim + 8 * c;
    store_value(a.w.cache, row_at(slot, h, hkv, a.w.bs_log2), c, ld16(src), ld16(src + 64));
    return;
  }
  const bool is_q = vec < a.num_heads;
  const int h = is_q ? vec : vec - a.num_heads;
  if (!is_q && slot < 0 && a.k_out == nullptr) return;
  const u16 *src = (is_q ? a.q + t * a.q_stride : a.w.k + t * a.w.k_stride) + h * kHeadDim + 8 * c;
  const u16 *wt = (is_q ? a.q_w : a.k_w) + 8 * c;
  u32x4 lo = ld16(src), hi = ld16(src + 64);
  const u32x4 w_lo = ld16(wt), w_hi = ld16(wt + 64);
  int64_t pos = a.positions[t];
  if (pos < 0 || pos >= a.max_positions) {
    if (vec == 0 && c == 0) flag_index_error(a.w.err, NVAMD_ERR_POSITION);
    pos = pos < 0 ? 0 : a.max_positions - 1;
  }
  norm_rope_f64(lo, hi, w_lo, w_hi, a.cos_sin + pos * kHeadDim, c, a.eps);
  u16 *dst = is_q ? a.q_out + t * a.q_out_stride : a.k_out ? a.k_out + t * a.k_out_stride : nullptr;
  if (dst != nullptr) {
    st16(dst + h * kHeadDim + 8 * c, lo);
    st16(dst + h * kHeadDim + 8 * c + 64, hi);
  }
  if (!is_q && slot >= 0) store_key(a.w.cache, row_at(slot, h, hkv, a.w.bs_log2), c, lo, hi);
}

bool rows_ok(const void *p, int64_t stride, int heads) {
  return p && aligned16(p) && stride % 8 == 0 && stride >= (int64_t)heads * kHeadDim;
}

int vector_blocks(int64_t vectors, unsigned *blocks) {
  const int64_t n = (vectors + 31) / 32;
  if (n > 0x7fffffff) return NVAMD_EINVAL;
  *blocks = (unsigned)n;
  return NVAMD_OK;
}

// Checks shared by the entry points; fills what they share.
int fill_write_args(WriteArgs &w, const void *k, int64_t k_stride, const void *v, int64_t v_stride, void *k_codes,
                    void *k_scales, void *v_codes, void *v_scales, const int64_t *slots, int num_tokens,
                    int num_kv_heads, int head_dim, int num_blocks, int block_size) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0) return NVAMD_EINVAL;
  if (head_dim != kHeadDim) return NVAMD_EUNSUPPORTED;
  const int bs_log2 = log2_exact(block_size);
  if (bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!rows_ok(k, k_stride, num_kv_heads) || !rows_ok(v, v_stride, num_kv_heads) ||
      !fp4_cache_ok(k_codes, k_scales, v_codes, v_scales) || !slots)
    return NVAMD_EINVAL;
  w = WriteArgs{};
  w.k = static_cast<const u16 *>(k);
  w.k_stride = k_stride;
  w.v = static_cast<const u16 *>(v);
  w.v_stride = v_stride;
  w.cache = Fp4Cache{static_cast<u8 *>(k_codes), static_cast<u8 *>(k_scales), static_cast<u8 *>(v_codes),
                     static_cast<u8 *>(v_scales)};
  w.slots = slots;
  w.num_slots = (int64_t)num_blocks << bs_log2;
  w.num_tokens = num_tokens;
  w.num_kv_heads = num_kv_heads;
  w.bs_log2 = bs_log2;
  w.err = index_error_word();
  return NVAMD_OK;
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" int nvamd_kv_cache_write_fp4(const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                                        void *k_codes, void *k_scales, void *v_codes, void *v_scales, int num_blocks,
                                        int block_size, const int64_t *slot_mapping, int num_tokens, int num_kv_heads,
                                        int head_dim, hipStream_t stream) {
  if (num_tokens == 0) return NVAMD_OK;
  WriteArgs w;
  const int st = fill_write_args(w, k, k_stride, v, v_stride, k_codes, k_scales, v_codes, v_scales, slot_mapping,
                                 num_tokens, num_kv_heads, head_dim, num_blocks, block_size);
  if (st != NVAMD_OK) return st;
  unsigned blocks;
  if (vector_blocks((int64_t)num_tokens * 2 * num_kv_heads, &blocks) != NVAMD_OK) return NVAMD_EINVAL;
  hipLaunchKernelGGL(kv_write_fp4_kernel, dim3(blocks), dim3(256), 0, stream, w);
  return launch_status();
}

extern "C" int nvamd_kv_cache_read_fp4(void *k, int64_t k_stride, void *v, int64_t v_stride, const void *k_codes,
                                       const void *k_scales, const void *v_codes, const void *v_scales,
                                       int num_blocks, int block_size, const int64_t *slot_mapping, int num_tokens,
                                       int num_kv_heads, int head_dim, hipStream_t stream) {
  if (num_tokens == 0) return NVAMD_OK;
  WriteArgs w;
  const int st = fill_write_args(w, k, k_stride, v, v_stride, const_cast<void *>(k_codes), const_cast<void *>(k_scales),
                                 const_cast<void *>(v_codes), const_cast<void *>(v_scales), slot_mapping, num_tokens,
                                 num_kv_heads, head_dim, num_blocks, block_size);
  if (st != NVAMD_OK) return st;
  unsigned blocks;
  if (vector_blocks((int64_t)num_tokens * 2 * num_kv_heads, &blocks) != NVAMD_OK) return NVAMD_EINVAL;
  ReadArgs a{static_cast<u16 *>(k), k_stride, static_cast<u16 *>(v), v_stride, w.cache, w.slots, w.num_slots,
             num_tokens, num_kv_heads, w.bs_log2, w.err};
  hipLaunchKernelGGL(kv_read_fp4_kernel, dim3(blocks), dim3(256), 0, stream, a);
  return launch_status();
}

extern "C" int nvamd_qk_norm_rope_fp4(void *q_out, int64_t q_out_stride, void *k_out, int64_t k_out_stride,
                                      const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v,
                                      int64_t v_stride, const void *q_weight, const void *k_weight,
                                      const int64_t *positions, const float *cos_sin, int max_positions,
                                      void *k_codes, void *k_scales, void *v_codes, void *v_scales, int num_blocks,
                                      int block_size, const int64_t *slot_mapping, int num_tokens, int num_heads,
                                      int num_kv_heads, int head_dim, float eps, hipStream_t stream) {
  if (num_tokens == 0) return NVAMD_OK;
  NormRopeFp4Args a = {};
  const int st = fill_write_args(a.w, k, k_stride, v, v_stride, k_codes, k_scales, v_codes, v_scales, slot_mapping,
                                 num_tokens, num_kv_heads, head_dim, num_blocks, block_size);
  if (st != NVAMD_OK) return st;
  if (num_heads <= 0 || max_positions <= 0 || !q_weight || !k_weight || !positions || !cos_sin ||
      !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(cos_sin) || !rows_ok(q, q_stride, num_heads) ||
      !rows_ok(q_out, q_out_stride, num_heads) || (k_out && !rows_ok(k_out, k_out_stride, num_kv_heads)))
    return NVAMD_EINVAL;
  a.q_out = static_cast<u16 *>(q_out);
  a.q_out_stride = q_out_stride;
  a.k_out = static_cast<u16 *>(k_out);
  a.k_out_stride = k_out_stride;
  a.q = static_cast<const u16 *>(q);
  a.q_stride = q_stride;
  a.q_w = static_cast<const u16 *>(q_weight);
  a.k_w = static_cast<const u16 *>(k_weight);
  a.positions = positions;
  a.cos_sin = cos_sin;
  a.max_positions = max_positions;
  a.num_heads = num_heads;
  a.eps = eps;
  unsigned blocks;
  if (vector_blocks((int64_t)num_tokens * (num_heads + 2 * num_kv_heads), &blocks) != NVAMD_OK) return NVAMD_EINVAL;
  hipLaunchKernelGGL(qk_norm_rope_fp4_kernel, dim3(blocks), dim3(256), 0, stream, a);
  return launch_status();
}
