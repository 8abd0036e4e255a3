// The 4-bit paged KV cache: writing rows, reading rows back, and the per-head QK-RMSNorm + RoPE that
// writes them in the same pass (the 4-bit counterparts of kv_store.hip).
//
// A wave takes 8 consecutive tokens, an aligned group of 8 lanes each, and one head or a run of them: rows of a head
// that follow one another in a page are written together, and the 8 tokens of a head's values meet in LDS so that bytes
// of consecutive tokens leave as one store.  Of a head vector, lane c of a group holds dims 8c..8c+7 and
// 64+8c..64+8c+7: a block of 32 dims is the low (or high) half of 4 consecutive lanes, its maximum two DPP steps away,
// and RoPE needs no lane exchange.
//
// All three are bound by memory: per head vector 256 bytes of bf16 and 68 of the cache, once.  36,488 tokens, 8 kv
// heads (and 16 query heads): write 189 MB in 37 us (5.2 TB/s), read 189 MB in 34 us (5.6 TB/s), norm + RoPE + write
// with the keys returned 564 MB in 117 us (4.8 TB/s); a large copy reaches 5.0 TB/s.  One token: 3 us, the launch.
#include "fp4_rows.h"

namespace nvamd {
namespace {

// A 64-bit value of one lane, as a scalar.
__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const u32 lo = (u32)__builtin_amdgcn_readlane((int)(u32)v, lane);
  const u32 hi = (u32)__builtin_amdgcn_readlane((int)(u32)((uint64_t)v >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t uniform64(int64_t v) { return lane_value(v, 0); }

// The 8 tokens' bytes of row byte `lane` to their slots.  Where the slots follow one another the bytes are turned to
// their places in 8-byte half rows: one store if they fill one, else those of each side of the border, words where
// whole.
__device__ __forceinline__ void store_values(const Fp4Cache &cache, const u8 *tile, int64_t slot, bool run, int head,
                                             int num_kv_heads, int bs_log2, int lane) {
  auto place = [&](int64_t s) {  // of the byte of slot s
    const Fp4Row r = row_at(s, head, num_kv_heads, bs_log2);
    return cache.v_codes + r.tile * kFp4TileBytes + lane * kFp4Tile + r.t;
  };
  const u32x2 w = *reinterpret_cast<const u32x2 *>(tile + lane * 8);
  if (run) {
    const int64_t s0 = uniform64(slot);
    const int o = (int)(s0 & 7);
    if (o == 0) {
      *reinterpret_cast<u32x2 *>(place(s0)) = w;
      return;
    }
    const uint64_t x = ((uint64_t)w[1] << 32) | w[0];
    const uint64_t y = (x << (8 * o)) | (x >> (64 - 8 * o));  // byte i: the token of slot i mod 8
    u8 *before = place(s0) - o, *after = place(s0 + 8 - o);   // the half rows that the run ends and begins
    const int border = o >> 2;                                // the word that holds bytes of both, if o % 4
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const u32 v = (u32)(y >> (32 * k));
      if (k != border || (o & 3) == 0) {
        *reinterpret_cast<u32 *>((4 * k >= o ? before : after) + 4 * k) = v;
      } else {
#pragma unroll
        for (int i = 4 * k; i < 4 * k + 4; ++i) (i >= o ? before : after)[i] = (u8)(v >> (8 * (i & 3)));
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t s = lane_value(slot, 8 * i);
    if (s >= 0) *place(s) = (u8)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// Rows too many for the caches until their next use go past them (32 MB a tensor: half of the 256 MB Infinity Cache for
// two tensors in and out).  36,488 x 8 heads, plain / nontemporal: written 43.8 / 39.2 us, read 46.5 / 38.2; 12,345 x 8
// heads written and read back 27.6 / 31.9.
constexpr int64_t kStreamElems = 16 << 20;
template <bool STREAM>
__device__ __forceinline__ void put16(u16 *p, u32x4 v) {
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(p));
  else
    st16(p, v);
}
template <bool STREAM>
__device__ __forceinline__ u32x4 get16(const u16 *p) {
  if constexpr (STREAM) return ld16_stream(p);
  else return ld16(p);
}

// Heads that a wave of the rotation takes one after another: the table's row, the weights and the slots are read once
// for them.  Fewer where that leaves less than four waves for each SIMD of 256 CUs.  (36,488 tokens: 118 us with 8 or
// 4, 142 with 2.) Without the rotation a wave has one head (8: 42.2 us, 1: 40.1; 12,345 tokens 17.6, 16.7).
constexpr int kRopeHeads = 8;
constexpr int kWantedWaves = 4096;

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
  int heads_per_wave;
  u32 *err;
};

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

// The other way round.  A wave takes one key or value head of 8 tokens: it waits for its loads once, and more waves are
// all that hides that (36,488 x 8 heads: 50 us with 8 heads one after another, 45 with 2, 37.4 so; 34 since the scale
// loads with the bytes).  A row without a
// slot, or with one outside the cache, is zeros.
template <bool STREAM>
__global__ void __launch_bounds__(256)
kv_read_fp4_kernel(ReadArgs a) {
  __shared__ __attribute__((aligned(16))) u8 s_tile[4][512];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 7, tok = lane >> 3;
  const int hkv = a.num_kv_heads;
  const int v = blockIdx.y * 2 + (w >> 1);  // key heads, then value heads
  if (v >= 2 * hkv || blockIdx.x * 16 + (w & 1) * 8 >= a.num_tokens) return;
  const int t = blockIdx.x * 16 + (w & 1) * 8 + tok;
  const bool exists = t < a.num_tokens;
  int64_t slot = exists ? a.slots[t] : -1;
  if (slot >= a.num_slots || slot < -1) {
    if (v == 0 && c == 0) flag_index_error(a.err, NVAMD_ERR_SLOT);
    slot = -1;
  }
  const bool live = slot >= 0;
  const int h = v < hkv ? v : v - hkv;
  const Fp4Row r = row_at(live ? slot : 0, h, hkv, a.bs_log2);
  const u32x4 zero = {0u, 0u, 0u, 0u};
  if (v < hkv) {
    u32x4 lo = zero, hi = zero;
    if (live) {
      const u32 *row = reinterpret_cast<const u32 *>(a.cache.k_codes + r.tile * kFp4TileBytes + r.t * kFp4RowBytes);
      const u8 *s = a.cache.k_scales + r.tile * kFp4TileScales;
      lo = fp4_values(row[c], fp4_scale(s[fp4_key_scale_at(r.t, c >> 2)]));
      hi = fp4_values(row[8 + c], fp4_scale(s[fp4_key_scale_at(r.t, 2 + (c >> 2))]));
    }
    if (exists) {
      u16 *dst = a.k + t * a.k_stride + h * kHeadDim + 8 * c;
      put16<STREAM>(dst, lo);
      put16<STREAM>(dst + 64, hi);
    }
    return;
  }
  // Row byte `lane` of the 8 tokens, then through LDS to lane c of each: bytes 8 (c % 2) .. +7 of block c / 2.
  auto place = [&](int64_t s) {
    const Fp4Row x = row_at(s, h, hkv, a.bs_log2);
    return a.cache.v_codes + x.tile * kFp4TileBytes + lane * kFp4Tile + x.t;
  };
  u8 *tile = s_tile[w];
  const u32 scale_byte = live ? a.cache.v_scales[r.tile * kFp4TileScales + fp4_value_scale_at(r.t, c >> 1)] : 0u;
  uint64_t bytes = 0;
  if (__all(live && slot == uniform64(slot) + tok)) {
    const int64_t s0 = uniform64(slot);
    const int o = (int)(s0 & 7);
    bytes = *reinterpret_cast<const uint64_t *>(place(s0) - o);
    if (o != 0) bytes = (bytes >> (8 * o)) | (*reinterpret_cast<const uint64_t *>(place(s0 + 8 - o)) << (64 - 8 * o));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t s = lane_value(slot, 8 * i);
      if (s >= 0) bytes |= (uint64_t)*place(s) << (8 * i);
    }
  }
  *reinterpret_cast<uint64_t *>(tile + lane * 8) = bytes;
  wave_lds_fence();
  u32x4 first = zero, last = zero;
  if (live) {
    const u8 *p = tile + (16 * (c >> 1) + 8 * (c & 1)) * 8 + tok;
    const float scale = fp4_scale(scale_byte);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32 x = fp4_pair<0>(p[2 * j * 8], scale), y = fp4_pair<0>(p[(2 * j + 1) * 8], scale);
      first[j] = pair_lo(x, y);
      last[j] = pair_hi(x, y);
    }
  }
  if (exists) {
    u16 *dst = a.v + t * a.v_stride + h * kHeadDim + 32 * (c >> 1) + 8 * (c & 1);
    put16<STREAM>(dst, first);
    put16<STREAM>(dst + 16, last);
  }
}

struct NormRopeFp4Args {
  WriteArgs w;
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
  int num_heads;  // 0: rows are only stored
  float eps;
};

// A wave: 8 tokens, heads_per_wave of the vectors of each: its query heads, its key heads, its value heads.
template <bool ROPE, bool STREAM>
__global__ void __launch_bounds__(256)
rows_fp4_kernel(NormRopeFp4Args a) {
  __shared__ __attribute__((aligned(16))) u8 s_tile[4][2][512];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 7, tok = lane >> 3;
  const int hkv = a.w.num_kv_heads, hq = ROPE ? a.num_heads : 0;
  const int h_begin = (blockIdx.y * 2 + (w >> 1)) * a.w.heads_per_wave;
  const int h_end = min(h_begin + a.w.heads_per_wave, hq + 2 * hkv);
  if (h_begin >= h_end || blockIdx.x * 16 + (w & 1) * 8 >= a.w.num_tokens) return;
  const int t = blockIdx.x * 16 + (w & 1) * 8 + tok;
  const bool exists = t < a.w.num_tokens;
  int64_t slot = exists ? a.w.slots[t] : -1;
  if (slot >= a.w.num_slots || slot < -1) {  // skip the row, report it once per token
    if (h_begin == 0 && c == 0) flag_index_error(a.w.err, NVAMD_ERR_SLOT);
    slot = -1;
  }
  const bool run = __all(slot >= 0 && slot == uniform64(slot) + tok);

  float cs[8], sn[8];
  u32x4 qw_lo, qw_hi, kw_lo, kw_hi;
  if constexpr (ROPE) {
    if (h_begin < hq + hkv) {
      int64_t pos = exists ? a.positions[t] : 0;
      if (pos < 0 || pos >= a.max_positions) {  // clamp and report
        if (h_begin == 0 && c == 0) flag_index_error(a.w.err, NVAMD_ERR_POSITION);
        pos = pos < 0 ? 0 : a.max_positions - 1;
      }
      const float *row = a.cos_sin + pos * kHeadDim + 8 * c;
      const f32x4 c0 = *reinterpret_cast<const f32x4 *>(row), c1 = *reinterpret_cast<const f32x4 *>(row + 4);
      const f32x4 s0 = *reinterpret_cast<const f32x4 *>(row + 64), s1 = *reinterpret_cast<const f32x4 *>(row + 68);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = e < 4 ? c0[e & 3] : c1[e & 3];
        sn[e] = e < 4 ? s0[e & 3] : s1[e & 3];
      }
      qw_lo = ld16(a.q_w + 8 * c);
      qw_hi = ld16(a.q_w + 64 + 8 * c);
      kw_lo = ld16(a.k_w + 8 * c);
      kw_hi = ld16(a.k_w + 64 + 8 * c);
    }
  }
  const int64_t tt = exists ? t : 0;  // lanes without a token read the first one's rows and write nothing
  auto source = [&](int v) {
    const u16 *p = v < hq ? a.q + tt * a.q_stride + v * kHeadDim
                 : v < hq + hkv ? a.w.k + tt * a.w.k_stride + (v - hq) * kHeadDim
                                : a.w.v + tt * a.w.v_stride + (v - hq - hkv) * kHeadDim;
    return p + 8 * c;
  };
  const u16 *src = source(h_begin);
  u32x4 next_lo = get16<STREAM>(src), next_hi = get16<STREAM>(src + 64);
#pragma unroll 1
  for (int v = h_begin; v < h_end; ++v) {
    u32x4 lo = next_lo, hi = next_hi;
    if (v + 1 < h_end) {  // the next head's row is on its way during this one's work
      src = source(v + 1);
      next_lo = get16<STREAM>(src);
      next_hi = get16<STREAM>(src + 64);
    }
    if (v >= hq + hkv) {
      const int h = v - hq - hkv;
      u8 *tile = s_tile[w][v & 1];  // the other one's reads are done: they have left as stores
      const Fp4Row r = row_at(slot < 0 ? 0 : slot, h, hkv, a.w.bs_log2);
      value_bytes(a.w.cache, r, slot >= 0, c, tok, lo, hi, tile);
      wave_lds_fence();
      store_values(a.w.cache, tile, slot, run, h, hkv, a.w.bs_log2, lane);
      continue;
    }
    const bool is_q = v < hq;
    if constexpr (ROPE) {
      // Keeps the conversions of the row's 16 numbers and of the weights inside the loop: hoisted, they would hold 64
      // registers and with them a third of the waves.
#pragma unroll
      for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(cs[e]), "+v"(sn[e]));
      asm volatile("" : "+v"(qw_lo), "+v"(qw_hi), "+v"(kw_lo), "+v"(kw_hi));
      const double rstd = norm_factor(dpp_sum8(sum_squares(lo, hi)), (double)a.eps);
      // The row's 64-bit numbers are made anew: kept from the sum they hold 16 registers more, with them one wave of
      // four (36,488 tokens 127 us, so 117).
      asm volatile("" : "+v"(lo), "+v"(hi));
      norm_rope_f64(lo, hi, is_q ? qw_lo : kw_lo, is_q ? qw_hi : kw_hi, cs, sn, rstd);
      u16 *dst = is_q ? a.q_out + tt * a.q_out_stride + v * kHeadDim
                      : a.k_out ? a.k_out + tt * a.k_out_stride + (v - hq) * kHeadDim : nullptr;
      if (dst != nullptr && exists) {
        st16(dst + 8 * c, lo);
        st16(dst + 8 * c + 64, hi);
      }
    }
    if (!is_q && slot >= 0) store_key(a.w.cache, row_at(slot, v - hq, hkv, a.w.bs_log2), c, lo, hi);
  }
}

// A workgroup is 2 x 8 tokens x 2 waves' heads: the two halves of a tile's value bytes share lines, and meet in one L2
// (8 tokens x 4 waves': 12,345 rows read in 17.8 us, so 15.0; 36,488 written in 39.9, so 36.6).  A wave takes up to
// `per_wave` heads; fewer where that leaves too few waves to fill the card.  0: more than a launch takes.
int heads_per_wave(int num_tokens, int vecs, int per_wave, dim3 *grid) {
  const int64_t octets = ((int64_t)num_tokens + 7) / 8;
  while (per_wave > 1 && octets * ceil_div(vecs, per_wave) < kWantedWaves) per_wave >>= 1;
  *grid = dim3((unsigned)((octets + 1) / 2), (unsigned)ceil_div(ceil_div(vecs, per_wave), 2));
  return octets < (1 << 24) && grid->y <= 65535 ? per_wave : 0;
}

bool streams(int num_tokens, int num_kv_heads) { return (int64_t)num_tokens * num_kv_heads * kHeadDim >= kStreamElems; }

template <bool ROPE>
int launch_rows(NormRopeFp4Args &a, hipStream_t stream) {
  dim3 grid;
  a.w.heads_per_wave = heads_per_wave(a.w.num_tokens, (ROPE ? a.num_heads : 0) + 2 * a.w.num_kv_heads,
                                      ROPE ? kRopeHeads : 1, &grid);
  if (a.w.heads_per_wave == 0) return NVAMD_EUNSUPPORTED;
  // (the rotation measured the same either way)
  if (!ROPE && streams(a.w.num_tokens, a.w.num_kv_heads))
    hipLaunchKernelGGL((rows_fp4_kernel<ROPE, !ROPE>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((rows_fp4_kernel<ROPE, false>), grid, dim3(256), 0, stream, a);
  return launch_status();
}

bool rows_ok(const void *p, int64_t stride, int heads) {
  return p && aligned16(p) && stride % 8 == 0 && stride >= (int64_t)heads * kHeadDim;
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
  NormRopeFp4Args a = {};
  a.w = w;
  return launch_rows<false>(a, stream);
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
  dim3 grid;
  if (heads_per_wave(num_tokens, 2 * num_kv_heads, 1, &grid) == 0) return NVAMD_EUNSUPPORTED;
  ReadArgs a{static_cast<u16 *>(k), k_stride, static_cast<u16 *>(v), v_stride, w.cache, w.slots, w.num_slots,
             num_tokens, num_kv_heads, w.bs_log2, w.err};
  if (streams(num_tokens, num_kv_heads))
    hipLaunchKernelGGL((kv_read_fp4_kernel<true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((kv_read_fp4_kernel<false>), grid, dim3(256), 0, stream, a);
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
  return launch_rows<true>(a, stream);
}
