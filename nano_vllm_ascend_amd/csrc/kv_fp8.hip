// The 8-bit paged KV cache: writing rows, reading rows back, and the per-head QK-RMSNorm + RoPE that writes them in the
// same pass (the 8-bit counterparts of kv_store.hip).
//
// The 16 tokens of a tile share a scale, so a wave takes all rows that a call writes to a head's tile: a run of rows
// that follow one another, as their slots do.  It finds the runs that begin among its own rows by itself, from the
// slots.  A key's row is 8 lanes of 16 dims (the rotation then needs no lane exchange); of the values a lane takes two
// dims of all tokens, so that what it writes, 16 tokens of a dim in consecutive bytes, needs no transpose.
//
// All three are bound by memory: per head vector 256 bytes of bf16 and 128 of the cache, once.  12,345 tokens of 8 kv
// heads written and read back 152 MB in 28 us (5.4 TB/s); 36,488 tokens of prompts, 16 query heads, rotated and stored with
// the keys returned 598 MB in 139 us (4.3 TB/s: the 64-bit arithmetic is 40% of its time and hides behind four waves a
// SIMD; at two it took 164), and with the rows read back 842 MB in 163 us (5.1).  One token: 3 us, the launch.
#include "fp8_rows.h"
#include "norm_rope64.h"

namespace nvamd {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// A 64-bit value of one lane, as a scalar.
__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const u32 lo = (u32)__builtin_amdgcn_readlane((int)(u32)v, lane);
  const u32 hi = (u32)__builtin_amdgcn_readlane((int)(u32)((uint64_t)v >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

struct RowsArgs {
  const u16 *k;
  int64_t k_stride;
  const u16 *v;
  int64_t v_stride;
  Fp8Cache cache;
  const int64_t *slots;
  int64_t num_slots;
  int num_tokens;
  int num_kv_heads;
  int bs_log2;
  u32 *err;
  // the rotation's
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
  int q_heads;    // of a wave
  int k_heads;
  float eps;
};

// The table's row of dims 8c .. 8c + 7 of a token.
__device__ __forceinline__ void rope_row(const RowsArgs &a, int64_t t, int c, bool report, float (&cs)[8], float (&sn)[8]) {
  int64_t pos = a.positions[t];
  if (pos < 0 || pos >= a.max_positions) {  // clamp and report
    if (report) flag_index_error(a.err, NVAMD_ERR_POSITION);
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
}

// Keeps the conversions of a row's 16 numbers and of the weights inside a loop over heads: hoisted, they would hold 64
// registers and with them half of the waves.
__device__ __forceinline__ void keep_here(float (&cs)[8], float (&sn)[8], u32x4 &w_lo, u32x4 &w_hi) {
#pragma unroll
  for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(cs[e]), "+v"(sn[e]));
  asm volatile("" : "+v"(w_lo), "+v"(w_hi));
}

// Runs among rows base .. base + ROWS - 1: calls body(first row, its slot, rows).  A run is rows whose slots follow one
// another inside a tile; it may go on past the wave's own rows.  Rows without a slot come as runs of one, slot -1, if
// asked for.  So does a run in a tile that an earlier row of the wave's window lies in (two waves would write the tile at
// once): it is reported, and stored by nobody.
template <int ROWS, typename Body>
__device__ __forceinline__ void for_runs(const RowsArgs &a, int64_t base, int lane, bool report, bool slotless,
                                         Body &&body) {
  // Of the window's 64 rows these lie before the wave's own, and behind those the ones that a run may go on in.
  constexpr int kBefore = 64 - ROWS - (kFp8Tile - 1);
  static_assert(kBefore >= NVAMD_FP8_ORDER_ROWS);
  const int64_t r = base - kBefore + lane;
  const bool exists = r >= 0 && r < a.num_tokens;
  int64_t slot = exists ? a.slots[r] : -1;
  if (slot >= a.num_slots || slot < -1) {  // skip the row, report it once
    if (report && lane >= kBefore && lane < kBefore + ROWS) flag_index_error(a.err, NVAMD_ERR_SLOT);
    slot = -1;
  }
  const int64_t before = __shfl_up(slot, 1);
  const bool follows = lane > 0 && slot >= 0 && (slot & (kFp8Tile - 1)) != 0 && before + 1 == slot;
  const uint64_t go_on = __ballot(follows);
  uint64_t begins = __ballot(exists && !follows && (slot >= 0 || slotless)) & (((1ull << ROWS) - 1) << kBefore);
  while (begins != 0) {
    const int j = __ffsll((unsigned long long)begins) - 1;
    begins &= begins - 1;
    int64_t first = lane_value(slot, j);
    if (first >= 0 && __ballot(lane < j && slot >= 0 && (slot ^ first) < kFp8Tile) != 0) {
      if (report && lane == 0) flag_index_error(a.err, NVAMD_ERR_ORDER);
      if (!slotless) continue;
      first = -1;
    }
    body(base - kBefore + j, first, __ffsll((unsigned long long)~(go_on >> (j + 1))));
  }
}

// Heads that a wave of the rotation takes one after another: the table's rows and the weights are read once for them.
// Fewer where that leaves less than four waves for each SIMD of 256 CUs.  us, with the rows read back, of 36,488 tokens at
// query / key heads of 8 / 8, 8 / 4, 8 / 2, 4 / 4, 1 / 1: 183, 176, 179, 188, 201; of 2,600 tokens 47 (8 / 8), 20 (1 / 1).
constexpr int kQueryHeads = 8, kKeyHeads = 4;
constexpr int kWantedWaves = 4096;

// blockIdx.y: groups of query heads, groups of key heads (of one without the rotation), value heads.  ROWS rows of the
// call to a wave: 16, or 1 where there are few.
template <bool ROPE, int ROWS>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4)))
rows_fp8_kernel(RowsArgs a) {
  // A lane's own numbers of the table for its two tokens of a run: kept in registers they take 32, and with them one wave
  // of four.
  __shared__ f32x4 s_turn[ROPE ? kWaves : 1][2][4][ROPE ? 64 : 1];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 7, tok = lane >> 3;
  const int64_t base = ((int64_t)blockIdx.x * kWaves + w) * ROWS;
  if (base >= a.num_tokens) return;
  const int hkv = a.num_kv_heads;
  int y = blockIdx.y;
  if constexpr (ROPE) {
    const int q_groups = (a.num_heads + a.q_heads - 1) / a.q_heads;
    if (y < q_groups) {
      const int h0 = y * a.q_heads, h1 = min(h0 + a.q_heads, a.num_heads);
      u32x4 w_lo = ld16(a.q_w + 8 * c), w_hi = ld16(a.q_w + 64 + 8 * c);
      // 16 rows: 8 at a time, head after head; one row: its heads at a time.
#pragma unroll 1
      for (int p = 0; p < (ROWS + 7) / 8; ++p) {
        const int64_t t = ROWS == 1 ? base : base + 8 * p + tok;
        const bool exists = t < a.num_tokens;
        const int64_t tt = exists ? t : base;
        float cs[8], sn[8];
        rope_row(a, tt, c, y == 0 && c == 0 && (ROWS > 1 || tok == 0), cs, sn);
        auto head_of = [&](int i) { return ROWS == 1 ? min(h0 + tok, h1 - 1) : i; };
        auto source = [&](int i) { return a.q + tt * a.q_stride + head_of(i) * kHeadDim + 8 * c; };
        const int end = ROWS == 1 ? h0 + 1 : h1;
        u32x4 next_lo = ld16(source(h0)), next_hi = ld16(source(h0) + 64);
#pragma unroll 1
        for (int i = h0; i < end; ++i) {
          u32x4 lo = next_lo, hi = next_hi;
          if (i + 1 < end) {  // the next head's row is on its way during this one's work
            next_lo = ld16(source(i + 1));
            next_hi = ld16(source(i + 1) + 64);
          }
          keep_here(cs, sn, w_lo, w_hi);
          const double rstd = norm_factor(dpp_sum8(sum_squares(lo, hi)), (double)a.eps);
          asm volatile("" : "+v"(lo), "+v"(hi));  // the row's 64-bit numbers are made anew
          norm_rope_f64(lo, hi, w_lo, w_hi, cs, sn, rstd);
          u16 *dst = a.q_out + tt * a.q_out_stride + head_of(i) * kHeadDim + 8 * c;
          if (exists && (ROWS > 1 || h0 + tok < h1)) {
            st16(dst, lo);
            st16(dst + 64, hi);
          }
        }
      }
      return;
    }
    y -= q_groups;
  }
  const int k_groups = (hkv + a.k_heads - 1) / a.k_heads;
  if (y < k_groups) {
    const int h0 = y * a.k_heads, h1 = min(h0 + a.k_heads, hkv);
    for_runs<ROWS>(a, base, lane, y == 0, ROPE && a.k_out != nullptr, [&](int64_t row, int64_t slot, int n) {
      const int o = slot < 0 ? 0 : (int)(slot & (kFp8Tile - 1));
      const int64_t block = slot < 0 ? 0 : slot >> a.bs_log2;
      const int token = slot < 0 ? 0 : (int)(slot & ((1 << a.bs_log2) - 1));
      u32x4 w_lo, w_hi;
      int64_t at[2];  // of the lane's two tokens; lanes without one read the first row's
      bool in[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int i = 8 * p + tok - o;
        in[p] = i >= 0 && i < n;
        at[p] = in[p] ? row + i : row;
      }
      if constexpr (ROPE) {
        w_lo = ld16(a.k_w + 8 * c);
        w_hi = ld16(a.k_w + 64 + 8 * c);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float cs[8], sn[8];
          rope_row(a, at[p], c, false, cs, sn);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            s_turn[w][p][x][lane] = f32x4{cs[4 * x], cs[4 * x + 1], cs[4 * x + 2], cs[4 * x + 3]};
            s_turn[w][p][2 + x][lane] = f32x4{sn[4 * x], sn[4 * x + 1], sn[4 * x + 2], sn[4 * x + 3]};
          }
        }
      }
#pragma unroll 1
      for (int h = h0; h < h1; ++h) {
        const int64_t tile = fp8_tile(block, token, h, hkv, a.bs_log2);
        const u32 held = o > 0 ? a.cache.k_scales[tile] : 0u;
        u32 x[16];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const u16 *src = a.k + at[p] * a.k_stride + h * kHeadDim + 8 * c;
          u32x4 lo = ld16(src), hi = ld16(src + 64);
          if constexpr (ROPE) {
            asm volatile("" ::: "memory");  // read anew for each head
            float cs[8], sn[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              cs[e] = s_turn[w][p][e >> 2][lane][e & 3];
              sn[e] = s_turn[w][p][2 + (e >> 2)][lane][e & 3];
            }
            keep_here(cs, sn, w_lo, w_hi);
            const double rstd = norm_factor(dpp_sum8(sum_squares(lo, hi)), (double)a.eps);
            asm volatile("" : "+v"(lo), "+v"(hi));
            norm_rope_f64(lo, hi, w_lo, w_hi, cs, sn, rstd);
            if (a.k_out != nullptr && in[p]) {
              u16 *dst = a.k_out + at[p] * a.k_out_stride + h * kHeadDim + 8 * c;
              st16(dst, lo);
              st16(dst + 64, hi);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[8 * p + i] = in[p] ? lo[i] : 0u;
            x[8 * p + 4 + i] = in[p] ? hi[i] : 0u;
          }
        }
        if (slot >= 0) store_keys(a.cache, tile, o, n, held, tok, c, x);
      }
    });
    return;
  }
  const int h = y - k_groups;
  for_runs<ROWS>(a, base, lane, false, false, [&](int64_t row, int64_t slot, int n) {
    const int o = (int)(slot & (kFp8Tile - 1));
    const int64_t tile = fp8_tile(slot >> a.bs_log2, (int)(slot & ((1 << a.bs_log2) - 1)), h, hkv, a.bs_log2);
    u32 held = 0;
    u32x4 old[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
    if (o > 0) {
      const u32x4 *p = reinterpret_cast<const u32x4 *>(a.cache.v_codes + tile * kFp8TileBytes + 2 * lane * kFp8Tile);
      held = a.cache.v_scales[tile];
      old[0] = p[0];
      old[1] = p[1];
    }
    const u16 *src = a.v + row * a.v_stride + h * kHeadDim + 2 * lane;
    u32 x[16];
#pragma unroll
    for (int t = 0; t < 16; ++t)
      x[t] = t >= o && t < o + n ? *reinterpret_cast<const u32 *>(src + (t - o) * a.v_stride) : 0u;
    store_values(a.cache, tile, o, n, held, old, lane, x);
  });
}

// The other way round: blockIdx.y is a key head or a value head; ROWS rows to a wave, 16, or 1 where there are few.  A
// row without a slot, or with one outside the cache, is zeros.
struct ReadArgs {
  RowsArgs r;  // cache, slots and their numbers
  u16 *k;
  int64_t k_stride;
  u16 *v;
  int64_t v_stride;
};

template <int ROWS>
__global__ void __launch_bounds__(kThreads)
kv_read_fp8_kernel(ReadArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t base = ((int64_t)blockIdx.x * kWaves + w) * ROWS;
  if (base >= a.r.num_tokens) return;
  const int hkv = a.r.num_kv_heads, bs_log2 = a.r.bs_log2;
  // Many rows pass the caches by: 36,488 written and read back 163 us, 177 with ordinary stores; 12,345 28.2, 30.0.
  auto put = [](auto *to, auto x) {
    if constexpr (ROWS == 1) *to = x;
    else __builtin_nontemporal_store(x, to);
  };
  const int h = (int)blockIdx.y < hkv ? blockIdx.y : blockIdx.y - hkv;
  if ((int)blockIdx.y < hkv) {
    const int c = lane & 7;
#pragma unroll
    for (int p = 0; p < (ROWS + 7) / 8; ++p) {
      const int64_t t = base + 8 * p + (lane >> 3);
      if (t >= a.r.num_tokens || 8 * p + (lane >> 3) >= ROWS) continue;
      int64_t slot = a.r.slots[t];
      if (slot >= a.r.num_slots || slot < -1) {
        if (h == 0 && c == 0) flag_index_error(a.r.err, NVAMD_ERR_SLOT);
        slot = -1;
      }
      u32x4 lo = {0u, 0u, 0u, 0u}, hi = lo;
      if (slot >= 0) {
        const int64_t tile = fp8_tile(slot >> bs_log2, (int)(slot & ((1 << bs_log2) - 1)), h, hkv, bs_log2);
        const u8 *src = a.r.cache.k_codes + tile * kFp8TileBytes + fp8_key_at((int)(slot & (kFp8Tile - 1)), 8 * c);
        const u32x2 x = *reinterpret_cast<const u32x2 *>(src), y = *reinterpret_cast<const u32x2 *>(src + kFp8TileBytes / 2);
        const float scale = fp8_scale(a.r.cache.k_scales[tile]);
        lo = u32x4{fp8_pair<false>(x[0], scale), fp8_pair<true>(x[0], scale), fp8_pair<false>(x[1], scale),
                   fp8_pair<true>(x[1], scale)};
        hi = u32x4{fp8_pair<false>(y[0], scale), fp8_pair<true>(y[0], scale), fp8_pair<false>(y[1], scale),
                   fp8_pair<true>(y[1], scale)};
      }
      u16 *dst = a.k + t * a.k_stride + h * kHeadDim + 8 * c;
      put(reinterpret_cast<u32x4 *>(dst), lo);
      put(reinterpret_cast<u32x4 *>(dst + 64), hi);
    }
    return;
  }
  // Values: a tile once for the rows of a run that the wave has.
  auto row = [&](int64_t t) { return reinterpret_cast<u32 *>(a.v + t * a.v_stride + h * kHeadDim + 2 * lane); };
  const int64_t r = base + lane;
  const bool exists = lane < ROWS && r < a.r.num_tokens;
  int64_t slot = exists ? a.r.slots[r] : -1;
  if (slot >= a.r.num_slots || slot < -1) slot = -1;
  const int64_t before = __shfl_up(slot, 1);
  const bool follows = lane > 0 && slot >= 0 && (slot & (kFp8Tile - 1)) != 0 && before + 1 == slot;
  const uint64_t go_on = __ballot(follows);
  uint64_t begins = __ballot(exists && !follows);
  while (begins != 0) {
    const int j = __ffsll((unsigned long long)begins) - 1;
    begins &= begins - 1;
    const int64_t s = lane_value(slot, j);
    if (s < 0) {
      *row(base + j) = 0u;
      continue;
    }
    const int n = __ffsll((unsigned long long)~(go_on >> (j + 1))), o = (int)(s & (kFp8Tile - 1));
    const int64_t tile = fp8_tile(s >> bs_log2, (int)(s & ((1 << bs_log2) - 1)), h, hkv, bs_log2);
    const u32x4 *p = reinterpret_cast<const u32x4 *>(a.r.cache.v_codes + tile * kFp8TileBytes + 2 * lane * kFp8Tile);
    const u32x4 x = p[0], y = p[1];
    const float scale = fp8_scale(a.r.cache.v_scales[tile]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32 a01 = __builtin_amdgcn_perm(y[i], x[i], 0x05010400u), a23 = __builtin_amdgcn_perm(y[i], x[i], 0x07030602u);
      const u32 out[4] = {fp8_pair<false>(a01, scale), fp8_pair<true>(a01, scale), fp8_pair<false>(a23, scale),
                          fp8_pair<true>(a23, scale)};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 4 * i + e;
        if (t >= o && t < o + n) put(row(base + j + t - o), out[e]);
      }
    }
  }
}

// Tiles that rows go behind, as they were before: [layer][row][kv head] records of the tile's keys, values, place and
// scales.  A wave to a record.  Bound by memory, up to 4.1 KB each way: 8 heads in 28 layers take 4.2 us for 1 row, 9.0 for
// 32 and 23 for 100, from a graph; kept before every step, 32 x 256 tokens decode in 1.100 ms for 1.088, 100 x 4,000 in 5.42
// for 5.40.  (Stores past the caches: 1.103 and 5.43.)
constexpr int kKeptBytes = 2 * kFp8TileBytes + 16;
struct KeptArgs {
  u8 *kept;
  Fp8Cache cache;  // of all layers
  int64_t layer_tiles;
  const int64_t *slots;
  int64_t num_slots;
  int num_layers;
  int num_tokens;
  int num_kv_heads;
  int bs_log2;
};

template <bool RESTORE>
__global__ void __launch_bounds__(kThreads)
kept_tiles_fp8_kernel(KeptArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)blockIdx.x * kWaves + w;
  if (item >= (int64_t)a.num_layers * a.num_tokens * a.num_kv_heads) return;
  u8 *rec = a.kept + item * kKeptBytes;
  int64_t *place = reinterpret_cast<int64_t *>(rec + 2 * kFp8TileBytes);  // 16 * the pool's tile + tokens; -1: no tile
  u8 *scales = rec + 2 * kFp8TileBytes + 8;
  int64_t at;
  if constexpr (RESTORE) {
    at = *place;
    if (at >= (a.num_layers * a.layer_tiles) * kFp8Tile) return;  // never leave the pool
  } else {
    const int64_t rest = item / a.num_kv_heads, layer = rest / a.num_tokens;
    const int head = (int)(item - rest * a.num_kv_heads);
    const int64_t slot = a.slots[rest - layer * a.num_tokens];
    const int o = (int)(slot & (kFp8Tile - 1));  // a row that begins its tile goes behind none
    const bool behind = slot >= 0 && slot < a.num_slots && o > 0;
    at = behind ? (layer * a.layer_tiles + fp8_tile(slot >> a.bs_log2, (int)(slot & ((1 << a.bs_log2) - 1)), head,
                                                    a.num_kv_heads, a.bs_log2)) * kFp8Tile + o
                : -1;
    if (lane == 0) *place = at;
  }
  if (at < 0) return;
  const int64_t tile = at / kFp8Tile;
  const int tokens = (int)(at % kFp8Tile);  // that the tile holds
  u32x4 *k = reinterpret_cast<u32x4 *>(a.cache.k_codes + tile * kFp8TileBytes), *kept_k = reinterpret_cast<u32x4 *>(rec);
  u32x4 *v = reinterpret_cast<u32x4 *>(a.cache.v_codes + tile * kFp8TileBytes), *kept_v = kept_k + kFp8TileBytes / 16;
  auto copy = [](auto *cache, auto *kept) {
    if constexpr (RESTORE) *cache = *kept;
    else *kept = *cache;
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (lane >> 2 < tokens) copy(k + 64 * i + lane, kept_k + 64 * i + lane);  // a key's half is four lanes
    copy(v + 64 * i + lane, kept_v + 64 * i + lane);
  }
  if (lane == 0) {
    copy(a.cache.k_scales + tile, scales);
    copy(a.cache.v_scales + tile, scales + 1);
  }
}

template <bool RESTORE>
int launch_kept(u8 *kept, size_t kept_bytes, void *k_codes, void *k_scales, void *v_codes, void *v_scales, int num_layers,
                int num_blocks, int block_size, const int64_t *slots, int num_tokens, int num_kv_heads, int head_dim,
                hipStream_t stream) {
  if (num_tokens == 0) return NVAMD_OK;
  if (num_layers <= 0 || num_blocks <= 0 || num_tokens < 0 || num_kv_heads <= 0) return NVAMD_EINVAL;
  const int bs_log2 = log2_exact(block_size);
  if (head_dim != kHeadDim || bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!kept || !aligned16(kept) || !fp8_cache_ok(k_codes, k_scales, v_codes, v_scales) || (!RESTORE && !slots))
    return NVAMD_EINVAL;
  if ((int64_t)num_layers * num_tokens > 0x7fffffff / num_kv_heads) return NVAMD_EUNSUPPORTED;
  const int64_t records = (int64_t)num_layers * num_tokens * num_kv_heads;
  if (kept_bytes < (size_t)records * kKeptBytes) return NVAMD_EWORKSPACE;
  const KeptArgs a = {kept,
                      {static_cast<u8 *>(k_codes), static_cast<u8 *>(k_scales), static_cast<u8 *>(v_codes),
                       static_cast<u8 *>(v_scales)},
                      ((int64_t)num_blocks * num_kv_heads << bs_log2) / kFp8Tile,
                      slots,
                      (int64_t)num_blocks << bs_log2,
                      num_layers,
                      num_tokens,
                      num_kv_heads,
                      bs_log2};
  hipLaunchKernelGGL(kept_tiles_fp8_kernel<RESTORE>, dim3((unsigned)((records + kWaves - 1) / kWaves)), dim3(kThreads), 0,
                     stream, a);
  return launch_status();
}

// A wave looks after the runs that begin in one row up to here, in 16 rows from there on: the rows of a decode step have a
// tile each, whose runs a wave takes one after another, those of a long prompt share tiles.  us from a graph, one / 16,
// written: rows of a tile each, 32 3.2 / 17.7, 512 7.1 / 20.1, 1,000 11.8 / 20.8; of one run, 300 3.7 / 3.5, 500 4.4 / 3.4,
// 1,000 6.6 / 3.6.  Rotated and stored, 16 query heads: of a tile each, 32 4.8 / 39.5, 512 13.5 / 42.4; of one run, 500 6.8 /
// 5.2, 1,000 12.2 / 6.6.
constexpr int kFewTokens = 512;

template <bool ROPE>
int launch_rows(RowsArgs &a, hipStream_t stream) {
  const bool few = a.num_tokens <= kFewTokens;
  const int64_t windows = ceil_div(a.num_tokens, few ? 1 : 16);
  // one row: its query heads side by side in a wave; else and of keys one after another
  a.q_heads = kQueryHeads;
  a.k_heads = ROPE && !few ? kKeyHeads : 1;
  if (ROPE && !few) {
    while (a.q_heads > 1 && windows * ceil_div(a.num_heads, a.q_heads) < kWantedWaves) a.q_heads /= 2;
    while (a.k_heads > 1 && windows * ceil_div(a.num_kv_heads, a.k_heads) < kWantedWaves) a.k_heads /= 2;
  }
  const int y = (ROPE ? ceil_div(a.num_heads, a.q_heads) : 0) + ceil_div(a.num_kv_heads, a.k_heads) + a.num_kv_heads;
  if (y > 65535) return NVAMD_EUNSUPPORTED;
  const dim3 grid((unsigned)((windows + kWaves - 1) / kWaves), (unsigned)y);
  if (few)
    hipLaunchKernelGGL((rows_fp8_kernel<ROPE, 1>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((rows_fp8_kernel<ROPE, 16>), grid, dim3(kThreads), 0, stream, a);
  return launch_status();
}

bool rows_ok(const void *p, int64_t stride, int heads) {
  return p && aligned16(p) && stride % 8 == 0 && stride >= (int64_t)heads * kHeadDim;
}

// Checks shared by the entry points; fills what they share.
int fill_rows_args(RowsArgs &a, const void *k, int64_t k_stride, const void *v, int64_t v_stride, void *k_codes,
                   void *k_scales, void *v_codes, void *v_scales, const int64_t *slots, int num_tokens,
                   int num_kv_heads, int head_dim, int num_blocks, int block_size) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0) return NVAMD_EINVAL;
  if (head_dim != kHeadDim) return NVAMD_EUNSUPPORTED;
  const int bs_log2 = log2_exact(block_size);
  if (bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!rows_ok(k, k_stride, num_kv_heads) || !rows_ok(v, v_stride, num_kv_heads) ||
      !fp8_cache_ok(k_codes, k_scales, v_codes, v_scales) || !slots)
    return NVAMD_EINVAL;
  if (num_tokens >= 1 << 27 || 2 * (int64_t)num_kv_heads > 65535) return NVAMD_EUNSUPPORTED;
  a = RowsArgs{};
  a.k = static_cast<const u16 *>(k);
  a.k_stride = k_stride;
  a.v = static_cast<const u16 *>(v);
  a.v_stride = v_stride;
  a.cache = Fp8Cache{static_cast<u8 *>(k_codes), static_cast<u8 *>(k_scales), static_cast<u8 *>(v_codes),
                     static_cast<u8 *>(v_scales)};
  a.slots = slots;
  a.num_slots = (int64_t)num_blocks << bs_log2;
  a.num_tokens = num_tokens;
  a.num_kv_heads = num_kv_heads;
  a.bs_log2 = bs_log2;
  a.err = index_error_word();
  return NVAMD_OK;
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" int nvamd_kv_cache_write_fp8(const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                                        void *k_codes, void *k_scales, void *v_codes, void *v_scales, int num_blocks,
                                        int block_size, const int64_t *slot_mapping, int num_tokens, int num_kv_heads,
                                        int head_dim, hipStream_t stream) {
  if (num_tokens == 0) return NVAMD_OK;
  RowsArgs a;
  const int st = fill_rows_args(a, k, k_stride, v, v_stride, k_codes, k_scales, v_codes, v_scales, slot_mapping,
                                num_tokens, num_kv_heads, head_dim, num_blocks, block_size);
  if (st != NVAMD_OK) return st;
  return launch_rows<false>(a, stream);
}

extern "C" int nvamd_kv_cache_read_fp8(void *k, int64_t k_stride, void *v, int64_t v_stride, const void *k_codes,
                                       const void *k_scales, const void *v_codes, const void *v_scales,
                                       int num_blocks, int block_size, const int64_t *slot_mapping, int num_tokens,
                                       int num_kv_heads, int head_dim, hipStream_t stream) {
  if (num_tokens == 0) return NVAMD_OK;
  ReadArgs a;
  const int st = fill_rows_args(a.r, k, k_stride, v, v_stride, const_cast<void *>(k_codes),
                                const_cast<void *>(k_scales), const_cast<void *>(v_codes),
                                const_cast<void *>(v_scales), slot_mapping, num_tokens, num_kv_heads, head_dim,
                                num_blocks, block_size);
  if (st != NVAMD_OK) return st;
  a.k = static_cast<u16 *>(k);
  a.k_stride = k_stride;
  a.v = static_cast<u16 *>(v);
  a.v_stride = v_stride;
  // us, one / 16 rows to a wave, from a graph: rows of a tile each, 32 2.5 / 10.3, 512 3.8 / 10.5, 1,000 5.5 / 10.5; of one
  // run, 500 3.9 / 2.9, 1,000 5.8 / 3.0.
  const bool few = num_tokens <= kFewTokens;
  const dim3 grid((unsigned)ceil_div(num_tokens, few ? kWaves : kWaves * 16), 2u * num_kv_heads);
  if (few)
    hipLaunchKernelGGL(kv_read_fp8_kernel<1>, grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(kv_read_fp8_kernel<16>, grid, dim3(kThreads), 0, stream, a);
  return launch_status();
}

extern "C" int nvamd_qk_norm_rope_fp8(void *q_out, int64_t q_out_stride, void *k_out, int64_t k_out_stride,
                                      const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v,
                                      int64_t v_stride, const void *q_weight, const void *k_weight,
                                      const int64_t *positions, const float *cos_sin, int max_positions,
                                      void *k_codes, void *k_scales, void *v_codes, void *v_scales, int num_blocks,
                                      int block_size, const int64_t *slot_mapping, int num_tokens, int num_heads,
                                      int num_kv_heads, int head_dim, float eps, hipStream_t stream) {
  if (num_tokens == 0) return NVAMD_OK;
  RowsArgs a;
  const int st = fill_rows_args(a, k, k_stride, v, v_stride, k_codes, k_scales, v_codes, v_scales, slot_mapping,
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

extern "C" size_t nvamd_kv_cache_kept_size_fp8(int num_layers, int num_tokens, int num_kv_heads) {
  if (num_layers <= 0 || num_tokens <= 0 || num_kv_heads <= 0) return 0;
  return (size_t)num_layers * num_tokens * num_kv_heads * kKeptBytes;
}

extern "C" int nvamd_kv_cache_keep_fp8(void *kept, size_t kept_bytes, const void *k_codes, const void *k_scales,
                                       const void *v_codes, const void *v_scales, int num_layers, int num_blocks,
                                       int block_size, const int64_t *slot_mapping, int num_tokens, int num_kv_heads,
                                       int head_dim, hipStream_t stream) {
  return launch_kept<false>(static_cast<u8 *>(kept), kept_bytes, const_cast<void *>(k_codes), const_cast<void *>(k_scales),
                            const_cast<void *>(v_codes), const_cast<void *>(v_scales), num_layers, num_blocks, block_size,
                            slot_mapping, num_tokens, num_kv_heads, head_dim, stream);
}

extern "C" int nvamd_kv_cache_restore_fp8(const void *kept, size_t kept_bytes, void *k_codes, void *k_scales,
                                          void *v_codes, void *v_scales, int num_layers, int num_blocks, int block_size,
                                          int num_tokens, int num_kv_heads, int head_dim, hipStream_t stream) {
  return launch_kept<true>(const_cast<u8 *>(static_cast<const u8 *>(kept)), kept_bytes, k_codes, k_scales, v_codes, v_scales,
                           num_layers, num_blocks, block_size, nullptr, num_tokens, num_kv_heads, head_dim, stream);
}
