// GQA paged decode attention over the 4-bit KV cache (the counterpart of paged_decode.hip).
//
// For a query token of each sequence and its heads h of kv head g: out = softmax(q . K^T * scale) V over the cached
// context.
//
// Work: a unit (sequence, kv head) is cut into partitions of equal length, a workgroup of 8 waves each.  Every
// workgroup reads the context lengths and derives the same length from them (partition_tokens), so the cut follows the
// contexts themselves and not the bound that the launch was made with.  (A sequence of more than kLeastPart tokens is so
// summed in an order that depends on the sequences beside it.)  A partition leaves (max, sum, numerator) per head in the
// workspace and counts its arrival; the last one of a unit joins them.
//
// A wave takes 64 tokens at a time, four 16-token tiles, one per 16 lanes (gq = lane / 16):
//   S^T = K . Q^T  v_mfma_scale_f32_16x16x128_f8f6f4 on the codes as they lie in the cache, A = 16 rows of K: a lane's
//        16 bytes are one block of a row, under one scale.  B = the heads as 16 columns, in 8 bits twice: a bf16 query
//        is the sum of two e4m3 numbers under a scale for each block (QueryScale), so two products give the scores.
//        That takes the matrix cores as long as four bf16 products, and the vector ALUs no expansion of K.
//        Row 4a + i of product t is token 4t + i of tile a: lane (h, gq) then finds the scores of tile gq's tokens
//        4t .. 4t+3 of head h in its accumulator of product t, that is of all 16 tokens in the four products;
//   softmax  on up to 4 (8) heads the accumulators' 16 columns are mostly repeats: products 1..3 (2, 3) move into the
//        idle columns by DPP, and one lane does 4 (8) scores instead of 16;
//   O^T += V^T . P^T  v_mfma_f32_16x16x32_bf16, A = 16 dims of V^T expanded by v_cvt_scalef32_pk_bf16_fp4 (two values
//        and their scale in one instruction, exact), B = P^T, whose 8 k-slots per lane are tokens 0..7 (8..15) of tile
//        gq: just what the lane holds.  The cache keeps V with 16 tokens of a dim pair in consecutive bytes, so the
//        lane's 16 bytes give both products' operands of two dims: no lane movement.
// The score of a token past the context is replaced by -inf and the scales of its values by zero, whatever bytes it
// holds.
//
// Bound by memory where contexts are long: 100 x U[2048, 4096] tokens of 8 kv heads, 330 MB, 59 .. 63 us (5.2 .. 5.6
// TB/s, part of it from the Infinity Cache; a large copy 5.0); 4 x U[8192, 40960], 91 MB, 21 us.  Below that by what
// every call pays: some 2 us of launch, 1.3 to the first load (contexts, table, query) and 2 to 4 for the join: 32 x
// U[256, 2304], 46 MB, 16 us, 4 x U[1, 512] 6.2.
#include "decode_workspace.h"
#include "fp4_attention.h"
#include "fp4_rows.h"

#include <type_traits>

namespace nvamd {
namespace {

constexpr int kWaves = 8;
constexpr int kHalvesLog2 = 4, kHalves = 2 * kWaves;  // half-waves of a workgroup
static_assert(kHalves == 1 << kHalvesLog2);
constexpr int kLeastPart = 64 * kWaves;  // tokens of the smallest partition: one step of each wave
static_assert(kLeastPart >= kMinPart, "the workspace has records for these partitions");
constexpr int kCus = 256;
constexpr int kMaxHeads = 16;  // query heads of a kv head in one launch: the MFMA's columns

struct DecodeFp4Args {
  u16 *out;
  int64_t out_stride;
  const u16 *q;
  int64_t q_stride;
  Fp4Cache cache;
  const int32_t *block_tables;
  const int32_t *context_lens;
  float *partials;
  unsigned *counters;
  int bt_stride;
  int bt_width;
  int num_blocks;
  int num_kv_heads;
  int bs_log2;
  int max_ctx;
  int max_parts;  // partition records that the workspace holds per unit
  int batch;
  float scale_log2e;
  // Query heads of kv head g: q_group * g + q_head0 + (0 .. q_sub-1).
  int q_group;
  int q_head0;
  int q_sub;
  u32 *err;
};

// The step before the attention, where the kernel makes it too: q, k and v as they are projected.
struct StepArgs {
  const u16 *k;
  int64_t k_stride;
  const u16 *v;
  int64_t v_stride;
  const u16 *q_w;
  const u16 *k_w;
  const int64_t *positions;
  const float *cos_sin;
  const int64_t *slots;
  int64_t num_slots;
  int max_positions;
  float eps;
};
struct Nothing {};

__device__ __forceinline__ double swap_sum16(double v) {  // over lanes l and l ^ 16
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const auto lo = __builtin_amdgcn_permlane16_swap((u32)b, (u32)b, false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap((u32)(b >> 32), (u32)(b >> 32), false, false);
  return __builtin_bit_cast(double, (uint64_t)(u32)hi[0] << 32 | (u32)lo[0]) +
         __builtin_bit_cast(double, (uint64_t)(u32)hi[1] << 32 | (u32)lo[1]);
}
__device__ __forceinline__ double swap_sum32(double v) {  // over lanes l and l ^ 32
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const auto lo = __builtin_amdgcn_permlane32_swap((u32)b, (u32)b, false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap((u32)(b >> 32), (u32)(b >> 32), false, false);
  return __builtin_bit_cast(double, (uint64_t)(u32)hi[0] << 32 | (u32)lo[0]) +
         __builtin_bit_cast(double, (uint64_t)(u32)hi[1] << 32 | (u32)lo[1]);
}
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = e < 4 ? a[e & 3] : b[e & 3];
}

// Norm and rotation of a query row whose lane gq holds dims 16 gq .. +15 and 64 + 16 gq .. +15: what two lanes of 8
// hold elsewhere, summed in the same order, so that the bits are the same.
__device__ __forceinline__ void norm_rope_row(u32x4 (&x)[4], const u16 *weight, const float *row, int gq, double eps) {
  const double pair = sum_squares(x[0], x[2]) + sum_squares(x[1], x[3]);
  const double rstd = norm_factor(swap_sum32(swap_sum16(pair)), eps);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int at = 16 * gq + 8 * j;
    float cs[8], sn[8];
    load8(row + at, cs);
    load8(row + 64 + at, sn);
    norm_rope_f64(x[j], x[2 + j], ld16(weight + at), ld16(weight + 64 + at), cs, sn, rstd);
  }
}

// The new token's k (normed and rotated) and v of a kv head into its slot: lanes 0 .. 7 of a wave the key, 8 .. 15 the
// value, whose bytes go through 512 bytes of LDS.
__device__ __forceinline__ void store_row(const Fp4Cache &cache, const StepArgs &s, int b, int g, int64_t slot,
                                          const float *row, int num_kv_heads, int bs_log2, int lane, u8 *tile) {
  const int c = lane & 7;
  const bool is_key = lane < 8;
  const Fp4Row at = row_at(slot, g, num_kv_heads, bs_log2);
  if (lane < 16) {
    const u16 *p = (is_key ? s.k + b * s.k_stride : s.v + b * s.v_stride) + g * kHeadDim + 8 * c;
    u32x4 lo = ld16(p), hi = ld16(p + 64);
    if (is_key) {
      float cs[8], sn[8];
      load8(row + 8 * c, cs);
      load8(row + 64 + 8 * c, sn);
      const double rstd = norm_factor(dpp_sum8(sum_squares(lo, hi)), (double)s.eps);
      norm_rope_f64(lo, hi, ld16(s.k_w + 8 * c), ld16(s.k_w + 64 + 8 * c), cs, sn, rstd);
      store_key(cache, at, c, lo, hi);
    } else {
      value_bytes(cache, at, true, c, 0, lo, hi, tile);
    }
  }
  wave_lds_fence();
  cache.v_codes[at.tile * kFp4TileBytes + lane * kFp4Tile + at.t] = tile[lane * 8];
}

// Cutting units of `tokens` tokens in all every `length` tokens ends in tokens / length + units / 2 partitions on
// average, and in a whole unit more than the quotient each at most.  The length is chosen for this quotient (share):
//   few units: partitions fill the card once, with one workgroup on each CU while that leaves two per unit, else two.
//     Anything between one and two workgroups per CU has half of the CUs do double the work;
//   many units: twice the mean context.  Units then go round by themselves, and only contexts far longer than the
//     others are cut.
// Measured (us): 4 x U[8192, 40960] at 8 kv heads 20.9 with one workgroup per CU, 22.8 with two, 25.8 where the length
// was the next power of two; 16 x U[512, 4096] at 8 groups of 8 heads 13.9 either way (16.4); 32 x U[256, 2304] at 8 kv
// heads 21.7 uncut, 16.0 with two (16.7); 100 x U[2048, 4096] 63 uncut, 76 cut in two.
__host__ __device__ constexpr int partition_share(int units) {
  const int slots = units * 2 <= kCus ? kCus : 2 * kCus;
  return slots - units / 2 > units / 2 ? slots - units / 2 : units / 2;
}
__device__ __forceinline__ int partition_tokens(u32 tokens, int units) {  // a multiple of 64
  const u32 share = (u32)partition_share(units);
  const u32 len = (tokens + share - 1) / share;
  return max((int)((len + 63) & ~63u), kLeastPart);
}
__host__ __device__ constexpr int max_partitions(int units) { return partition_share(units) + units; }

// GP: heads that the registers and LDS are laid out for (2 heads at 4 x U[1, 512]: 6.2 us as 4, 6.5 as 16; at 100 x
// U[2048, 4096] 63.2, 63.6).  WIDE: pages of 64 tokens or more, so that the 64 tokens of a wave's step lie in one page,
// whose id is a scalar (pages of 128 at 32 x U[256, 2304]: 16.3 us, without 20.8; at 100 x U[2048, 4096] 63, 73).
// FUSED: the norm, the rotation and the store of the step's rows first.  Every workgroup makes its own queries; the one
// whose partition ends the context stores the new row and waits for it, so that its loads find it.  Bits as of
// nvamd_qk_norm_rope_fp4 and this kernel after it, in less time (from a graph over three caches in turn; in brackets this
// kernel alone): 32 x U[256, 2304] 17.4 us for 19.7 (15.8), 16 x U[512, 4096] at 64 heads 15.5 for 17.8 (14.1), 100 x
// U[2048, 4096] 66.2 for 67.4 (62.3), 4 x U[1, 512] 6.8 for 8.0 (4.9).
template <int GP, bool WIDE, bool FUSED>
__global__ void __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(WIDE ? 4 : 3)))
paged_decode_fp4_kernel(DecodeFp4Args a, std::conditional_t<FUSED, StepArgs, Nothing> step_args) {
  constexpr int D = kHeadDim;
  constexpr int HS = kPartFloats;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][GP * HS];
  __shared__ float s_m[kWaves][GP];
  __shared__ float s_l[kWaves][GP];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hkv = a.num_kv_heads, G = a.q_sub;
  const int item = blockIdx.x;

  // The cut, and this workgroup's place in it.
  const int ctx_cap = min(a.max_ctx, a.bt_width << a.bs_log2);
  u32 err_bits = 0;
  u32 total = 0;  // tokens of one kv head, at most 2^31 with all of them
  int ctx0 = 0;   // the context of this lane's sequence of the first 64
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int bi = b0 + lane;
    const int raw = bi < a.batch ? a.context_lens[bi] : 0;
    if (__ballot(raw < 0 || raw > ctx_cap)) err_bits |= NVAMD_ERR_CONTEXT;
    const int ci = min(max(raw, 0), ctx_cap);
    if (b0 == 0) ctx0 = ci;
    total += (u32)__builtin_amdgcn_readlane(wave_incl_scan(bi < a.batch ? max(ci, 1) : 0, lane), 63);
  }
  const int part_tokens = partition_tokens(total * (u32)hkv, a.batch * hkv);
  const float per_part = 1.0f / (float)part_tokens;
  int b = -1, n_parts = 0, first = 0, ctx = 0;
  for (int b0 = 0, base = 0; b0 < a.batch; b0 += 64) {
    const int bi = b0 + lane;
    const int ci = b0 == 0 ? ctx0 : bi < a.batch ? min(max(a.context_lens[bi], 0), ctx_cap) : 0;
    int np = (int)((float)(ci + part_tokens - 1) * per_part);  // off by one at most: both are below 2^24
    np += np * part_tokens < ci ? 1 : (np - 1) * part_tokens >= ci ? -1 : 0;
    np = bi < a.batch ? max(np, 1) : 0;
    const int incl = wave_incl_scan(np, lane);
    const int sum = __builtin_amdgcn_readlane(incl, 63);
    if (item < (base + sum) * hkv) {
      const int sel = __ffsll((unsigned long long)__ballot((base + incl) * hkv > item)) - 1;
      b = b0 + sel;
      n_parts = __builtin_amdgcn_readlane(np, sel);
      first = base + __builtin_amdgcn_readlane(incl, sel) - n_parts;
      ctx = __builtin_amdgcn_readlane(ci, sel);
      break;
    }
    base += sum;
  }
  if (b < 0) return;  // past the last partition
  b = __builtin_amdgcn_readfirstlane(b);
  const int rem = item - first * hkv;
  const int g = rem / n_parts, p = rem - g * n_parts;
  const int n = lane & 15, gq = lane >> 4;
  const int head0 = g * a.q_group + a.q_head0;
  const int32_t *bt_row = a.block_tables + (int64_t)b * a.bt_stride;
  const int bs_mask = (1 << a.bs_log2) - 1;

  // Query operand of head n (columns past the last head repeat it and are never read).
  i32x8 q_hi, q_lo;
  u32 q_scale;
  auto load_query = [&](u32x4 (&x)[4]) {
    const u16 *qp = a.q + (int64_t)b * a.q_stride + (int64_t)(head0 + min(n, G - 1)) * D + 16 * gq;
    x[0] = ld16(qp);
    x[1] = ld16(qp + 8);
    x[2] = ld16(qp + 64);
    x[3] = ld16(qp + 72);
  };
  if constexpr (FUSED) {
    // One wave makes the operand for all (the 64-bit arithmetic of 8 waves at once takes 3 us more), another stores the
    // row.
    __shared__ __attribute__((aligned(16))) u32x4 s_q[4][64];
    __shared__ u32 s_q_scale[64];
    int64_t pos = step_args.positions[b];
    if (pos < 0 || pos >= step_args.max_positions) {  // clamp and report
      err_bits |= NVAMD_ERR_POSITION;
      pos = pos < 0 ? 0 : step_args.max_positions - 1;
    }
    const float *row = step_args.cos_sin + pos * D;
    if (w == 1) {
      u32x4 x[4];
      load_query(x);
      norm_rope_row(x, step_args.q_w, row, gq, (double)step_args.eps);
      s_q_scale[lane] = query_operand(x, gq, q_hi, q_lo);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s_q[j][lane] = u32x4{(u32)q_hi[4 * j], (u32)q_hi[4 * j + 1], (u32)q_hi[4 * j + 2], (u32)q_hi[4 * j + 3]};
        s_q[2 + j][lane] = u32x4{(u32)q_lo[4 * j], (u32)q_lo[4 * j + 1], (u32)q_lo[4 * j + 2], (u32)q_lo[4 * j + 3]};
      }
    } else if (w == 0 && p == n_parts - 1 && a.q_head0 == 0) {
      const int64_t slot = step_args.slots[b];
      if (slot < -1 || slot >= step_args.num_slots) {
        err_bits |= NVAMD_ERR_SLOT;
      } else if (slot >= 0) {
        store_row(a.cache, step_args, b, g, slot, row, hkv, a.bs_log2, lane, reinterpret_cast<u8 *>(&s_o[0][0]));
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_s_waitcnt(0);  // before this workgroup's loads of the row
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 h = s_q[j][lane], l = s_q[2 + j][lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q_hi[4 * j + i] = (int)h[i];
        q_lo[4 * j + i] = (int)l[i];
      }
    }
    q_scale = s_q_scale[lane];
  } else {
    u32x4 x[4];
    load_query(x);
    q_scale = query_operand(x, gq, q_hi, q_lo);
  }

  // The exponent's reference, the threshold above which it moves; the sum and the numerators at that reference.
  float m = kNoScore, m_thr = kNoScore, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A step's 64 tokens are the four tiles t0 .. t0+63.  The tile of each 16 lanes, as row owners of K (tile n / 4) and
  // as token owners of V (tile gq); tiles past the context repeat its last one.
  typedef const __attribute__((address_space(4))) int32_t const_i32;  // nothing writes the table: scalar loads
  const_i32 *bt = (const_i32 *)bt_row;
  const int t_end = min((p + 1) * part_tokens, ctx);
  const int last = (ctx - 1) & ~15;
  // The table's entries are asked for a step before their tiles.
  int entry_k = 0, entry_v = 0;
  auto look_up = [&](int t0) {
    if constexpr (WIDE) {
      entry_k = bt[min(t0, last) >> a.bs_log2];
    } else {
      entry_k = bt_row[min(t0 + 16 * (n >> 2), last) >> a.bs_log2];
      entry_v = bt_row[min(t0 + 16 * gq, last) >> a.bs_log2];
    }
  };
  // Where the next tiles lie: a tile that the lanes share (a scalar, WIDE) and each lane's tiles past it.
  int tile0 = 0;
  u32 k_tile = 0, v_tile = 0;
  auto locate = [&](int t0) {
    auto page = [&](int t, int e) {
      if ((unsigned)e >= (unsigned)a.num_blocks) err_bits |= NVAMD_ERR_BLOCK;
      return (int)fp4_tile(min(max(e, 0), a.num_blocks - 1), t & bs_mask, g, hkv, a.bs_log2);  // never leave the pool
    };
    if constexpr (WIDE) {
      tile0 = page(t0, entry_k);
      const int tiles = (last - t0) >> 4;  // 0 .. 3, or more: the last tile that exists
      k_tile = min(n >> 2, tiles);
      v_tile = min(gq, tiles);
    } else {
      k_tile = page(min(t0 + 16 * (n >> 2), last), entry_k);
      v_tile = page(min(t0 + 16 * gq, last), entry_v);
    }
  };
  // Byte `at` of tile `tile0 + tile`: a 32-bit offset from a scalar address where the tiles lie in one page.
  auto in_tiles = [&](const u8 *base, u32 tile, int tile_bytes, u32 at) {
    if constexpr (WIDE) return base + (int64_t)tile0 * tile_bytes + (tile * tile_bytes + at);
    else return base + (int64_t)tile * tile_bytes + at;
  };
  u32x4 kc[4], vc[4];
  u32 ks, vs;
  auto load_k = [&]() {
    const u8 *kp = in_tiles(a.cache.k_codes, k_tile, kFp4TileBytes, (n & 3) * kFp4RowBytes + 16 * gq);
#pragma unroll
    for (int t = 0; t < 4; ++t) kc[t] = load16(kp + 4 * t * kFp4RowBytes);
    ks = *reinterpret_cast<const u32 *>(in_tiles(a.cache.k_scales, k_tile, kFp4TileScales, fp4_key_scale_at(n & 3, gq)));
  };
  auto load_v = [&]() {
    const u8 *vp = in_tiles(a.cache.v_codes, v_tile, kFp4TileBytes, 16 * n);
#pragma unroll
    for (int q = 0; q < 4; ++q) vc[q] = load16(vp + 256 * q);
    // the 16 lanes of a tile share its 64 scale bytes out: lane n has those of block n / 4, tokens 4 (n % 4) .. +3
    vs = *reinterpret_cast<const u32 *>(in_tiles(a.cache.v_scales, v_tile, kFp4TileScales, 4 * n));
  };

  // K of the next step is asked for as soon as the scores have taken this step's, V as soon as the products have: each
  // is in flight during the other half of the step, without registers of its own.
  auto step = [&](const int t0, const int next) {
    constexpr int NP = GP <= 4 ? 1 : GP <= 8 ? 2 : 4;  // accumulators that hold all scores once packed
    f32x4 s[4];
    score<0>(s[0], kc[0], ks, q_hi, q_lo, q_scale);
    score<1>(s[1], kc[1], ks, q_hi, q_lo, q_scale);
    score<2>(s[2], kc[2], ks, q_hi, q_lo, q_scale);
    score<3>(s[3], kc[3], ks, q_hi, q_lo, q_scale);
    __builtin_amdgcn_sched_barrier(0);
    if (next < t_end) {
      locate(next);
      load_k();
      look_up(next + 64 * kWaves);
    }
    __builtin_amdgcn_sched_barrier(0);

    // Score x * 4 + i of a lane: token 16 gq + 4 (x + NP * its column group) + i, the group being n / (4 NP).
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (NP == 1) {
        s[0][i] = dpp_into<kRowShr4, 0x2>(s[0][i], s[1][i]);
        s[0][i] = dpp_into<kRowShr8, 0x4>(s[0][i], s[2][i]);
        s[0][i] = dpp_into<kRowShr12, 0x8>(s[0][i], s[3][i]);
      } else if constexpr (NP == 2) {
        s[0][i] = dpp_into<kRowShr8, 0xC>(s[0][i], s[2][i]);
        s[1][i] = dpp_into<kRowShr8, 0xC>(s[1][i], s[3][i]);
      }
    }
    const int group = NP == 4 ? 0 : n / (4 * NP);
    const int live = t_end - t0 - 16 * gq;  // this lane's tile's tokens that the partition holds
    float cm = kNoScore;
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] *= a.scale_log2e;
    if (t0 + 64 > t_end) {
#pragma unroll
      for (int x = 0; x < NP; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * (x + NP * group) + i >= live) s[x][i] = -INFINITY;
      vs = keep_bytes(vs, live - 4 * (n & 3));  // values past the partition's end weigh nothing, NaNs of stale rows too
    }
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) cm = fmaxf(cm, s[x][i]);
    if constexpr (NP == 1) cm = fmaxf(cm, dpp<kRowRor4>(cm));
    if constexpr (NP <= 2) cm = fmaxf(cm, dpp<kDppRowRor8>(cm));
    cm = max_over_quarters(cm);
    // Lazy rescale: the weights stay below 2^8 and the numerators are scaled only where some head's reference moves.
    if (__builtin_amdgcn_ballot_w64(cm > m_thr) != 0) {
      const bool up = cm > m_thr;
      const float alpha = up ? fast_exp2(m - cm) : 1.f;
      if (up) {
        m = cm;
        m_thr = cm + kRescaleLog2;
      }
      l *= alpha;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= alpha;
    }
    // P rounded to bf16 for the matrix cores; the sum takes the same rounded values.  The result is then off by 1.9e-3 to
    // 2.3e-3 of its size where its own rounding is 1.65e-3.  A second bf16 term of P, which the bf16 cache's kernel has
    // at no cost, takes 20 registers more here, with them one of the two workgroups of a CU, and the products twice:
    // 100 x U[2048, 4096] 73 us for 62, 32 x U[256, 2304] 20.8 for 16.2.  Back in the order of the products, the columns
    // past the heads hold weights of other tokens and give numerators that are never read.
    u32x4 pf[2];
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32 pr = pack_bf16x2(fast_exp2(s[x][2 * i] - m), fast_exp2(s[x][2 * i + 1] - m));
        l = dot2_bf16(pr, kBf16PairOne, l);
        pf[x >> 1][2 * (x & 1) + i] = pr;
        if constexpr (NP == 1) {
          pf[0][2 + i] = dpp_u32<kRowShl4>(pr);
          pf[1][i] = dpp_u32<kRowShl8>(pr);
          pf[1][2 + i] = dpp_u32<kRowShl12>(pr);
        } else if constexpr (NP == 2) {
          pf[1][2 * x + i] = dpp_u32<kRowShl8>(pr);
        }
      }
    add_values<0>(o, vc, vs, pf);
    add_values<1>(o, vc, vs, pf);
    add_values<2>(o, vc, vs, pf);
    add_values<3>(o, vc, vs, pf);
    __builtin_amdgcn_sched_barrier(0);
    if (next < t_end) load_v();
  };
  if (int t0 = p * part_tokens + 64 * w; t0 < t_end) {
    look_up(t0);
    locate(t0);
    load_k();
    load_v();
    look_up(t0 + 64 * kWaves);
#pragma unroll 1
    do {
      step(t0, t0 + 64 * kWaves);
      t0 += 64 * kWaves;
    } while (t0 < t_end);
  }

  {
    u32 bits = err_bits;  // a lane's own bits: any lane's count
#pragma unroll
    for (u32 bit = NVAMD_ERR_SLOT; bit <= NVAMD_ERR_BLOCK; bit <<= 1)
      if (__ballot(bits & bit) && lane == 0) flag_index_error(a.err, bit);
  }

  // Register i of o[e] is dim 16 e + 4 gq + i of head n.
  if constexpr (GP <= 4) l += dpp<kRowRor4>(l);
  if constexpr (GP <= 8) l += dpp<kDppRowRor8>(l);
  l = sum_over_quarters(l);
  if (n < G) {
#pragma unroll
    for (int e = 0; e < 8; ++e) *reinterpret_cast<f32x4 *>(&s_o[w][n * HS + 16 * e + 4 * gq]) = o[e];
    if (gq == 0) {
      s_m[w][n] = m;
      s_l[w][n] = l;
    }
  }
  __syncthreads();

  // The waves' results meet: a half-wave takes heads hw, hw + kHalves, its lane dims 4 dl .. 4 dl + 3.
  constexpr int HP = (GP + kHalves - 1) / kHalves;
  const int hw = tid >> 5, dl = lane & 31;
  f32x4 acc[HP];
  float mx[HP], ls[HP];
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = min(hw + kHalves * k, G - 1);
    float M = s_m[0][h];
#pragma unroll
    for (int x = 1; x < kWaves; ++x) M = fmaxf(M, s_m[x][h]);
    acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    ls[k] = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      const float f = fast_exp2(s_m[x][h] - M);
      acc[k] += f * *reinterpret_cast<const f32x4 *>(&s_o[x][h * HS + 4 * dl]);
      ls[k] += f * s_l[x][h];
    }
    mx[k] = M;
  }
  auto write_out = [&](int h, f32x4 v, float den) {
    const float inv = den > 0.f ? 1.f / den : 0.f;
    *reinterpret_cast<u32x2 *>(a.out + (int64_t)b * a.out_stride + (int64_t)(head0 + h) * D + 4 * dl) =
        u32x2{pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv)};
  };
  if (n_parts == 1) {
#pragma unroll
    for (int k = 0; k < HP; ++k)
      if (hw + kHalves * k < G) write_out(hw + kHalves * k, acc[k], ls[k]);
    return;
  }

  // Publish this partition's record past the caches that are not coherent, then count it.
  const int rec_bytes = G * HS * (int)sizeof(float);
  float *base = a.partials + ((int64_t)b * hkv + g) * a.max_parts * (G * HS);
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(base, 0, n_parts * rec_bytes, kBufferRsrcWord3);
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = hw + kHalves * k;
    if (h < G) {
      const int off = p * rec_bytes + h * (HS * (int)sizeof(float));
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[k]), rsrc, off + 16 + 16 * dl, 0,
                                             kCachePolicyAgent);
      if (dl == 0)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(mx[k]), __float_as_uint(ls[k])}, rsrc, off, 0,
                                              kCachePolicyAgent);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // keep the stores above the wait
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();  // every wave's stores are acknowledged
  if (tid == 0)
    s_last = (int)__builtin_amdgcn_atomic_inc32(a.counters + (int64_t)b * hkv + g, (unsigned)(n_parts - 1),
                                                __ATOMIC_RELAXED, "agent");
  __syncthreads();
  if (s_last != n_parts - 1) return;

  // The last arriver joins the partitions.  The heads share out the half-waves: `split` of them take a head, each every
  // split-th run of kRun partitions, whose records it loads together; their shares meet in LDS, in order.
  constexpr int kRun = 8;
  const int slots_log2 = min(G <= 1 ? 0 : 32 - __builtin_clz(G - 1), kHalvesLog2);
  const int split = kHalves >> slots_log2;
  const int sp = hw >> slots_log2;
  float *so = &s_o[0][0];  // free: every wave has passed two barriers since it read them
#pragma unroll 1
  for (int h = hw & ((1 << slots_log2) - 1); h < G; h += kHalves) {
    const int hoff = h * (HS * (int)sizeof(float));
    float M = kNoScore, den = 0.f;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int y0 = sp * kRun; y0 < n_parts; y0 += split * kRun) {
      u32x2 ml[kRun];
      u32x4 v[kRun];
#pragma unroll
      for (int y = 0; y < kRun; ++y) {  // past n_parts: zeros without a memory access
        ml[y] = __builtin_amdgcn_raw_buffer_load_b64(rsrc, (y0 + y) * rec_bytes + hoff, 0, kCachePolicyAgent);
        v[y] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (y0 + y) * rec_bytes + hoff + 16 + 16 * dl, 0,
                                                     kCachePolicyAgent);
      }
      float up = M;
#pragma unroll
      for (int y = 0; y < kRun; ++y)
        if (y0 + y < n_parts) up = fmaxf(up, __uint_as_float(ml[y][0]));
      const float f_old = fast_exp2(M - up);
      num *= f_old;
      den *= f_old;
#pragma unroll
      for (int y = 0; y < kRun; ++y) {
        const float f = y0 + y < n_parts ? fast_exp2(__uint_as_float(ml[y][0]) - up) : 0.f;
        num += f * __builtin_bit_cast(f32x4, v[y]);
        den += f * __uint_as_float(ml[y][1]);
      }
      M = up;
    }
    if (split > 1) {  // then every half-wave has one head at most
      *reinterpret_cast<f32x4 *>(so + hw * HS + 4 + 4 * dl) = num;
      if (dl == 0) *reinterpret_cast<u32x2 *>(so + hw * HS) = u32x2{__float_as_uint(M), __float_as_uint(den)};
    } else {
      write_out(h, num, den);
    }
  }
  if (split > 1) {
    __syncthreads();
    if (sp == 0 && hw < G) {
      float M = kNoScore, den = 0.f;
      f32x4 num = {0.f, 0.f, 0.f, 0.f};
      for (int x = 0; x < split; ++x) M = fmaxf(M, so[((x << slots_log2) + hw) * HS]);
      for (int x = 0; x < split; ++x) {
        const float *r = so + ((x << slots_log2) + hw) * HS;
        const float f = fast_exp2(r[0] - M);
        num += f * *reinterpret_cast<const f32x4 *>(r + 4 + 4 * dl);
        den += f * r[1];
      }
      write_out(hw, num, den);
    }
  }
}

template <int GP, typename Step>
int launch(const DecodeFp4Args &a, const Step &s, hipStream_t stream) {
  constexpr bool FUSED = std::is_same_v<Step, StepArgs>;
  static_assert(kWaves * GP >= kHalves, "the shares of a join fit s_o");
  const int units = a.batch * a.num_kv_heads;  // <= kCounterSlots
  const int64_t items = min((int64_t)units * a.max_parts, (int64_t)max_partitions(units));
  const dim3 grid((unsigned)items), block(kWaves * 64);
  if (a.bs_log2 >= 6)
    hipLaunchKernelGGL((paged_decode_fp4_kernel<GP, true, FUSED>), grid, block, 0, stream, a, s);
  else
    hipLaunchKernelGGL((paged_decode_fp4_kernel<GP, false, FUSED>), grid, block, 0, stream, a, s);
  return launch_status();
}

template <typename Step>
int launch_groups(DecodeFp4Args &a, const Step &s, hipStream_t stream) {
  for (a.q_head0 = 0; a.q_head0 < a.q_group; a.q_head0 += a.q_sub) {
    a.q_sub = min(a.q_group - a.q_head0, kMaxHeads);
    const int st = a.q_sub <= 4   ? launch<4>(a, s, stream)
                   : a.q_sub <= 8 ? launch<8>(a, s, stream)
                                  : launch<16>(a, s, stream);
    if (st != NVAMD_OK) return st;
  }
  return NVAMD_OK;
}

// Checks shared by the entry points; fills what they share.
int fill_decode_args(DecodeFp4Args &a, void *out, int64_t out_stride, const void *q, int64_t q_stride,
                     const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales,
                     int num_blocks, int block_size,
                     const int32_t *block_tables, int bt_stride, int bt_width, const int32_t *context_lens, int batch,
                     int num_heads, int num_kv_heads, int head_dim, float scale, int max_context_len, void *workspace,
                     size_t workspace_bytes) {
  if (!out || !q || !fp4_cache_ok(k_codes, k_scales, v_codes, v_scales) || !block_tables || !context_lens)
    return NVAMD_EINVAL;
  if (batch < 0 || num_blocks <= 0 || num_kv_heads <= 0 || num_heads <= 0 || bt_width <= 0 || bt_stride < bt_width ||
      max_context_len <= 0 || num_heads % num_kv_heads != 0)
    return NVAMD_EINVAL;
  const int bs_log2 = log2_exact(block_size);
  if (head_dim != kHeadDim || bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!aligned16(q) || !aligned16(out) || q_stride % 8 != 0 || out_stride % 8 != 0 ||
      q_stride < (int64_t)num_heads * head_dim || out_stride < (int64_t)num_heads * head_dim)
    return NVAMD_EINVAL;
  if ((int64_t)batch * num_kv_heads > kCounterSlots || batch > 65535 || max_context_len > kMaxContext ||
      ((int64_t)bt_width << bs_log2) > 0x7fffffff || (((int64_t)num_blocks * num_kv_heads) << bs_log2) >> 4 > 0x7fffffff)
    return NVAMD_EUNSUPPORTED;
  if (!workspace ||
      workspace_bytes < decode_workspace_bytes(batch, num_heads, num_kv_heads, max_context_len))
    return NVAMD_EWORKSPACE;
  if (!aligned16(workspace)) return NVAMD_EINVAL;

  a = {};
  a.out = static_cast<u16 *>(out);
  a.out_stride = out_stride;
  a.q = static_cast<const u16 *>(q);
  a.q_stride = q_stride;
  a.cache = Fp4Cache{const_cast<u8 *>(static_cast<const u8 *>(k_codes)),
                     const_cast<u8 *>(static_cast<const u8 *>(k_scales)),
                     const_cast<u8 *>(static_cast<const u8 *>(v_codes)),
                     const_cast<u8 *>(static_cast<const u8 *>(v_scales))};
  a.block_tables = block_tables;
  a.context_lens = context_lens;
  a.counters = static_cast<unsigned *>(workspace);
  a.partials = reinterpret_cast<float *>(static_cast<char *>(workspace) + kCounterBytes);
  a.bt_stride = bt_stride;
  a.bt_width = bt_width;
  a.num_blocks = num_blocks;
  a.num_kv_heads = num_kv_heads;
  a.bs_log2 = bs_log2;
  a.max_ctx = max_context_len;
  a.max_parts = ceil_div(max_context_len, kLeastPart);
  a.batch = batch;
  a.scale_log2e = scale * kLog2e;
  a.q_group = num_heads / num_kv_heads;
  a.err = index_error_word();
  return NVAMD_OK;
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" int nvamd_paged_decode_fp4(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                      const void *k_codes, const void *k_scales, const void *v_codes,
                                      const void *v_scales, int num_blocks, int block_size,
                                      const int32_t *block_tables, int bt_stride, int bt_width,
                                      const int32_t *context_lens, int batch, int num_heads, int num_kv_heads,
                                      int head_dim, float scale, int max_context_len, void *workspace,
                                      size_t workspace_bytes, hipStream_t stream) {
  if (batch == 0) return NVAMD_OK;
  DecodeFp4Args a;
  const int st = fill_decode_args(a, out, out_stride, q, q_stride, k_codes, k_scales, v_codes, v_scales, num_blocks,
                                  block_size, block_tables, bt_stride, bt_width, context_lens, batch, num_heads,
                                  num_kv_heads, head_dim, scale, max_context_len, workspace, workspace_bytes);
  if (st != NVAMD_OK) return st;
  return launch_groups(a, Nothing{}, stream);
}

extern "C" int nvamd_paged_decode_fused_fp4(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                            const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                                            const void *q_weight, const void *k_weight, const int64_t *positions,
                                            const float *cos_sin, int max_positions, float eps, void *k_codes,
                                            void *k_scales, void *v_codes, void *v_scales, int num_blocks,
                                            int block_size, const int64_t *slot_mapping, const int32_t *block_tables,
                                            int bt_stride, int bt_width, const int32_t *context_lens, int batch,
                                            int num_heads, int num_kv_heads, int head_dim, float scale,
                                            int max_context_len, void *workspace, size_t workspace_bytes,
                                            hipStream_t stream) {
  if (batch == 0) return NVAMD_OK;
  DecodeFp4Args a;
  const int st = fill_decode_args(a, out, out_stride, q, q_stride, k_codes, k_scales, v_codes, v_scales, num_blocks,
                                  block_size, block_tables, bt_stride, bt_width, context_lens, batch, num_heads,
                                  num_kv_heads, head_dim, scale, max_context_len, workspace, workspace_bytes);
  if (st != NVAMD_OK) return st;
  const int64_t row = (int64_t)num_kv_heads * kHeadDim;
  if (!k || !v || !aligned16(k) || !aligned16(v) || k_stride % 8 || v_stride % 8 || k_stride < row || v_stride < row ||
      !q_weight || !k_weight || !aligned16(q_weight) || !aligned16(k_weight) || !positions || !cos_sin ||
      !aligned16(cos_sin) || max_positions <= 0 || !slot_mapping)
    return NVAMD_EINVAL;
  StepArgs s;
  s.k = static_cast<const u16 *>(k);
  s.k_stride = k_stride;
  s.v = static_cast<const u16 *>(v);
  s.v_stride = v_stride;
  s.q_w = static_cast<const u16 *>(q_weight);
  s.k_w = static_cast<const u16 *>(k_weight);
  s.positions = positions;
  s.cos_sin = cos_sin;
  s.slots = slot_mapping;
  s.num_slots = (int64_t)num_blocks * block_size;
  s.max_positions = max_positions;
  s.eps = eps;
  return launch_groups(a, s, stream);
}
