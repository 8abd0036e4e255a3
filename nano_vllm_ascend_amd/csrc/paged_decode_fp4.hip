// GQA paged decode attention over the 4-bit KV cache (the counterpart of paged_decode.hip).
//
// For a query token of each sequence and its heads h of kv head g: out = softmax(q . K^T * scale) V over the cached
// context.
//
// Work: partitions of a (sequence, kv head), a workgroup of 8 waves each (decode_quantised.h).
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
#include "decode_quantised.h"
#include "fp4_attention.h"
#include "fp4_rows.h"

namespace nvamd {
namespace {

constexpr int kWaves = 8;
constexpr int kLeastPart = 64 * kWaves;  // tokens of the smallest partition: one step of each wave

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
paged_decode_fp4_kernel(DecodeArgs<Fp4Cache> a, std::conditional_t<FUSED, StepArgs, Nothing> step_args) {
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][GP * kPartFloats];
  __shared__ float s_m[kWaves][GP];
  __shared__ float s_l[kWaves][GP];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hkv = a.num_kv_heads;

  u32 err_bits = 0;
  Part part;
  if (!find_part(a, blockIdx.x, lane, kLeastPart, err_bits, part)) return;
  const int b = part.b, g = part.g, p = part.p, ctx = part.ctx, part_tokens = part.tokens;
  const int n = lane & 15, gq = lane >> 4;
  const int head0 = g * a.q_group + a.q_head0;
  const int32_t *bt_row = a.block_tables + (int64_t)b * a.bt_stride;
  const int bs_mask = (1 << a.bs_log2) - 1;

  i32x8 q_hi, q_lo;
  u32 q_scale;
  if constexpr (FUSED) {
    __shared__ __attribute__((aligned(16))) u32x4 s_q[4][64];
    __shared__ u32 s_q_scale[64];
    step_query(a, step_args, part, head0, w, lane, s_q, s_q_scale, err_bits, q_hi, q_lo, q_scale,
               [&](int64_t slot, const float *row) {
                 if (w != 0) return;
                 store_row(a.cache, step_args, b, g, slot, row, hkv, a.bs_log2, lane, reinterpret_cast<u8 *>(&s_o[0][0]));
                 __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
                 __builtin_amdgcn_s_waitcnt(0);  // before this workgroup's loads of the row
               });
  } else {
    u32x4 x[4];
    load_query(a, b, head0, n, gq, x);
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

  report(a.err, err_bits, lane);
  if constexpr (GP <= 4) l += dpp<kRowRor4>(l);
  if constexpr (GP <= 8) l += dpp<kDppRowRor8>(l);
  finish<kWaves, GP>(a, part, head0, tid, w, o, m, l, s_o, s_m, s_l, s_last);
}

template <typename Step>
int launch(DecodeArgs<Fp4Cache> &a, const Step &s, hipStream_t stream) {
  constexpr bool FUSED = std::is_same_v<Step, StepArgs>;
  return launch_groups(a, [&](auto heads) {
    constexpr int GP = decltype(heads)::value;
    const dim3 grid(decode_items(a)), block(kWaves * 64);
    if (a.bs_log2 >= 6)
      hipLaunchKernelGGL((paged_decode_fp4_kernel<GP, true, FUSED>), grid, block, 0, stream, a, s);
    else
      hipLaunchKernelGGL((paged_decode_fp4_kernel<GP, false, FUSED>), grid, block, 0, stream, a, s);
    return launch_status();
  });
}

Fp4Cache cache_of(const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales) {
  return Fp4Cache{const_cast<u8 *>(static_cast<const u8 *>(k_codes)), const_cast<u8 *>(static_cast<const u8 *>(k_scales)),
                  const_cast<u8 *>(static_cast<const u8 *>(v_codes)), const_cast<u8 *>(static_cast<const u8 *>(v_scales))};
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
  DecodeArgs<Fp4Cache> a;
  const int st = fill_decode_args<kLeastPart>(a, out, out_stride, q, q_stride, cache_of(k_codes, k_scales, v_codes, v_scales),
                                    fp4_cache_ok(k_codes, k_scales, v_codes, v_scales), num_blocks, block_size,
                                    block_tables, bt_stride, bt_width, context_lens, batch, num_heads, num_kv_heads,
                                    head_dim, scale, max_context_len, workspace, workspace_bytes);
  if (st != NVAMD_OK) return st;
  return launch(a, Nothing{}, stream);
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
  DecodeArgs<Fp4Cache> a;
  int st = fill_decode_args<kLeastPart>(a, out, out_stride, q, q_stride, cache_of(k_codes, k_scales, v_codes, v_scales),
                                    fp4_cache_ok(k_codes, k_scales, v_codes, v_scales), num_blocks, block_size,
                                    block_tables, bt_stride, bt_width, context_lens, batch, num_heads, num_kv_heads,
                                    head_dim, scale, max_context_len, workspace, workspace_bytes);
  if (st != NVAMD_OK) return st;
  StepArgs s;
  st = fill_step_args(s, k, k_stride, v, v_stride, q_weight, k_weight, positions, cos_sin, max_positions, eps, slot_mapping,
                      num_blocks, block_size, num_kv_heads);
  if (st != NVAMD_OK) return st;
  return launch(a, s, stream);
}
