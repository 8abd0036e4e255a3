// GQA paged decode attention over the 8-bit KV cache (the counterpart of paged_decode.hip).
//
// For a query token of each sequence and its heads h of kv head g: out = softmax(q . K^T * scale) V over the cached
// context.
//
// Work: partitions of a (sequence, kv head), a workgroup of kWaves waves each (decode_quantised.h).  A wave takes 32
// tokens at a time, two 16-token tiles (n = lane % 16, gq = lane / 16):
//   S^T = K . Q^T  v_mfma_scale_f32_16x16x128_f8f6f4 on the codes as they lie in the cache, A = 16 rows of K under their
//        tiles' scales, B = the heads as 16 columns, in e4m3 twice: a bf16 query is the sum of two e4m3 numbers under a
//        scale for each block (QueryScale), so two products give the scores.  Row 4a + i of product t is token
//        8a + 4t + i of the step: lane (h, gq) then finds the scores of tokens 8 gq + 4t + i of head h in its accumulator
//        of product t;
//   softmax  on up to 8 heads the accumulators' 16 columns are repeats: product 1 moves into the idle columns by DPP, and
//        one lane does 4 scores instead of 8;
//   O^T += V^T . P^T  v_mfma_f32_16x16x32_bf16, A = 16 dims of V^T expanded by v_cvt_scalef32_pk_bf16_fp8 (two tokens of
//        a dim and the tile's scale in one instruction, exact), B = P^T, whose 8 k-slots per lane are tokens 8 gq .. + 7:
//        just what the lane holds.  The cache keeps the 16 tokens of a dim in consecutive bytes: lanes gq and gq ^ 1 load
//        16 bytes each of different dims of the same tile and swap halves, so that every load is whole.
//
// Bound by memory on long contexts, by latency on short ones: a token of a head is 256 bytes and 2 scales.  Measured (8
// kv heads, 16 query heads unless said; the first and the last from a graph): 4 contexts of up to 512 tokens 5.6 us; 32
// of 256..2304 19.3 to 19.7 us (4.4 TB/s); 100 of 2048..4096 102 us (6.1 TB/s); 4 of 8192..40960, 64 query heads, 31.2
// to 31.7 us (5.5 TB/s); 16 of 512..4096, 64 query heads, 15.9 us.  Steps of 64 tokens, a tile to 16 lanes, need
// registers for two waves a SIMD; four waves with half the step hide more of the loads' latency: those 32 contexts took
// 23.7 us, the 100 as long, the 4 longest 2% less.
// The score of a token past the context is replaced by -inf and its values by zero, whatever bytes it holds.
#include "decode_quantised.h"
#include "fp8_attention.h"
#include "fp8_rows.h"

namespace nvamd {
namespace {

constexpr int kWaves = 8;
constexpr int kStep = 32;                // tokens of a wave
constexpr int kLeastPart = 64 * kWaves;  // of the smallest partition: two steps of each wave

// The new token's k (normed and rotated) into its slot, by a wave: every 8 lanes make the row, those of the token keep it.
__device__ __forceinline__ void store_key_row(const Fp8Cache &cache, const StepArgs &s, int b, int g, int64_t slot,
                                              const float *row, int num_kv_heads, int bs_log2, int lane) {
  const int c = lane & 7, tok = lane >> 3, o = (int)(slot & (kFp8Tile - 1));
  const int64_t tile = fp8_tile(slot >> bs_log2, (int)(slot & ((1 << bs_log2) - 1)), g, num_kv_heads, bs_log2);
  const u32 held = o > 0 ? cache.k_scales[tile] : 0u;
  const u16 *p = s.k + b * s.k_stride + g * kHeadDim + 8 * c;
  u32x4 lo = ld16(p), hi = ld16(p + 64);
  float cs[8], sn[8];
  load8(row + 8 * c, cs);
  load8(row + 64 + 8 * c, sn);
  const double rstd = norm_factor(dpp_sum8(sum_squares(lo, hi)), (double)s.eps);
  norm_rope_f64(lo, hi, ld16(s.k_w + 8 * c), ld16(s.k_w + 64 + 8 * c), cs, sn, rstd);
  u32 x[16];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[8 * p + i] = 8 * p + tok == o ? lo[i] : 0u;
      x[8 * p + 4 + i] = 8 * p + tok == o ? hi[i] : 0u;
    }
  store_keys(cache, tile, o, 1, held, tok, c, x);
}
__device__ __forceinline__ void store_value_row(const Fp8Cache &cache, const StepArgs &s, int b, int g, int64_t slot,
                                                int num_kv_heads, int bs_log2, int lane) {
  const int o = (int)(slot & (kFp8Tile - 1));
  const int64_t tile = fp8_tile(slot >> bs_log2, (int)(slot & ((1 << bs_log2) - 1)), g, num_kv_heads, bs_log2);
  u32 held = 0;
  u32x4 old[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
  if (o > 0) {
    const u32x4 *p = reinterpret_cast<const u32x4 *>(cache.v_codes + tile * kFp8TileBytes + 2 * lane * kFp8Tile);
    held = cache.v_scales[tile];
    old[0] = p[0];
    old[1] = p[1];
  }
  const u32 v = *reinterpret_cast<const u32 *>(s.v + b * s.v_stride + g * kHeadDim + 2 * lane);
  u32 x[16];
#pragma unroll
  for (int t = 0; t < 16; ++t) x[t] = t == o ? v : 0u;
  store_values(cache, tile, o, 1, held, old, lane, x);
}

// The query's operand, for every wave of the workgroup: each of the first four makes a quarter, and they meet in LDS.
// (Made whole by every wave, a call takes 0.3 us more: 5.8 us, so 5.5, for 4 contexts of 384..512 tokens.)
struct SharedQuery {
  u32x2 words[2][4][64];  // [hi, lo][8 dims of a lane][lane]
  u32 scale[2][64];       // of the blocks of a lane's dims 16 gq .. and 64 + 16 gq ..
};
__device__ __forceinline__ void shared_query(const DecodeArgs<Fp8Cache> &a, int b, int head0, int w, int lane,
                                             SharedQuery &s, i32x8 &q_hi, i32x8 &q_lo, u32 &q_scale) {
  const int n = lane & 15, gq = lane >> 4;
  if (w < 4) {
    const u16 *qp = a.q + (int64_t)b * a.q_stride + (int64_t)(head0 + min(n, a.q_sub - 1)) * kHeadDim + 16 * gq +
                    64 * (w >> 1);
    const u32x4 x[2] = {ld16(qp), ld16(qp + 8)};
    const u32 top = max(largest(x[0]), largest(x[1]));
    const auto r = __builtin_amdgcn_permlane16_swap(top, top, false, false);  // lanes gq and gq ^ 1 hold a block
    const QueryScale scale = query_scale(max((u32)r[0], (u32)r[1]));
    const u32x4 mine = w & 1 ? x[1] : x[0];
    int hi[2], lo[2];
    split4(mine[0], mine[1], scale.up, hi[0], lo[0]);
    split4(mine[2], mine[3], scale.up, hi[1], lo[1]);
    s.words[0][w][lane] = u32x2{(u32)hi[0], (u32)hi[1]};
    s.words[1][w][lane] = u32x2{(u32)lo[0], (u32)lo[1]};
    if ((w & 1) == 0) s.scale[w >> 1][lane] = scale.byte;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const u32x2 h = s.words[0][j][lane], l = s.words[1][j][lane];
    q_hi[2 * j] = (int)h[0];
    q_hi[2 * j + 1] = (int)h[1];
    q_lo[2 * j] = (int)l[0];
    q_lo[2 * j + 1] = (int)l[1];
  }
  q_scale = s.scale[gq >> 1][(gq & 1) * 32 + n];  // block gq's: of the lanes that hold it
}

// GP: heads that the registers and LDS are laid out for.  WIDE: pages of 32 tokens or more, so that the 32 tokens of a
// wave's step lie in one page, and one entry of the table finds both tiles (on pages of 16: 22.2 us against 21.6 for 32
// contexts of 1000..2000).  FUSED: the norm, the rotation and the store of the step's rows
// first: every workgroup makes its own queries; the one whose partition ends the context stores the new row (one wave the
// key, another the value) and waits for it, so that its loads find it.  Bits as of nvamd_qk_norm_rope_fp8 and this kernel
// after it.
template <int GP, bool WIDE, bool FUSED>
__global__ void __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(4)))
paged_decode_fp8_kernel(DecodeArgs<Fp8Cache> a, std::conditional_t<FUSED, StepArgs, Nothing> step_args) {
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
                 if (w == 0)
                   store_key_row(a.cache, step_args, b, g, slot, row, hkv, a.bs_log2, lane);
                 else if (w == 2)
                   store_value_row(a.cache, step_args, b, g, slot, hkv, a.bs_log2, lane);
                 else
                   return;
                 __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
                 __builtin_amdgcn_s_waitcnt(0);  // before this workgroup's loads of the row
               });
  } else {
    __shared__ __attribute__((aligned(16))) SharedQuery s_q;
    shared_query(a, b, head0, w, lane, s_q, q_hi, q_lo, q_scale);
  }

  // The exponent's reference, the threshold above which it moves; the sum and the numerators at that reference.
  float m = kNoScore, m_thr = kNoScore, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A step's 32 tokens are two tiles: a lane owns a row of K in tile n / 8 and tokens of V in tile gq / 2.  Tiles past the
  // context repeat its last one.
  typedef const __attribute__((address_space(4))) int32_t const_i32;  // nothing writes the table: scalar loads
  const_i32 *bt = (const_i32 *)bt_row;
  const int t_end = min((p + 1) * part_tokens, ctx);
  const int last = (ctx - 1) & ~15;
  // The table's entries are asked for a step before their tiles.
  int entry[2];
  auto look_up = [&](int t0) {
    entry[0] = bt[min(t0, last) >> a.bs_log2];
    if constexpr (!WIDE) entry[1] = bt[min(t0 + 16, last) >> a.bs_log2];
  };
  int tile[2];  // of the pool, scalars
  auto locate = [&](int t0) {
    auto page = [&](int t, int e) {
      if ((unsigned)e >= (unsigned)a.num_blocks) err_bits |= NVAMD_ERR_BLOCK;
      return (int)fp8_tile(min(max(e, 0), a.num_blocks - 1), t & bs_mask, g, hkv, a.bs_log2);  // never leave the pool
    };
    tile[0] = page(t0, entry[0]);
    tile[1] = WIDE ? tile[0] + (t0 + 16 <= last ? 1 : 0) : page(min(t0 + 16, last), entry[1]);
  };
  // Byte `at` of the lane's one of the two tiles: a 32-bit offset from a scalar address where they lie in one page.
  auto in_tile = [&](const u8 *base, bool second, int tile_bytes, u32 at) {
    if constexpr (WIDE) return base + (int64_t)tile[0] * tile_bytes + ((second ? (tile[1] - tile[0]) * tile_bytes : 0) + at);
    else return base + (int64_t)(second ? tile[1] : tile[0]) * tile_bytes + at;
  };
  u32x4 kc[2][2];
  u32x4 vc[4];  // 16 tokens of dims 64 (gq % 2) + 16 j + n
  u32 ks, vs;  // scale bytes of the tile that the lane owns a row of K in, and of its tile of V
  auto load_k = [&]() {
    const u8 *kp = in_tile(a.cache.k_codes, n >= 8, kFp8TileBytes, (2 * (n & 4) + (n & 3)) * 64 + 16 * gq);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      kc[t][0] = load16(kp + 4 * t * 64);
      kc[t][1] = load16(kp + 4 * t * 64 + kFp8TileBytes / 2);
    }
    ks = *in_tile(a.cache.k_scales, n >= 8, 1, 0);
  };
  auto load_v = [&]() {
    const u8 *vp = in_tile(a.cache.v_codes, gq >= 2, kFp8TileBytes, (64 * (gq & 1) + n) * kFp8Tile);
#pragma unroll
    for (int j = 0; j < 4; ++j) vc[j] = load16(vp + 16 * kFp8Tile * j);
    vs = *in_tile(a.cache.v_scales, gq >= 2, 1, 0);
  };

  // K of the next step is asked for as soon as the scores have taken this step's, V as soon as the products have: each
  // is in flight during the other half of the step, without registers of its own.
  auto step = [&](const int t0, const int next) {
    constexpr int NP = GP <= 8 ? 1 : 2;  // accumulators that hold all scores once packed
    f32x4 s[2];
    score(s[0], kc[0], ks, q_hi, q_lo, q_scale);
    score(s[1], kc[1], ks, q_hi, q_lo, q_scale);
    __builtin_amdgcn_sched_barrier(0);
    if (next < t_end) {
      locate(next);
      load_k();
      look_up(next + kStep * kWaves);
    }
    __builtin_amdgcn_sched_barrier(0);

    // Score x * 4 + i of a lane: token 8 gq + 4 (x + n / 8) + i where packed, else 8 gq + 4 x + i.
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if constexpr (NP == 1) s[0][i] = dpp_into<kRowShr8, 0xC>(s[0][i], s[1][i]);
    const int group = NP == 1 ? n >> 3 : 0;
    const int live = t_end - t0 - 8 * gq;  // this lane's tokens that the partition holds
    float cm = kNoScore;
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] *= a.scale_log2e;
    if (t0 + kStep > t_end) {
#pragma unroll
      for (int x = 0; x < NP; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * (x + group) + i >= live) s[x][i] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)  // values past the end weigh nothing, NaNs of stale rows too
        keep_tokens(vc[j], t_end - t0 - 16 * (gq >> 1));
    }
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) cm = fmaxf(cm, s[x][i]);
    if constexpr (NP == 1) cm = fmaxf(cm, dpp<kDppRowRor8>(cm));
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
    // P rounded to bf16 for the matrix cores; the sum takes the same rounded values.  Back in the order of the products,
    // the columns past the heads hold weights of other tokens and give numerators that are never read.
    u32x4 pf;
#pragma unroll
    for (int x = 0; x < NP; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32 pr = pack_bf16x2(fast_exp2(s[x][2 * i] - m), fast_exp2(s[x][2 * i + 1] - m));
        l = dot2_bf16(pr, kBf16PairOne, l);
        pf[2 * x + i] = pr;
        if constexpr (NP == 1) pf[2 + i] = dpp_u32<kRowShl8>(pr);
      }
    const float v_scale = fp8_scale(vs);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // Lanes gq and gq ^ 1 hold 64 dims each of 16 tokens; they swap for all dims of 8 tokens.
      const auto x = __builtin_amdgcn_permlane16_swap(vc[j][0], vc[j][2], false, false);
      const auto y = __builtin_amdgcn_permlane16_swap(vc[j][1], vc[j][3], false, false);
      o[j] = mfma16(expand8(u32x2{(u32)x[0], (u32)y[0]}, v_scale), pf, o[j]);
      o[4 + j] = mfma16(expand8(u32x2{(u32)x[1], (u32)y[1]}, v_scale), pf, o[4 + j]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (next < t_end) load_v();
  };
  if (int t0 = p * part_tokens + kStep * w; t0 < t_end) {
    look_up(t0);
    locate(t0);
    load_k();
    load_v();
    look_up(t0 + kStep * kWaves);
#pragma unroll 1
    do {
      step(t0, t0 + kStep * kWaves);
      t0 += kStep * kWaves;
    } while (t0 < t_end);
  }

  report(a.err, err_bits, lane);
  if constexpr (GP <= 8) l += dpp<kDppRowRor8>(l);
  finish<kWaves, GP>(a, part, head0, tid, w, o, m, l, s_o, s_m, s_l, s_last);
}

template <typename Step>
int launch(DecodeArgs<Fp8Cache> &a, const Step &s, hipStream_t stream) {
  constexpr bool FUSED = std::is_same_v<Step, StepArgs>;
  return launch_groups(a, [&](auto heads) {
    constexpr int GP = decltype(heads)::value;
    const dim3 grid(decode_items(a)), block(kWaves * 64);
    if (a.bs_log2 >= 5)
      hipLaunchKernelGGL((paged_decode_fp8_kernel<GP, true, FUSED>), grid, block, 0, stream, a, s);
    else
      hipLaunchKernelGGL((paged_decode_fp8_kernel<GP, false, FUSED>), grid, block, 0, stream, a, s);
    return launch_status();
  });
}

Fp8Cache cache_of(const void *k_codes, const void *k_scales, const void *v_codes, const void *v_scales) {
  return Fp8Cache{const_cast<u8 *>(static_cast<const u8 *>(k_codes)), const_cast<u8 *>(static_cast<const u8 *>(k_scales)),
                  const_cast<u8 *>(static_cast<const u8 *>(v_codes)), const_cast<u8 *>(static_cast<const u8 *>(v_scales))};
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" int nvamd_paged_decode_fp8(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                      const void *k_codes, const void *k_scales, const void *v_codes,
                                      const void *v_scales, int num_blocks, int block_size,
                                      const int32_t *block_tables, int bt_stride, int bt_width,
                                      const int32_t *context_lens, int batch, int num_heads, int num_kv_heads,
                                      int head_dim, float scale, int max_context_len, void *workspace,
                                      size_t workspace_bytes, hipStream_t stream) {
  if (batch == 0) return NVAMD_OK;
  DecodeArgs<Fp8Cache> a;
  const int st = fill_decode_args<kLeastPart>(a, out, out_stride, q, q_stride, cache_of(k_codes, k_scales, v_codes, v_scales),
                                    fp8_cache_ok(k_codes, k_scales, v_codes, v_scales), num_blocks, block_size,
                                    block_tables, bt_stride, bt_width, context_lens, batch, num_heads, num_kv_heads,
                                    head_dim, scale, max_context_len, workspace, workspace_bytes);
  if (st != NVAMD_OK) return st;
  return launch(a, Nothing{}, stream);
}

extern "C" int nvamd_paged_decode_fused_fp8(void *out, int64_t out_stride, const void *q, int64_t q_stride,
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
  DecodeArgs<Fp8Cache> a;
  int st = fill_decode_args<kLeastPart>(a, out, out_stride, q, q_stride, cache_of(k_codes, k_scales, v_codes, v_scales),
                                    fp8_cache_ok(k_codes, k_scales, v_codes, v_scales), num_blocks, block_size,
                                    block_tables, bt_stride, bt_width, context_lens, batch, num_heads, num_kv_heads,
                                    head_dim, scale, max_context_len, workspace, workspace_bytes);
  if (st != NVAMD_OK) return st;
  StepArgs s;
  st = fill_step_args(s, k, k_stride, v, v_stride, q_weight, k_weight, positions, cos_sin, max_positions, eps, slot_mapping,
                      num_blocks, block_size, num_kv_heads);
  if (st != NVAMD_OK) return st;
  return launch(a, s, stream);
}
