// Causal prefill attention over the 8-bit paged KV cache (the counterpart of prefill.hip's paged route): the queries are
// the last q_len positions of a context of kv_len, query row r sees keys 0 .. kv_len - q_len + r, all of them in the
// cache.  Rows, ways out and the choice of kernel are shared with the 4-bit cache's (prefill_quantised.h).
//
// In all kernels
//   S^T = K . Q^T   v_mfma_scale_f32_*_f8f6f4 on the codes as they lie in the cache, under their tiles' scales: a lane loads
//        its dims of a key straight into the operand, and the row comes as two e4m3 numbers per value.  No expansion of
//        K, and none of it in LDS;
//   O^T += V^T . P^T   v_mfma_f32_*_bf16 on V expanded by v_cvt_scalef32_pk_bf16_fp8, exact.
// The rows of K are taken in such an order that a lane's registers of S^T are the consecutive keys that its operand of
// P^T needs: a repack in registers.  Three kernels, which differ in how many rows share an expansion of V:
//
// Tiles (the card is full).  Workgroup = 4 waves = 128 rows, a wave 32 of them, tiles of 32 keys.  The workgroup
//   expands a tile of V once, to bf16 operands in LDS (every access is 64 lanes x 16 consecutive bytes): a wave takes 32
//   dims, a lane a dim of 16 tokens.  Key 16a + 8b + 4c + x sits in row 16a + 8c + 4b + x of K.  K of the next tile loads
//   as the scores have taken this one's, V's codes are two tiles ahead, V's operands one (two stages, one barrier a tile).
// Strips (one long prompt, or several short ones).  Workgroup = 4 waves = 32 rows, a wave every fourth 32 keys; no
//   barrier in the loop, the waves' results meet in LDS.  A lane expands 16 tokens of a dim straight into operands.
// Few rows (a chat's next turn).  Workgroup = 8 waves = 16 rows, a wave every eighth 64 keys, as in
//   paged_decode_fp8.hip with rows in the place of heads and a last key for each row.  On long contexts the keys are cut as
//   well.
//
// Bounds and figures (16 query heads on 8 kv heads unless said).  Tiles: bound by the issue of instructions, since
// matrix products and softmax (a tile of 32 keys: 12 products, some 75 vector instructions, 16 of them exponentials) do
// not overlap, neither a wave's own nor, by the counters, those of different waves.  32 prompts of 512..2,048 tokens on
// 1,152 cached take 655 to 664 us (929 to 941 TFLOP/s) at three waves a SIMD, 842 at two; 40 query heads, 2 x U[3000,
// 4000] on 4,096 cached 940 to 947 us (1,057 TFLOP/s).  Of the first, 12 us are the maximum that is only looked for
// where it matters (weigh_scores), 25 V's operands, which are on their way from LDS before they are needed, and 10 the
// fewer registers and instructions of the pages' bookkeeping.  One barrier for two tiles, with four stages, gives 654:
// not worth it.
// Strips: 1 x 4,000 on 4,096 217 us (925 TFLOP/s), 8 x 1..64 on 1,040 13.4 us.  Few short rows are bound by one step after
// another in a wave, some 0.6 us, whose products, softmax and expansion wait for one another: loads two steps ahead (14.5)
// and eight waves to a strip (13.6) gain nothing.  The registers of the 8-bit operands leave room for two waves a SIMD, and
// strips and few rows take as long as the 4-bit cache's kernels at three.
//
// Weights are rounded to bf16 once for the matrix cores, and the sums take the rounded values, as in the other caches'
// prefill.
//
// A value that reads as NaN must reach the rows that see its key and no others, though masked rows multiply it by a weight
// of zero.  Where every row of a workgroup sees every key of a tile the products do that; in the others, which cross the
// diagonal, such values enter the products as zeros, and the rows that see the key get the NaN afterwards.
#include "fp8_attention.h"
#include "prefill_quantised.h"

namespace nvamd {
namespace {

// 0x80 in the bytes that are codes of NaN (127 and 255).
__device__ __forceinline__ u32 nan_bytes(u32 codes) { return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ u32 without(u32 codes, u32 nans) { return codes & ~((nans >> 7) * 0xffu); }
// Replaces a dim's NaNs by zeros and returns their tokens, a bit each.
__device__ __forceinline__ u32 take_nans(u32x4 &codes) {
  u32 tokens = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32 bad = nan_bytes(codes[i]);
    codes[i] = without(codes[i], bad);
    tokens |= ((bad >> 7 & 1u) | (bad >> 14 & 2u) | (bad >> 21 & 4u) | (bad >> 28 & 8u)) << (4 * i);
  }
  return tokens;
}

// Weights of a row's 16 keys as bf16 pairs, in the order of the scores; their sum joins l_run.  The exponent's reference is
// 2^kHeadroom above a maximum of the row, so that a weight of 2 or more, that is a set top bit of its exponent, says that a
// score exceeds that maximum by 2^8: the maximum is looked for only then, and the reference, the numerators and the sum
// follow it.  (An infinity or a NaN is one of these; so is the first score that a row sees.)
constexpr float kHeadroom = kRescaleLog2 - 1.f;
__device__ __forceinline__ void weigh_scores(const f32x16 &sc, float scale, f32x16 (&acc)[4], float &neg_ref, float &l_run,
                                             u32x4 (&pf)[2]) {
  auto weights = [&]() {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        pf[hh][e] = pack_bf16x2(fast_exp2(fmaf(sc[8 * hh + 2 * e], scale, neg_ref)),
                                fast_exp2(fmaf(sc[8 * hh + 2 * e + 1], scale, neg_ref)));
  };
  weights();
  u32 seen = 0;
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int e = 0; e < 4; ++e) seen |= pf[hh][e];
  seen &= 0x40004000u;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(seen != 0) != 0, 0)) {
    const auto both = __builtin_amdgcn_permlane32_swap(seen, seen, false, false);  // lanes l and l ^ 32 hold a row
    const bool up = ((u32)both[0] | (u32)both[1]) != 0;                            // whatever the other rows do
    float tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, sc[i]);
    tmax = max_xor32(tmax) * scale;
    const float alpha = up ? fast_exp2(-neg_ref - tmax - kHeadroom) : 1.f;
    if (up) neg_ref = -tmax - kHeadroom;
    l_run *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
    weights();
  }
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int e = 0; e < 4; ++e) l_run = dot2_bf16(pf[hh][e], kBf16PairOne, l_run);  // both rounded values of the pair
}

// ------------------------------------------------------------------------------------------ tiles

// 64 dims: lane (n, half) gives dims 16 half .. +15 and 32 + 16 half .. +15 of row and column n, the scale byte of its row
// and that of block `half` of its column.
template <int BYTE = 0>  // of q_scale
__device__ __forceinline__ f32x16 mfma32_fp8_fp8(const u32x4 (&k)[2], u32 k_scale, i32x8 q, u32 q_scale, f32x16 c) {
  const i32x8 codes = {(int)k[0][0], (int)k[0][1], (int)k[0][2], (int)k[0][3],
                       (int)k[1][0], (int)k[1][1], (int)k[1][2], (int)k[1][3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes, q, c, 0, 0, 0, (int)k_scale, BYTE, (int)q_scale);
}

struct Stage {
  u32x4 v[2][4][64];  // [16-key step][32-dim block][lane]
  u32 any[4];         // on the diagonal, [wave that expanded them]: whether any of its values read as NaN,
  u32 nan[4][32][2];  // and which: of each dim, a bit for each of the 16 tokens of a step
};
__global__ void __launch_bounds__(kTileWaves * 64) __attribute__((amdgpu_waves_per_eu(3)))
prefill_fp8_kernel(PrefillArgs<Fp8Cache> a) {
  __shared__ __attribute__((aligned(16))) u8 s_mem[2 * sizeof(Stage) > kTurnBytes ? 2 * sizeof(Stage) : kTurnBytes];
  Stage *stages = reinterpret_cast<Stage *>(s_mem);

  Rows rows;
  if (!find_rows(a, kTileRows, blockIdx.y, rows)) return;
  const int g = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, n = lane & 31;
  const int kv_len = rows.kv_len;
  const int r0 = rows.first + 32 * w;  // the wave's first row
  const int row = min(r0 + n, rows.rows - 1);
  auto last_seen = [&]() {  // by this lane's row; made anew where it is needed: it would hold a register through the loop
    u32 lanes = ~0u;
    asm volatile("" : "+s"(lanes));
    const int r = min(r0 + (int)(__builtin_amdgcn_mbcnt_hi(lanes, __builtin_amdgcn_mbcnt_lo(lanes, 0)) & 31), rows.rows - 1);
    return min(rows.offset + r / a.group, kv_len - 1);
  };
  const int wave_first = rows.offset + r0 / a.group;           // the last key that the wave's first row sees
  const int wave_last = rows.offset + min(r0 + 31, rows.rows - 1) / a.group;
  const int end_row = min(rows.first + kTileRows, rows.rows) - 1;
  const int keys = min(kv_len, rows.offset + end_row / a.group + 1);  // that the workgroup needs
  const int n_tiles = keys > 0 ? ceil_div(keys, kBK) : 0;

  i32x8 q_hi[2], q_lo[2];
  u32 q_scale[2];
  load_query(a, rows, row, g, half, q_hi, q_lo, q_scale);
  const u32 q_scales = q_scale[0] | q_scale[1] << 8;

  f32x16 acc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
  float neg_ref = -kNoScore, l_run = 0.f;  // minus the exponent's reference; the sum at that reference

  // The two 16-token tiles of each tile of keys (past the keys: their last one), looked up a tile ahead.
  const_i32 *bt = (const_i32 *)(a.block_tables + (int64_t)blockIdx.z * a.bt_stride);
  const int last_tile = max(kv_len - 1, 0) & ~15;
  int entry[2];
  auto look_up = [&](int t) {
#pragma unroll
    for (int x = 0; x < 2; ++x) entry[x] = bt[min(t * kBK + 16 * x, last_tile) >> a.bs_log2];
  };
  int tile[2];  // of the latest tile that was located
  bool outside = false;  // some page; reported at the end
  auto locate = [&](int t) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      outside |= (unsigned)entry[x] >= (unsigned)a.num_blocks;
      tile[x] = tile_of(a, entry[x], min(t * kBK + 16 * x, last_tile), g, false);
    }
  };
  // K: key 16a + 8b + 4c + x of the tile in row n = 16a + 8c + 4b + x.
  const int k_token = (n & 3) | ((n & 8) >> 1) | ((n & 4) << 1);  // of its 16-token tile, n / 16
  u32x4 kc[2][2];
  u32 ks;
  auto load_k = [&](int t0, int t1) {
    const int64_t t = n < 16 ? t0 : t1;
    const u8 *kp = a.cache.k_codes + t * kFp8TileBytes + k_token * 64 + 16 * half;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int x = 0; x < 2; ++x) kc[s][x] = *reinterpret_cast<const u32x4 *>(kp + s * (kFp8TileBytes / 2) + 32 * x);
    ks = a.cache.k_scales[t];
  };
  // V: wave w expands dims 32 w .. +31, a lane the 16 tokens of tile `half` of one.
  u32x4 vc;
  u32 vs;
  auto load_v = [&]() {
    const int64_t t = half ? tile[1] : tile[0];
    vc = *reinterpret_cast<const u32x4 *>(a.cache.v_codes + t * kFp8TileBytes + (32 * w + n) * kFp8Tile);
    vs = a.cache.v_scales[t];
  };
  const int sees_all = rows.offset + rows.first / a.group;  // keys up to here every row of the workgroup sees
  auto on_diagonal = [&](int t) { return t * kBK + kBK - 1 > sees_all; };
  int v_at = ((half * 4 + w) * 64 + n) * (int)sizeof(u32x4);  // of the lane's operands in a stage
  asm volatile("" : "+v"(v_at));
  auto expand = [&](int t, Stage &st) {
    if (__builtin_expect(t * kBK + kBK > kv_len, 0)) keep_tokens(vc, kv_len - t * kBK - 16 * half);  // stale rows
    if (__builtin_expect(on_diagonal(t), 0)) {
      const u32 tokens = take_nans(vc);
      const bool some = __builtin_amdgcn_ballot_w64(tokens != 0) != 0;
      if (some) st.nan[w][n][half] = tokens;
      if (lane == 0) st.any[w] = some;
    }
    const float scale = fp8_scale(vs);
    u32x4 *at = reinterpret_cast<u32x4 *>(reinterpret_cast<u8 *>(&st.v) + v_at);
    at[0] = expand8<0>(vc, scale);
    at[32] = expand8<2>(vc, scale);
  };

  auto score = [&](f32x16 &sc) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
    sc = mfma32_fp8_fp8<0>(kc[0], ks, q_hi[0], q_scales, sc);
    sc = mfma32_fp8_fp8<0>(kc[0], ks, q_lo[0], q_scales, sc);
    sc = mfma32_fp8_fp8<1>(kc[1], ks, q_hi[1], q_scales, sc);
    sc = mfma32_fp8_fp8<1>(kc[1], ks, q_lo[1], q_scales, sc);
  };
  auto weigh = [&](int t, const Stage &st, f32x16 &sc) {
    const int base = t * kBK;
    // Key of register i: base + 16 (i / 8) + 8 half + i % 8.
    if (__builtin_expect(base + kBK - 1 > wave_first || base + kBK > kv_len, 0)) {
      const int lim = last_seen() - base - 8 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i / 8) + (i % 8) > lim) sc[i] = -INFINITY;
    }
    // V's operands are on their way from LDS two ahead of their products.
    u32x4 v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] = st.v[0][i][lane];
    __builtin_amdgcn_sched_barrier(0);
    u32x4 pf[2];
    weigh_scores(sc, a.scale_log2e, acc, neg_ref, l_run, pf);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc[i % 4] = mfma32(v[i % 2], pf[i / 4], acc[i % 4]);
      if (i + 2 < 8) v[i % 2] = st.v[(i + 2) / 4][(i + 2) % 4][lane];
    }
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    if (__builtin_expect(on_diagonal(t), 0)) {
      const int seen = last_seen() - base;  // the last key of the tile that this lane's row sees
      const u32 mask = seen < 0 ? 0u : seen >= 31 ? 0xffffffffu : (2u << seen) - 1u;
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        if (__builtin_amdgcn_readfirstlane(st.any[db]) == 0) continue;
#pragma unroll 1
        for (int x = 0; x < 16; ++x) {  // a register at a time: unrolled, the loads would take registers from the loop
          const u32 *tokens = st.nan[db][8 * (x >> 2) + 4 * half + (x & 3)];
          const float poison = ((tokens[0] | tokens[1] << 16) & mask) != 0 ? NAN : 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[db][i] += i == x ? poison : 0.f;
        }
      }
    }
  };

  if (n_tiles > 0) {
    look_up(0);
    locate(0);
    load_k(tile[0], tile[1]);
    load_v();
    look_up(1);
    expand(0, stages[0]);
    locate(1);
    load_v();
    look_up(2);
    __syncthreads();
    // Here K holds tile t, V's registers tile t + 1, stage t % 2 V's operands of tile t; `tile` is t + 1's, `entry` t +
    // 2's.
#pragma unroll 1
    for (int t = 0; t < n_tiles; ++t) {
      const bool visible = r0 < rows.rows && t * kBK <= wave_last;
      const int2 next = {tile[0], tile[1]};
      if (t + 1 < n_tiles) {
        expand(t + 1, stages[(t + 1) & 1]);
        locate(t + 2);
        load_v();
        look_up(t + 3);
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16 sc;  // of this tile alone: its registers are free while V is added
      if (visible) score(sc);
      __builtin_amdgcn_sched_barrier(0);
      if (t + 1 < n_tiles) load_k(next.x, next.y);
      if (visible) weigh(t, stages[t & 1], sc);
      __syncthreads();
    }
  }

  if (outside && threadIdx.x == 0) flag_index_error(a.err, NVAMD_ERR_BLOCK);
  write_tile_rows(a, rows, g, r0, row, w, lane, acc, l_run, s_mem);
}

// ------------------------------------------------------------------------------------------ strips
constexpr int kStripsOnCu = 2;  // a wave of the workgroup on each SIMD
__global__ void __launch_bounds__(kStripWaves * 64) __attribute__((amdgpu_waves_per_eu(kStripsOnCu)))
prefill_strip_fp8_kernel(PrefillArgs<Fp8Cache> a) {
  __shared__ __attribute__((aligned(16))) float s_o[kStripWaves][kStripRows / 2][kRec];
  __shared__ float s_m[kStripWaves][kStripRows];
  __shared__ float s_l[kStripWaves][kStripRows];

  Rows rows;
  if (!find_rows(a, kStripRows, blockIdx.y, rows)) return;
  const int piece = blockIdx.x / a.num_kv_heads, g = blockIdx.x - piece * a.num_kv_heads;
  const Cut cut = find_cut(a, rows, kStripRows);
  if (piece >= cut.pieces) return;
  const int begin = piece * cut.length, end = min(begin + cut.length, cut.keys);
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, n = lane & 31;
  const int row = min(rows.first + n, rows.rows - 1);
  const int last_seen = min(rows.offset + row / a.group, rows.kv_len - 1);
  const int first_seen = rows.offset + rows.first / a.group;  // the last key that the first row sees

  i32x8 q_hi[2], q_lo[2];
  u32 q_scale[2];
  load_query(a, rows, row, g, half, q_hi, q_lo, q_scale);

  f32x16 acc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
  float neg_ref = -kNoScore, l_run = 0.f;  // minus the exponent's reference; the sum at that reference

  const_i32 *bt = (const_i32 *)(a.block_tables + (int64_t)blockIdx.z * a.bt_stride);
  const int last_tile = max(rows.kv_len - 1, 0) & ~15;
  int entry[2], tile[2];
  auto look_up = [&](int t0) {
#pragma unroll
    for (int x = 0; x < 2; ++x) entry[x] = bt[min(t0 + 16 * x, last_tile) >> a.bs_log2];
  };
  auto locate = [&](int t0) {
#pragma unroll
    for (int x = 0; x < 2; ++x) tile[x] = tile_of(a, entry[x], min(t0 + 16 * x, last_tile), g, lane == 0);
  };
  // Byte `at` of the lane's one of the two tiles.
  auto in_tile = [&](const u8 *base, int second, int tile_bytes, u32 at) {  // (second as a bool: 25 us for 14)
    return base + (int64_t)(second ? tile[1] : tile[0]) * tile_bytes + at;
  };
  // Row n of K is token 4 (n / 8) + n % 4 of tile (n / 4) % 2: then register i of the scores is token i of tile `half`.
  const int k_token = 4 * (n >> 3) + (n & 3);
  const int k_second = (n & 4) ? -1 : 0, v_second = -half;
  u32x4 kc[2][2], vc[4];
  u32 ks, vs;
  auto load_k = [&]() {
    const u8 *kp = in_tile(a.cache.k_codes, k_second, kFp8TileBytes, k_token * 64 + 16 * half);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int x = 0; x < 2; ++x) kc[s][x] = *reinterpret_cast<const u32x4 *>(kp + s * (kFp8TileBytes / 2) + 32 * x);
    ks = *in_tile(a.cache.k_scales, k_second, 1, 0);
  };
  // Dims n, 32 + n .. of V, 16 tokens of tile `half` each.
  auto load_v = [&]() {
    const u8 *vp = in_tile(a.cache.v_codes, v_second, kFp8TileBytes, n * kFp8Tile);
#pragma unroll
    for (int db = 0; db < 4; ++db) vc[db] = *reinterpret_cast<const u32x4 *>(vp + 32 * kFp8Tile * db);
    vs = *in_tile(a.cache.v_scales, v_second, 1, 0);
  };
  auto step = [&](const int t0, const int next) {
    f32x16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      sc = mfma32_fp8_fp8(kc[s], ks, q_hi[s], q_scale[s], sc);
      sc = mfma32_fp8_fp8(kc[s], ks, q_lo[s], q_scale[s], sc);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (next < end) {
      locate(next);
      load_k();
      look_up(next + 32 * kStripWaves);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t0 + 31 > first_seen || t0 + 32 > rows.kv_len) {
      const int lim = last_seen - t0 - 16 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i > lim) sc[i] = -INFINITY;
    }
    u32x4 pf[2];
    weigh_scores(sc, a.scale_log2e, acc, neg_ref, l_run, pf);
    if (t0 + 31 > first_seen || t0 + 32 > rows.kv_len) {
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        keep_tokens(vc[db], rows.kv_len - t0 - 16 * half);  // stale rows past the keys
        const u32 bad = take_nans(vc[db]);                  // tokens of tile `half` whose value of dim 32 db + n is NaN
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) == 0, 1)) continue;
#pragma unroll 1
        for (int x = 0; x < 64; ++x) {  // dim 32 db + x % 32, tile x / 32
          const u32 tokens = (u32)__builtin_amdgcn_readlane((int)bad, x);
          if (tokens == 0) continue;
          const int at = t0 + 16 * (x >> 5) + __ffs((int)tokens) - 1;  // the first of them
          const bool hit = last_seen >= at && half == ((x >> 2) & 1);
          const int reg = 4 * ((x & 31) >> 3) + (x & 3);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[db][i] += hit && i == reg ? NAN : 0.f;
        }
      }
    }
    const float v_scale = fp8_scale(vs);
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      acc[db] = mfma32(expand8<0>(vc[db], v_scale), pf[0], acc[db]);
      acc[db] = mfma32(expand8<2>(vc[db], v_scale), pf[1], acc[db]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (next < end) load_v();
  };
  if (int t0 = begin + 32 * w; t0 < end) {
    look_up(t0);
    locate(t0);
    load_k();
    load_v();
    look_up(t0 + 32 * kStripWaves);
#pragma unroll 1
    do {
      step(t0, t0 + 32 * kStripWaves);
      t0 += 32 * kStripWaves;
    } while (t0 < end);
  }

  write_strip(a, rows, cut, piece, g, w, lane, acc, neg_ref, l_run, s_o, s_m, s_l, [](int db, int i, int half) {
    return 32 * db + 2 * i + 4 * half;
  });
}

// ------------------------------------------------------------------------------------------ few rows
__global__ void __launch_bounds__(kFewWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
prefill_few_fp8_kernel(PrefillArgs<Fp8Cache> a) {
  constexpr int D = kHeadDim;
  __shared__ __attribute__((aligned(16))) float s_o[kFewWaves][kFewRows * kRec];
  __shared__ float s_m[kFewWaves][kFewRows];
  __shared__ float s_l[kFewWaves][kFewRows];

  Rows rows;
  if (!find_rows(a, kFewRows, blockIdx.y, rows)) return;
  const int piece = blockIdx.x / a.num_kv_heads, g = blockIdx.x - piece * a.num_kv_heads;
  const Cut cut = find_cut(a, rows, kFewRows);
  if (piece >= cut.pieces) return;
  const int begin = piece * cut.length, end = min(begin + cut.length, cut.keys);
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, gq = lane >> 4;
  const int row = min(rows.first + n, rows.rows - 1);
  const int token = row / a.group, head = g * a.group + row - token * a.group;
  const int last_seen = min(rows.offset + token, rows.kv_len - 1);
  const int first_seen = rows.offset + rows.first / a.group;  // the last key that the first row sees

  i32x8 q_hi, q_lo;
  u32 q_scale;
  {
    const u16 *qp = a.q + (int64_t)(rows.q_start + token) * a.q_stride + (int64_t)head * D + 16 * gq;
    const u32x4 x[4] = {ld16(qp), ld16(qp + 8), ld16(qp + 64), ld16(qp + 72)};
    q_scale = query_operand(x, gq, q_hi, q_lo);
  }

  float m = kNoScore, m_thr = kNoScore, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int32_t *bt = a.block_tables + (int64_t)blockIdx.z * a.bt_stride;
  const int last_tile = max(rows.kv_len - 1, 0) & ~15;
  int entry_k = 0, entry_v = 0;
  auto look_up = [&](int t0) {
    entry_k = bt[min(t0 + 16 * (n >> 2), last_tile) >> a.bs_log2];
    entry_v = bt[min(t0 + 16 * gq, last_tile) >> a.bs_log2];
  };
  u32x4 kc[4][2], vc[8];
  u32 ks, vs;
  int k_tile, v_tile;
  auto locate = [&](int t0) {
    k_tile = tile_of(a, entry_k, min(t0 + 16 * (n >> 2), last_tile), g, true);
    v_tile = tile_of(a, entry_v, min(t0 + 16 * gq, last_tile), g, true);
  };
  auto load_k = [&]() {
    const u8 *kp = a.cache.k_codes + (int64_t)k_tile * kFp8TileBytes + (n & 3) * 64 + 16 * gq;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        kc[t][x] = *reinterpret_cast<const u32x4 *>(kp + 4 * t * 64 + x * (kFp8TileBytes / 2));
    ks = a.cache.k_scales[k_tile];
  };
  auto load_v = [&]() {
    const u8 *vp = a.cache.v_codes + (int64_t)v_tile * kFp8TileBytes + n * kFp8Tile;
#pragma unroll
    for (int e = 0; e < 8; ++e) vc[e] = *reinterpret_cast<const u32x4 *>(vp + 16 * kFp8Tile * e);
    vs = a.cache.v_scales[v_tile];
  };
  auto step = [&](const int t0, const int next) {
    f32x4 s[4];
    score(s[0], kc[0], ks, q_hi, q_lo, q_scale);
    score(s[1], kc[1], ks, q_hi, q_lo, q_scale);
    score(s[2], kc[2], ks, q_hi, q_lo, q_scale);
    score(s[3], kc[3], ks, q_hi, q_lo, q_scale);
    __builtin_amdgcn_sched_barrier(0);
    if (next < end) {
      locate(next);
      load_k();
      look_up(next + 64 * kFewWaves);
    }
    __builtin_amdgcn_sched_barrier(0);
    float cm = kNoScore;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] *= a.scale_log2e;
    if (t0 + 63 > first_seen || t0 + 64 > rows.kv_len) {
      const int lim = last_seen - t0 - 16 * gq;  // token 4 t + i of tile gq
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * t + i > lim) s[t][i] = -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) cm = fmaxf(cm, s[t][i]);
    cm = max_over_quarters(cm);
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
    u32x4 pf[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32 pr = pack_bf16x2(fast_exp2(s[t][2 * i] - m), fast_exp2(s[t][2 * i + 1] - m));
        l = dot2_bf16(pr, kBf16PairOne, l);
        pf[t >> 1][2 * (t & 1) + i] = pr;
      }
    if (t0 + 63 > first_seen || t0 + 64 > rows.kv_len) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        keep_tokens(vc[e], rows.kv_len - t0 - 16 * gq);  // stale rows past the keys
        const u32 bad = take_nans(vc[e]);                // tokens of tile gq whose value of dim 16 e + n is NaN
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) == 0, 1)) continue;
#pragma unroll 1
        for (int x = 0; x < 64; ++x) {  // dim 16 e + x % 16, tile x / 16
          const u32 tokens = (u32)__builtin_amdgcn_readlane((int)bad, x);
          if (tokens == 0) continue;
          const int at = t0 + 16 * (x >> 4) + __ffs((int)tokens) - 1;  // the first of them
          const bool hit = last_seen >= at && gq == ((x & 15) >> 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[e][i] += hit && i == (x & 3) ? NAN : 0.f;
        }
      }
    }
    const float v_scale = fp8_scale(vs);
#pragma unroll
    for (int e = 0; e < 8; ++e) add_values(o[e], vc[e], v_scale, pf);
    __builtin_amdgcn_sched_barrier(0);
    if (next < end) load_v();
  };
  if (int t0 = begin + 64 * w; t0 < end) {
    look_up(t0);
    locate(t0);
    load_k();
    load_v();
    look_up(t0 + 64 * kFewWaves);
#pragma unroll 1
    do {
      step(t0, t0 + 64 * kFewWaves);
      t0 += 64 * kFewWaves;
    } while (t0 < end);
  }

  write_few(a, rows, cut, piece, g, w, lane, o, m, l, s_o, s_m, s_l);
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" size_t nvamd_paged_prefill_fp8_workspace_size(int n_seqs, int max_q_len, int num_heads, int num_kv_heads,
                                                         int block_size, int bt_width) {
  return prefill_workspace_bytes<kStripsOnCu>(n_seqs, max_q_len, num_heads, num_kv_heads, block_size, bt_width);
}

extern "C" int nvamd_paged_prefill_fp8(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                       const void *k_codes, const void *k_scales, const void *v_codes,
                                       const void *v_scales, int num_blocks, int block_size,
                                       const int32_t *block_tables, int bt_stride, int bt_width,
                                       const int32_t *cu_seqlens_q, const int32_t *kv_lens, int n_seqs, int num_tokens,
                                       int max_q_len, int num_heads, int num_kv_heads, int head_dim, float scale,
                                       void *workspace, size_t workspace_bytes, hipStream_t stream) {
  const Fp8Cache cache = {const_cast<u8 *>(static_cast<const u8 *>(k_codes)),
                          const_cast<u8 *>(static_cast<const u8 *>(k_scales)),
                          const_cast<u8 *>(static_cast<const u8 *>(v_codes)),
                          const_cast<u8 *>(static_cast<const u8 *>(v_scales))};
  return prefill<kStripsOnCu>(prefill_few_fp8_kernel, prefill_strip_fp8_kernel, prefill_fp8_kernel, cache,
                 fp8_cache_ok(k_codes, k_scales, v_codes, v_scales), out, out_stride, q, q_stride, num_blocks, block_size,
                 block_tables, bt_stride, bt_width, cu_seqlens_q, kv_lens, n_seqs, num_tokens, max_q_len, num_heads,
                 num_kv_heads, head_dim, scale, workspace, workspace_bytes, stream);
}
