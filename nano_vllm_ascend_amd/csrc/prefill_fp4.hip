// Causal prefill attention over the 4-bit paged KV cache (the counterpart of prefill.hip's paged route): the queries
// are the last q_len positions of a context of kv_len, query row r sees keys 0 .. kv_len - q_len + r, all of them in
// the cache.
//
// The G query heads of a kv head and the q_len tokens make q_len * G rows, R = token * G + head, that share the keys; a
// workgroup takes rows that follow one another, whatever G is.  In all kernels
//   S^T = K . Q^T   v_mfma_scale_f32_*_f8f6f4 on the codes as they lie in the cache: a lane loads 32 dims of a key and their
//        scale straight into the operand, and the row comes as two e4m3 numbers per value (fp4_attention.h).  No
//        expansion of K, and none of it in LDS;
//   O^T += V^T . P^T   v_mfma_f32_*_bf16 on V expanded by v_cvt_scalef32_pk_bf16_fp4, exact.
// The rows of K are taken in such an order that a lane's registers of S^T are the consecutive keys that its operand of
// P^T needs: a repack in registers.  Three kernels, which differ in how many rows share an expansion of V:
//
// Tiles (the card is full).  Workgroup = 4 waves = 128 rows, a wave 32 of them, tiles of 32 keys.  The workgroup
//   expands a tile of V once, to bf16 operands in LDS (every access is 64 lanes x 16 consecutive bytes): a wave takes 8
//   tokens of a 16-token tile, a lane a dim pair of them.  Key 16a + 8b + 4c + x sits in row 16a + 8c + 4b + x of K.  K
//   of the next tile loads as the scores have taken this one's, V's codes are two tiles ahead, V's operands one (two
//   stages, one barrier a tile). Bound by issue: the matrix cores are busy 43.5% of the time and the vector ALUs
//   (exponents, rounding, expansion) 55%, one or the other at 98.5% of it.  32 x U[512, 2048] rows on 1,152 cached keys
//   695 us (887 TFLOP/s), 2 x U[3000, 4000] rows of 40 query heads on 4,096 1,004 us (990 TFLOP/s), on a card whose bf16
//   matrix product of 8,192^3 reaches 1,252 (where it reaches 1,185, 754 and 1,113 us).
//
// Strips (one long prompt, or several short ones).  Workgroup = 4 waves = 32 rows, a wave every fourth 32 keys; no
//   barrier in the loop, the waves' results meet in LDS.  A lane expands 16 tokens of a dim pair straight into
//   operands: four times the tile kernel's expansion for each row, for four times the workgroups.  1 x 4,000 rows on
//   4,096 keys 232 us (859 TFLOP/s).
//
// Few rows (a chat's next turn).  Workgroup = 8 waves = 16 rows, a wave every eighth 64 keys, as in
//   paged_decode_fp4.hip with rows in the place of heads and a last key for each row.  Bound by the latency of a launch
//   and of a wave's steps: 8 x 20 rows on 1,040 keys 10 us.  On long contexts the keys are cut as well.
//
// Weights are rounded to bf16 once for the matrix cores, and the sums take the rounded values, as in the bf16 cache's
// prefill: a second term would double the products with V, where the matrix cores' and the vector ALUs' issue already
// fills the time.
//
// A block of values that reads as NaN must reach the rows that see its key and no others, though masked rows
// multiply it by a weight of zero: such values enter the products as zeros, and the rows that see
// the key get the NaN afterwards (a branch that no other tile takes).
#include "fp4_attention.h"
#include "prefill_quantised.h"

namespace nvamd {
namespace {

// 0x80 in the bytes that are 255: only there do the low seven bits carry into a set top bit.
__device__ __forceinline__ u32 nan_bytes(u32 scales) {
  return ((scales & 0x7f7f7f7fu) + 0x01010101u) & scales & 0x80808080u;
}
__device__ __forceinline__ u32 without(u32 scales, u32 nans) { return scales & ~((nans >> 7) * 0xffu); }

// ------------------------------------------------------------------------------------------ tiles

// 64 dims: lane (n, half) gives block `half` of them of row n, dims 16 half .. +15 and 32 + 16 half .. +15 of column n,
// and the scales of block `half` of either (checked on gfx950).
__device__ __forceinline__ f32x16 mfma32_fp4_fp8(u32x4 k, u32 k_scale, i32x8 q, u32 q_scale, f32x16 c) {
  const i32x8 codes = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes, q, c, 4, 0, 0, (int)k_scale, 0, (int)q_scale);
}

struct Stage {
  u32x4 v[2][4][64];  // [16-key step][32-dim block][lane]
  u32 any[4];         // [wave that expanded them]: whether any of its values read as NaN,
  u32 nan[4][2];      // and which: two blocks of dims a word, a bit for each of the 8 tokens in its half
};
__global__ void __launch_bounds__(kTileWaves * 64) __attribute__((amdgpu_waves_per_eu(3)))
prefill_fp4_kernel(PrefillArgs<Fp4Cache> a) {
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
  int row = min(r0 + n, rows.rows - 1);
  const int last_seen = min(rows.offset + row / a.group, kv_len - 1);  // by this lane's row
  const int wave_first = rows.offset + r0 / a.group;           // the last key that the wave's first row sees
  const int wave_last = rows.offset + min(r0 + 31, rows.rows - 1) / a.group;
  const int end_row = min(rows.first + kTileRows, rows.rows) - 1;
  const int keys = min(kv_len, rows.offset + end_row / a.group + 1);  // that the workgroup needs
  const int n_tiles = keys > 0 ? ceil_div(keys, kBK) : 0;

  i32x8 q_hi[2], q_lo[2];
  u32 q_scale[2];
  load_query(a, rows, row, g, half, q_hi, q_lo, q_scale);

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
  auto locate = [&](int t) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
      tile[x] = tile_of(a, entry[x], min(t * kBK + 16 * x, last_tile), g, threadIdx.x == 0);
  };
  // K: key 16a + 8b + 4c + x of the tile in row n = 16a + 8c + 4b + x.
  const int k_token = (n & 3) | ((n & 8) >> 1) | ((n & 4) << 1);  // of its 16-token tile, n / 16
  u32x4 kc[2];
  u32 ks[2];
  const u32 k_at = k_token * kFp4RowBytes + 16 * half, ks_at = fp4_key_scale_at(k_token, half);
  auto load_k = [&](int t0, int t1) {
    const int64_t t = n < 16 ? t0 : t1;
    const u8 *kp = a.cache.k_codes + t * kFp4TileBytes + k_at, *sp = a.cache.k_scales + t * kFp4TileScales + ks_at;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      kc[s] = *reinterpret_cast<const u32x4 *>(kp + 32 * s);
      ks[s] = sp[8 * s];
    }
  };
  // V: wave w expands tokens 8 (w % 2) .. +7 of 16-token tile w / 2, a lane one pair of dims.
  u32x2 vc, vs;
  auto load_v = [&]() {
    const int64_t t = w < 2 ? tile[0] : tile[1];
    vc = *reinterpret_cast<const u32x2 *>(a.cache.v_codes + t * kFp4TileBytes + 16 * lane + 8 * (w & 1));
    vs = *reinterpret_cast<const u32x2 *>(a.cache.v_scales + t * kFp4TileScales + 16 * (lane >> 4) + 8 * (w & 1));
  };
  auto expand = [&](int t, Stage &st) {
    const int left = kv_len - t * kBK - 8 * w;  // of the wave's 8 tokens
    if (__builtin_expect(left < 8, 0)) {  // stale rows past the keys: under some scales a code is past bf16, and a weight
      vs[0] = keep_bytes(vs[0], left);    // of zero does not cancel it
      vs[1] = keep_bytes(vs[1], left - 4);
    }
    const u32 bad0 = nan_bytes(vs[0]), bad1 = nan_bytes(vs[1]);
    u32 seen0 = 0, seen1 = 0;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64((bad0 | bad1) != 0) != 0, 0)) {
      vs[0] = without(vs[0], bad0);
      vs[1] = without(vs[1], bad1);
      u32 bits = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) bits |= ((bad0 >> (8 * i + 7)) & 1) << i | ((bad1 >> (8 * i + 7)) & 1) << (4 + i);
      // blocks 0, 1 and 2, 3 in two words of 16 bits each
      seen0 = (u32)__builtin_amdgcn_readlane((int)bits, 0) | (u32)__builtin_amdgcn_readlane((int)bits, 16) << 16;
      seen1 = (u32)__builtin_amdgcn_readlane((int)bits, 32) | (u32)__builtin_amdgcn_readlane((int)bits, 48) << 16;
      if (lane == 0) *reinterpret_cast<u32x2 *>(st.nan[w]) = u32x2{seen0, seen1};
    }
    if (lane == 0) st.any[w] = seen0 | seen1;
    u32x4 lo, hi;
    {
      u32 x[8];
      expand4(vc[0], vs[0], x[0], x[1], x[4], x[5]);
      expand4(vc[1], vs[1], x[2], x[3], x[6], x[7]);
      lo = u32x4{x[0], x[1], x[2], x[3]};
      hi = u32x4{x[4], x[5], x[6], x[7]};
    }
    u32x4 *dst = st.v[w >> 1][lane >> 4] + 32 * (w & 1) + (lane & 15);
    dst[0] = lo;
    dst[16] = hi;
  };

  f32x16 sc;
  auto score = [&]() {
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      sc = mfma32_fp4_fp8(kc[s], ks[s], q_hi[s], q_scale[s], sc);
      sc = mfma32_fp4_fp8(kc[s], ks[s], q_lo[s], q_scale[s], sc);
    }
  };
  auto weigh = [&](int t, const Stage &st) {
    const int base = t * kBK;
    // Key of register i: base + 16 (i / 8) + 8 half + i % 8.
    if (__builtin_expect(base + kBK - 1 > wave_first || base + kBK > kv_len, 0)) {
      const int lim = last_seen - base - 8 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i / 8) + (i % 8) > lim) sc[i] = -INFINITY;
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, sc[i]);
    tmax = max_xor32(tmax) * a.scale_log2e;
    // Lazy rescale: the weights stay below 2^8, and O and l are scaled only where some row's reference moves.
    const bool up = tmax + neg_ref > kRescaleLog2;
    if (__builtin_amdgcn_ballot_w64(up) != 0) {
      const float alpha = up ? fast_exp2(-neg_ref - tmax) : 1.f;
      if (up) neg_ref = -tmax;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
    }
    u32x4 pf[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32 pr = pack_bf16x2(fast_exp2(fmaf(sc[8 * hh + 2 * e], a.scale_log2e, neg_ref)),
                                   fast_exp2(fmaf(sc[8 * hh + 2 * e + 1], a.scale_log2e, neg_ref)));
        l_run = dot2_bf16(pr, kBf16PairOne, l_run);  // both rounded values of the pair
        pf[hh][e] = pr;
      }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int db = 0; db < 4; ++db) acc[db] = mfma32(st.v[hh][db][lane], pf[hh], acc[db]);
    const u32x4 any = *reinterpret_cast<const u32x4 *>(st.any);
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(any[0] | any[1] | any[2] | any[3]) != 0, 0)) {
      const int seen = last_seen - base;  // the last key of the tile that this lane's row sees
      const u32 mask = seen < 0 ? 0u : seen >= 31 ? 0xffffffffu : (2u << seen) - 1u;
#pragma unroll 1
      for (int x = 0; x < 4; ++x) {  // 8 tokens each
        if (__builtin_amdgcn_readfirstlane(st.any[x]) == 0) continue;
        const u32 word[2] = {(u32)__builtin_amdgcn_readfirstlane(st.nan[x][0]),
                             (u32)__builtin_amdgcn_readfirstlane(st.nan[x][1])};
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          const u32 bits = ((word[db >> 1] >> (16 * (db & 1))) & 0xffu) << (8 * x);
          const float poison = (bits & mask) != 0 ? NAN : 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[db][i] += poison;
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
      if (visible) score();
      __builtin_amdgcn_sched_barrier(0);
      if (t + 1 < n_tiles) load_k(next.x, next.y);
      if (visible) weigh(t, stages[t & 1]);
      __syncthreads();
    }
  }

  write_tile_rows(a, rows, g, r0, row, w, lane, acc, l_run, s_mem);
}

// ------------------------------------------------------------------------------------------ strips
// acc[2 J], acc[2 J + 1] += V^T P^T for row bytes 32 J .. +31 and 32 tokens (lane (n, half): 16 tokens of tile `half`;
// scales in lanes 4 J .. 4 J + 3 of each 16).
template <int J>
__device__ __forceinline__ void add_strip(f32x16 (&acc)[4], u32x4 codes, u32 v_scales, const u32x4 (&p)[2]) {
  const u32 sc[4] = {dpp_u32<kRowBcast + 4 * J>(v_scales), dpp_u32<kRowBcast + 4 * J + 1>(v_scales),
                     dpp_u32<kRowBcast + 4 * J + 2>(v_scales), dpp_u32<kRowBcast + 4 * J + 3>(v_scales)};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32 x[4], y[4];
    expand4(codes[2 * h], sc[2 * h], x[0], x[1], y[0], y[1]);
    expand4(codes[2 * h + 1], sc[2 * h + 1], x[2], x[3], y[2], y[3]);
    acc[2 * J] = mfma32(u32x4{x[0], x[1], x[2], x[3]}, p[h], acc[2 * J]);
    acc[2 * J + 1] = mfma32(u32x4{y[0], y[1], y[2], y[3]}, p[h], acc[2 * J + 1]);
  }
}

constexpr int kStripsOnCu = 3;  // a wave of the workgroup on each SIMD
__global__ void __launch_bounds__(kStripWaves * 64) __attribute__((amdgpu_waves_per_eu(kStripsOnCu)))
prefill_strip_fp4_kernel(PrefillArgs<Fp4Cache> a) {
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
    for (int x = 0; x < 2; ++x) tile[x] = tile_of<true>(a, entry[x], min(t0 + 16 * x, last_tile), g, lane == 0);
  };
  // Byte `at` of the lane's one of the two tiles.
  auto in_tile = [&](const u8 *base, int second, int tile_bytes, u32 at) {  // (second as a bool: 25 us for 14)
    return base + (int64_t)(second ? tile[1] : tile[0]) * tile_bytes + at;
  };
  // Row n of K is token 4 (n / 8) + n % 4 of tile (n / 4) % 2: then register i of the scores is token i of tile `half`.
  const int k_token = 4 * (n >> 3) + (n & 3);
  const int k_second = (n & 4) ? -1 : 0, v_second = -half;
  const u32 k_at = k_token * kFp4RowBytes + 16 * half, ks_at = fp4_key_scale_at(k_token, half);
  // Row bytes n and 32 + n of V, 16 tokens of tile `half` each: the low nibbles are one operand's row, the high ones
  // another's. Their scales: lane i of a row of 16 holds tokens 4 (i % 4) .. +3 of block 2 (i / 4 % 2) + n / 16.
  const u32 vs_at = 16 * (2 * ((n >> 2) & 1) + (n >> 4)) + 4 * (n & 3);
  u32x4 kc[2], vc[2];
  u32 ks[2], vs;
  auto load_k = [&]() {
    const u8 *kp = in_tile(a.cache.k_codes, k_second, kFp4TileBytes, k_at);
    const u8 *sp = in_tile(a.cache.k_scales, k_second, kFp4TileScales, ks_at);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      kc[s] = *reinterpret_cast<const u32x4 *>(kp + 32 * s);
      ks[s] = sp[8 * s];
    }
  };
  auto load_v = [&]() {
    const u8 *vp = in_tile(a.cache.v_codes, v_second, kFp4TileBytes, 16 * n);
#pragma unroll
    for (int j = 0; j < 2; ++j) vc[j] = *reinterpret_cast<const u32x4 *>(vp + 512 * j);
    vs = *reinterpret_cast<const u32 *>(in_tile(a.cache.v_scales, v_second, kFp4TileScales, vs_at));
  };
  auto step = [&](const int t0, const int next) {
    f32x16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      sc = mfma32_fp4_fp8(kc[s], ks[s], q_hi[s], q_scale[s], sc);
      sc = mfma32_fp4_fp8(kc[s], ks[s], q_lo[s], q_scale[s], sc);
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
      vs = keep_bytes(vs, rows.kv_len - t0 - 16 * half - 4 * (n & 3));  // stale rows past the keys
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, sc[i]);
    tmax = max_xor32(tmax) * a.scale_log2e;
    const bool up = tmax + neg_ref > kRescaleLog2;
    if (__builtin_amdgcn_ballot_w64(up) != 0) {
      const float alpha = up ? fast_exp2(-neg_ref - tmax) : 1.f;
      if (up) neg_ref = -tmax;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
    }
    u32x4 pf[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32 pr = pack_bf16x2(fast_exp2(fmaf(sc[8 * hh + 2 * e], a.scale_log2e, neg_ref)),
                                   fast_exp2(fmaf(sc[8 * hh + 2 * e + 1], a.scale_log2e, neg_ref)));
        l_run = dot2_bf16(pr, kBf16PairOne, l_run);
        pf[hh][e] = pr;
      }
    const u32 bad = nan_bytes(vs);
    vs = without(vs, bad);
    add_strip<0>(acc, vc[0], vs, pf);
    add_strip<1>(acc, vc[1], vs, pf);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) != 0, 0)) {
      u32 hit = 0;  // a bit for each block that this lane's row sees a NaN of
#pragma unroll 1
      for (int x = 0; x < 64; ++x) {  // of lane x's scales
        const u32 b = (u32)__builtin_amdgcn_readlane((int)bad, x);
        if (b == 0) continue;
        const int at = t0 + 16 * (x >> 5) + 4 * (x & 3) + (__ffs((int)b) >> 3) - 1;  // the first of them (bit 7 of a byte)
        hit |= last_seen >= at ? 1u << (2 * ((x >> 2) & 1) + ((x >> 4) & 1)) : 0u;
      }
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] += hit >> (2 * (db >> 1) + (i >> 3)) & 1 ? NAN : 0.f;
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
    return 64 * (db >> 1) + 32 * (i >> 3) + 16 * (db & 1) + 2 * (i & 4) + 4 * half;
  });
}

// ------------------------------------------------------------------------------------------ few rows
__global__ void __launch_bounds__(kFewWaves * 64) __attribute__((amdgpu_waves_per_eu(3)))
prefill_few_fp4_kernel(PrefillArgs<Fp4Cache> a) {
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
  u32x4 kc[4], vc[4];
  u32 ks, vs;
  int k_tile, v_tile;
  auto locate = [&](int t0) {
    k_tile = tile_of(a, entry_k, min(t0 + 16 * (n >> 2), last_tile), g, true);
    v_tile = tile_of(a, entry_v, min(t0 + 16 * gq, last_tile), g, true);
  };
  auto load_k = [&]() {
    const u8 *kp = a.cache.k_codes + (int64_t)k_tile * kFp4TileBytes + (n & 3) * kFp4RowBytes + 16 * gq;
#pragma unroll
    for (int t = 0; t < 4; ++t) kc[t] = *reinterpret_cast<const u32x4 *>(kp + 4 * t * kFp4RowBytes);
    ks = *reinterpret_cast<const u32 *>(a.cache.k_scales + (int64_t)k_tile * kFp4TileScales + fp4_key_scale_at(n & 3, gq));
  };
  auto load_v = [&]() {
    const u8 *vp = a.cache.v_codes + (int64_t)v_tile * kFp4TileBytes + 16 * n;
#pragma unroll
    for (int q = 0; q < 4; ++q) vc[q] = *reinterpret_cast<const u32x4 *>(vp + 256 * q);
    vs = *reinterpret_cast<const u32 *>(a.cache.v_scales + (int64_t)v_tile * kFp4TileScales + 4 * n);
  };
  auto step = [&](const int t0, const int next) {
    f32x4 s[4];
    score<0>(s[0], kc[0], ks, q_hi, q_lo, q_scale);
    score<1>(s[1], kc[1], ks, q_hi, q_lo, q_scale);
    score<2>(s[2], kc[2], ks, q_hi, q_lo, q_scale);
    score<3>(s[3], kc[3], ks, q_hi, q_lo, q_scale);
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
      vs = keep_bytes(vs, rows.kv_len - t0 - 16 * gq - 4 * (n & 3));  // stale rows past the keys
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
    const u32 bad = nan_bytes(vs);
    vs = without(vs, bad);
    add_values<0>(o, vc, vs, pf);
    add_values<1>(o, vc, vs, pf);
    add_values<2>(o, vc, vs, pf);
    add_values<3>(o, vc, vs, pf);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad != 0) != 0, 0)) {
      u32 hit = 0;  // a bit for each block that this lane's row sees a NaN of
#pragma unroll 1
      for (int x = 0; x < 64; ++x) {  // lane x noted tokens 4 (x % 4) .. of tile x / 16, block (x % 16) / 4
        const u32 b = (u32)__builtin_amdgcn_readlane((int)bad, x);
        if (b == 0) continue;
        const int at = t0 + 16 * (x >> 4) + 4 * (x & 3) + (__ffs((int)b) >> 3) - 1;  // the first of them (bit 7 of a byte)
        hit |= last_seen >= at ? 1u << ((x & 15) >> 2) : 0u;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += hit >> (e >> 1) & 1 ? NAN : 0.f;
    }
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

extern "C" size_t nvamd_paged_prefill_fp4_workspace_size(int n_seqs, int max_q_len, int num_heads, int num_kv_heads,
                                                         int block_size, int bt_width) {
  return prefill_workspace_bytes<kStripsOnCu>(n_seqs, max_q_len, num_heads, num_kv_heads, block_size, bt_width);
}

extern "C" int nvamd_paged_prefill_fp4(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                       const void *k_codes, const void *k_scales, const void *v_codes,
                                       const void *v_scales, int num_blocks, int block_size,
                                       const int32_t *block_tables, int bt_stride, int bt_width,
                                       const int32_t *cu_seqlens_q, const int32_t *kv_lens, int n_seqs, int num_tokens,
                                       int max_q_len, int num_heads, int num_kv_heads, int head_dim, float scale,
                                       void *workspace, size_t workspace_bytes, hipStream_t stream) {
  const Fp4Cache cache = {const_cast<u8 *>(static_cast<const u8 *>(k_codes)),
                          const_cast<u8 *>(static_cast<const u8 *>(k_scales)),
                          const_cast<u8 *>(static_cast<const u8 *>(v_codes)),
                          const_cast<u8 *>(static_cast<const u8 *>(v_scales))};
  return prefill<kStripsOnCu>(prefill_few_fp4_kernel, prefill_strip_fp4_kernel, prefill_fp4_kernel, cache,
                 fp4_cache_ok(k_codes, k_scales, v_codes, v_scales), out, out_stride, q, q_stride, num_blocks, block_size,
                 block_tables, bt_stride, bt_width, cu_seqlens_q, kv_lens, n_seqs, num_tokens, max_q_len, num_heads,
                 num_kv_heads, head_dim, scale, workspace, workspace_bytes, stream);
}
