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

namespace nvamd {
namespace {

struct PrefillFp4Args {
  u16 *out;
  int64_t out_stride;
  const u16 *q;
  int64_t q_stride;
  Fp4Cache cache;
  const int32_t *block_tables;
  const int32_t *cu_seqlens_q;
  const int32_t *kv_lens;
  int bt_stride;
  int bt_width;
  int num_blocks;
  int bs_log2;
  int num_kv_heads;
  int group;  // query heads of a kv head
  int max_tiles;
  int max_q_len;
  int num_tokens;
  float scale_log2e;
  int splits;       // that the keys of a workgroup's rows are cut into at most
  float *partials;  // [sequence][kv head][split][row][kRec]
  u32 *err;
};

// A workgroup's sequence and rows.
struct Rows {
  int q_start;
  int rows;    // q_len * group
  int kv_len;
  int offset;  // token t sees keys 0 .. offset + t
  int first;   // the workgroup's first row
};
// The y-th group of rows from a sequence's end: those with the most keys start first.  False if it has none.  Faults
// are reported once per sequence.
__device__ __forceinline__ bool find_rows(const PrefillFp4Args &a, int per_group, int y, Rows &r) {
  const int s = blockIdx.z;
  r.q_start = a.cu_seqlens_q[s];
  const int q_end = a.cu_seqlens_q[s + 1];
  const int q_len = (int)((unsigned)q_end - (unsigned)r.q_start);
  const int cap = a.bt_width << a.bs_log2;
  const int kv_len = a.kv_lens[s];
  const bool rows_in = r.q_start >= 0 && r.q_start <= q_end && q_end <= a.num_tokens;  // else no row is touched
  if ((!rows_in || q_len > a.max_q_len || kv_len > cap || kv_len < q_len) && blockIdx.x == 0 && blockIdx.y == 0 &&
      threadIdx.x == 0)
    flag_index_error(a.err, NVAMD_ERR_CONTEXT);
  r.rows = min(q_len, a.max_q_len) * a.group;
  r.first = (a.max_tiles - 1 - y) * per_group;
  r.kv_len = min(kv_len, cap);
  r.offset = r.kv_len - q_len;
  return rows_in && r.first < r.rows;
}

// The keys that rows first .. first + per_group - 1 need, and their cut: pieces of a multiple of kMinSplit.
constexpr int kMinSplit = 512;
constexpr int kRec = kHeadDim + 4;  // floats of a row's record: max, sum, 2 unused, numerators
struct Cut {
  int keys;
  int length;
  int pieces;
};
__device__ __forceinline__ Cut find_cut(const PrefillFp4Args &a, const Rows &r, int per_group) {
  const int keys = max(min(r.kv_len, r.offset + (min(r.first + per_group, r.rows) - 1) / a.group + 1), 0);
  if (a.splits == 1) return {keys, keys, 1};
  const int length = max(ceil_div(ceil_div(keys, a.splits), kMinSplit), 1) * kMinSplit;
  return {keys, length, max(ceil_div(keys, length), 1)};
}
__device__ __forceinline__ float *record(const PrefillFp4Args &a, int per_group, int g, int piece, int row) {
  const int64_t unit = ((int64_t)blockIdx.z * a.num_kv_heads + g) * a.splits + piece;
  return a.partials + (unit * (a.max_tiles * per_group) + row) * kRec;
}

__device__ __forceinline__ int tile_of(const PrefillFp4Args &a, int entry, int token, int g, bool report) {
  if ((unsigned)entry >= (unsigned)a.num_blocks && report) flag_index_error(a.err, NVAMD_ERR_BLOCK);
  entry = min(max(entry, 0), a.num_blocks - 1);  // never leave the pool
  return (int)fp4_tile(entry, token & ((1 << a.bs_log2) - 1), g, a.num_kv_heads, a.bs_log2);
}

// 0x80 in the bytes that are 255: only there do the low seven bits carry into a set top bit.
__device__ __forceinline__ u32 nan_bytes(u32 scales) {
  return ((scales & 0x7f7f7f7fu) + 0x01010101u) & scales & 0x80808080u;
}
__device__ __forceinline__ u32 without(u32 scales, u32 nans) { return scales & ~((nans >> 7) * 0xffu); }

// ------------------------------------------------------------------------------------------ tiles
constexpr int kBK = 32;  // keys per tile
constexpr int kWaves = 4;
constexpr int kTileRows = 32 * kWaves;

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0,
                                                 0, 0);
}
// 64 dims: lane (n, half) gives block `half` of them of row n, dims 16 half .. +15 and 32 + 16 half .. +15 of column n,
// and the scales of block `half` of either (checked on gfx950).
__device__ __forceinline__ f32x16 mfma32_fp4_fp8(u32x4 k, u32 k_scale, i32x8 q, u32 q_scale, f32x16 c) {
  const i32x8 codes = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes, q, c, 4, 0, 0, (int)k_scale, 0, (int)q_scale);
}

// A row's operands: dims 64 s + 16 half .. +15 and 64 s + 32 + 16 half .. +15, the scales of block 2 s + half.
__device__ __forceinline__ void load_query(const PrefillFp4Args &a, const Rows &rows, int row, int g, int half,
                                           i32x8 (&hi)[2], i32x8 (&lo)[2], u32 (&scale)[2]) {
  const int token = row / a.group, head = g * a.group + row - token * a.group;
  const u16 *qp = a.q + (int64_t)(rows.q_start + token) * a.q_stride + (int64_t)head * kHeadDim + 16 * half;
  auto over_halves = [](u32 v) {  // each has 16 dims of a block
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((u32)r[0], (u32)r[1]);
  };
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = ld16(qp + 64 * s + 32 * (j >> 1) + 8 * (j & 1));
    const QueryScale s0 = query_scale(over_halves(max(largest(x[0]), largest(x[1]))));
    const QueryScale s1 = query_scale(over_halves(max(largest(x[2]), largest(x[3]))));
    split32(x, s0.up, s1.up, hi[s], lo[s]);
    scale[s] = half ? s1.byte : s0.byte;
  }
}
typedef const __attribute__((address_space(4))) int32_t const_i32;  // block tables: nothing writes them, scalar loads

struct Stage {
  u32x4 v[2][4][64];  // [16-key step][32-dim block][lane]
  u32 any[4];         // [wave that expanded them]: whether any of its values read as NaN,
  u32 nan[4][2];      // and which: two blocks of dims a word, a bit for each of the 8 tokens in its half
};
constexpr int kRowPad = kHeadDim + 8;  // elements of a row in the output's turn: 16 bytes of padding spread the banks

__global__ void __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(3)))
prefill_fp4_kernel(PrefillFp4Args a) {
  constexpr int D = kHeadDim;
  constexpr size_t kTurn = (size_t)kWaves * 16 * kRowPad * sizeof(u16);
  __shared__ __attribute__((aligned(16))) u8 s_mem[2 * sizeof(Stage) > kTurn ? 2 * sizeof(Stage) : kTurn];
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

  // Normalise and write: the wave turns its rows around in LDS, 16 at a time, and stores whole 256-byte rows.
  asm volatile("" : "+v"(row));  // token and head anew: they would hold registers through the loop
  const int token = row / a.group, head = g * a.group + row - token * a.group;
  const float l_tot = sum_xor32(l_run);
  const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;
  u16 *so = reinterpret_cast<u16 *>(s_mem) + w * 16 * kRowPad;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    __syncthreads();
    if ((n >> 4) == part) {
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          u32x2 pk;
          pk[0] = pack_bf16x2(acc[db][4 * i4] * inv, acc[db][4 * i4 + 1] * inv);
          pk[1] = pack_bf16x2(acc[db][4 * i4 + 2] * inv, acc[db][4 * i4 + 3] * inv);
          *reinterpret_cast<u32x2 *>(so + (n & 15) * kRowPad + 32 * db + 8 * i4 + 4 * half) = pk;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + (lane >> 4);  // of the 16
      const int t = __shfl(token, 16 * part + r), h = __shfl(head, 16 * part + r);
      const u32x4 v = *reinterpret_cast<const u32x4 *>(so + r * kRowPad + 8 * (lane & 15));
      if (r0 + 16 * part + r < rows.rows)
        st16(a.out + (int64_t)(rows.q_start + t) * a.out_stride + (int64_t)h * D + 8 * (lane & 15), v);
    }
  }
}

// ------------------------------------------------------------------------------------------ strips
constexpr int kStripWaves = 4;
constexpr int kStripRows = 32;

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

__global__ void __launch_bounds__(kStripWaves * 64) __attribute__((amdgpu_waves_per_eu(3)))
prefill_strip_fp4_kernel(PrefillFp4Args a) {
  constexpr int D = kHeadDim;
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

  // The waves' results meet, 16 rows at a time.  Register i of acc[2 j + x] is dim 64 j + 32 (i / 8) + 16 x + 8 (i / 4
  // % 2) + 4 half + i % 4 of row n.
  l_run = sum_xor32(l_run);
  if (half == 0) {
    s_m[w][n] = -neg_ref;
    s_l[w][n] = l_run;
  }
  constexpr int kDims = 8;  // of a thread
  static_assert(kStripWaves * 64 * kDims == kStripRows / 2 * D);
  const int r = threadIdx.x / (D / kDims), d0 = threadIdx.x % (D / kDims) * kDims;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    if ((n >> 4) == part) {
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<f32x4 *>(&s_o[w][n & 15][64 * (db >> 1) + 32 * (i >> 3) + 16 * (db & 1) + 2 * (i & 4) + 4 * half]) =
              f32x4{acc[db][i], acc[db][i + 1], acc[db][i + 2], acc[db][i + 3]};
    }
    __syncthreads();
    const int rr = 16 * part + r;
    if (rows.first + rr < rows.rows) {
      float M = s_m[0][rr], den = 0.f, num[kDims];
#pragma unroll
      for (int x = 1; x < kStripWaves; ++x) M = fmaxf(M, s_m[x][rr]);
#pragma unroll
      for (int d = 0; d < kDims; ++d) num[d] = 0.f;
#pragma unroll
      for (int x = 0; x < kStripWaves; ++x) {
        const float f = fast_exp2(s_m[x][rr] - M);
        den += f * s_l[x][rr];
#pragma unroll
        for (int d = 0; d < kDims; ++d) num[d] += f * s_o[x][r][d0 + d];
      }
      if (cut.pieces > 1) {
        float *rec = record(a, kStripRows, g, piece, rows.first + rr);
        if (d0 == 0) *reinterpret_cast<f32x2 *>(rec) = f32x2{M, den};
#pragma unroll
        for (int d = 0; d < kDims; d += 4)
          *reinterpret_cast<f32x4 *>(rec + 4 + d0 + d) = f32x4{num[d], num[d + 1], num[d + 2], num[d + 3]};
      } else {
        const float inv = den > 0.f ? 1.f / den : 0.f;
        const int at = rows.first + rr, t = at / a.group, h = g * a.group + at - t * a.group;
        u32x4 v;
#pragma unroll
        for (int d = 0; d < 4; ++d) v[d] = pack_bf16x2(num[2 * d] * inv, num[2 * d + 1] * inv);
        st16(a.out + (int64_t)(rows.q_start + t) * a.out_stride + (int64_t)h * D + d0, v);
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------ few rows
// Dims 4 dl .. 4 dl + 3 of the workgroup's row r.
__device__ __forceinline__ void write_quad(const PrefillFp4Args &a, const Rows &rows, int g, int r, int dl, f32x4 num,
                                           float den) {
  const float inv = den > 0.f ? 1.f / den : 0.f;
  const int t = (rows.first + r) / a.group, h = g * a.group + rows.first + r - t * a.group;
  *reinterpret_cast<u32x2 *>(a.out + (int64_t)(rows.q_start + t) * a.out_stride + (int64_t)h * kHeadDim + 4 * dl) =
      u32x2{pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv)};
}

constexpr int kFewWaves = 8;
constexpr int kFewRows = 16;

__global__ void __launch_bounds__(kFewWaves * 64) __attribute__((amdgpu_waves_per_eu(3)))
prefill_few_fp4_kernel(PrefillFp4Args a) {
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

  // Register i of o[e] is dim 16 e + 4 gq + i of row n.
  l = sum_over_quarters(l);
#pragma unroll
  for (int e = 0; e < 8; ++e) *reinterpret_cast<f32x4 *>(&s_o[w][n * kRec + 16 * e + 4 * gq]) = o[e];
  if (gq == 0) {
    s_m[w][n] = m;
    s_l[w][n] = l;
  }
  __syncthreads();
  // A half-wave takes a row, its lane dims 4 dl .. 4 dl + 3.
  static_assert(2 * kFewWaves == kFewRows);
  const int r = threadIdx.x >> 5, dl = lane & 31;
  float M = s_m[0][r], den = 0.f;
#pragma unroll
  for (int x = 1; x < kFewWaves; ++x) M = fmaxf(M, s_m[x][r]);
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int x = 0; x < kFewWaves; ++x) {
    const float f = fast_exp2(s_m[x][r] - M);
    num += f * *reinterpret_cast<const f32x4 *>(&s_o[x][r * kRec + 4 * dl]);
    den += f * s_l[x][r];
  }
  if (rows.first + r >= rows.rows) return;
  if (cut.pieces > 1) {
    float *rec = record(a, kFewRows, g, piece, rows.first + r);
    if (dl == 0) *reinterpret_cast<f32x2 *>(rec) = f32x2{M, den};
    *reinterpret_cast<f32x4 *>(rec + 4 + 4 * dl) = num;
  } else {
    write_quad(a, rows, g, r, dl, num, den);
  }
}

// ------------------------------------------------------------------------------------------ pieces
// Joins the pieces of the rows whose keys were cut: 8 rows of a group a workgroup, a half-wave each, its lane dims 4 dl
// .. 4 dl + 3.  The records of kRun pieces load together.
constexpr int kRun = 8;

__global__ void __launch_bounds__(256)
prefill_join_fp4_kernel(PrefillFp4Args a, int per_group) {
  Rows rows;
  if (!find_rows(a, per_group, blockIdx.y / (per_group / 8), rows)) return;
  const int g = blockIdx.x, dl = threadIdx.x & 31, r = blockIdx.y % (per_group / 8) * 8 + (threadIdx.x >> 5);
  if (rows.first + r >= rows.rows) return;
  const Cut cut = find_cut(a, rows, per_group);
  if (cut.pieces == 1) return;
  const int64_t stride = (int64_t)a.max_tiles * per_group * kRec;  // from a piece's record to the next one's
  const float *rec = record(a, per_group, g, 0, rows.first + r);
  float M = kNoScore, den = 0.f;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int y0 = 0; y0 < cut.pieces; y0 += kRun) {
    f32x2 ml[kRun];
    f32x4 v[kRun];
#pragma unroll
    for (int y = 0; y < kRun; ++y) {
      const float *p = rec + min(y0 + y, cut.pieces - 1) * stride;
      ml[y] = *reinterpret_cast<const f32x2 *>(p);
      v[y] = *reinterpret_cast<const f32x4 *>(p + 4 + 4 * dl);
    }
    float up = M;
#pragma unroll
    for (int y = 0; y < kRun; ++y) up = fmaxf(up, ml[y][0]);  // the last piece's again past the end
    const float f_old = fast_exp2(M - up);
    num *= f_old;
    den *= f_old;
#pragma unroll
    for (int y = 0; y < kRun; ++y) {
      if (y0 + y >= cut.pieces) break;
      const float f = fast_exp2(ml[y][0] - up);
      num += f * v[y];
      den += f * ml[y][1];
    }
    M = up;
  }
  write_quad(a, rows, g, r, dl, num, den);
}

// Which kernel, by the workgroups that the bounds of a call allow (few sequences are as long as the longest).  us, few
// rows / strips / tiles, 16 query and 8 kv heads unless given:
//   1 x 20 rows on 4,096 cached   20 /  32 / 132        1 x 1,000 on 4,096    87 /  60 / 163
//   1 x 100 on 4,096              21 /  32 / 135        1 x 4,000 on none    171 /  96 / 151
//   the same, 40 and 8 heads      21 /  34 / 134        4 x 2,000 on 1,152     - / 194 / 194 (1,000 workgroups of tiles)
//   1 x 300 on none               10 / 8.7 /  16        3 x 3,000 on none      - / 163 / 146 (1,128)
//   8 x 64 on 1,040               19 /  15 /  41        16 x 2,000 on 1,152    - / 698 / 642 (4,096)
// Few rows: while one round over the CUs takes them all.  Tiles: from four workgroups a CU on; before, whole CUs wait
// for the longest rows.
constexpr int64_t kFewGroups = 256;
constexpr int64_t kStripGroups = 1024;  // of the tile kernel

// Where few rows or strips leave the card idle and contexts may be long, the keys are cut until the workgroups fill it
// once, at most kMaxSplits times, and a second kernel joins the pieces (some 3 us).  us, uncut / cut: 1 x 20 rows on
// 4,096 keys 20 / 12.4, 2 x 20 on 8,192 35 / 17.6, 1 x 300 on 8,192 61 / 44, 1 x 600 on 8,192 93 / 79.  Few rows take a
// CU each, strips a third of one (with half: 45 and 93).
constexpr int kSplitFrom = 4096;  // keys that the block tables hold
constexpr int kMaxSplits = 32;

struct Plan {
  int rows;  // of a workgroup: kFewRows, kStripRows or kTileRows
  int64_t tiles;
  int splits;
  size_t workspace;
};
Plan plan_prefill(int64_t n_seqs, int64_t max_rows, int64_t num_kv_heads, int64_t cap) {
  const int64_t units = n_seqs * num_kv_heads;
  const auto tiles_of = [&](int rows) { return (max_rows + rows - 1) / rows; };
  Plan p;
  int64_t slots = 0;  // workgroups that the card holds at once
  if (tiles_of(kFewRows) * units <= kFewGroups) {
    p.rows = kFewRows;
    slots = 256;
  } else if (tiles_of(kTileRows) * units <= kStripGroups) {
    p.rows = kStripRows;
    slots = 3 * 256;
  } else {
    p.rows = kTileRows;
  }
  p.tiles = tiles_of(p.rows);
  const int64_t wanted = cap < kSplitFrom ? 1 : min(slots / (p.tiles * units), min(cap / kMinSplit, (int64_t)kMaxSplits));
  p.splits = (int)max(wanted, (int64_t)1);
  p.workspace = p.splits == 1 ? 0 : (size_t)(units * p.splits * p.tiles * p.rows) * kRec * sizeof(float);
  return p;
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" size_t nvamd_paged_prefill_fp4_workspace_size(int n_seqs, int max_q_len, int num_heads, int num_kv_heads,
                                                         int block_size, int bt_width) {
  if (n_seqs <= 0 || max_q_len <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads || block_size <= 0 || bt_width <= 0)
    return 0;
  return plan_prefill(n_seqs, (int64_t)max_q_len * (num_heads / num_kv_heads), num_kv_heads,
                      (int64_t)bt_width * block_size)
      .workspace;
}

extern "C" int nvamd_paged_prefill_fp4(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                       const void *k_codes, const void *k_scales, const void *v_codes,
                                       const void *v_scales, int num_blocks, int block_size,
                                       const int32_t *block_tables, int bt_stride, int bt_width,
                                       const int32_t *cu_seqlens_q, const int32_t *kv_lens, int n_seqs, int num_tokens,
                                       int max_q_len, int num_heads, int num_kv_heads, int head_dim, float scale,
                                       void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (n_seqs == 0 || max_q_len == 0 || num_tokens == 0) return NVAMD_OK;
  const int bs_log2 = log2_exact(block_size);
  if (head_dim != kHeadDim || bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!(scale > 0.f)) return NVAMD_EINVAL;  // the softmax keeps its running max on raw scores
  if (!out || !q || !fp4_cache_ok(k_codes, k_scales, v_codes, v_scales) || !block_tables || !cu_seqlens_q || !kv_lens ||
      n_seqs < 0 || num_tokens < 0 || max_q_len < 0 || num_blocks <= 0 || num_kv_heads <= 0 || num_heads <= 0 ||
      num_heads % num_kv_heads != 0 || bt_width <= 0 || bt_stride < bt_width || n_seqs > 65535 || !aligned16(q) ||
      !aligned16(out) || q_stride % 8 || out_stride % 8 || q_stride < (int64_t)num_heads * head_dim ||
      out_stride < (int64_t)num_heads * head_dim)
    return NVAMD_EINVAL;
  if (((int64_t)bt_width << bs_log2) > 1 << 30 || (((int64_t)num_blocks * num_kv_heads) << bs_log2) >> 4 > 0x7fffffff)
    return NVAMD_EUNSUPPORTED;
  PrefillFp4Args a = {};
  a.out = static_cast<u16 *>(out);
  a.out_stride = out_stride;
  a.q = static_cast<const u16 *>(q);
  a.q_stride = q_stride;
  a.cache = Fp4Cache{const_cast<u8 *>(static_cast<const u8 *>(k_codes)),
                     const_cast<u8 *>(static_cast<const u8 *>(k_scales)),
                     const_cast<u8 *>(static_cast<const u8 *>(v_codes)),
                     const_cast<u8 *>(static_cast<const u8 *>(v_scales))};
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.bt_width = bt_width;
  a.num_blocks = num_blocks;
  a.bs_log2 = bs_log2;
  a.cu_seqlens_q = cu_seqlens_q;
  a.kv_lens = kv_lens;
  a.num_kv_heads = num_kv_heads;
  a.max_q_len = max_q_len;
  a.num_tokens = num_tokens;
  a.scale_log2e = scale * kLog2e;
  a.err = index_error_word();
  a.group = num_heads / num_kv_heads;
  const int64_t max_rows = (int64_t)max_q_len * a.group;
  if (max_rows > 0x7fffffff) return NVAMD_EUNSUPPORTED;
  const Plan plan = plan_prefill(n_seqs, max_rows, num_kv_heads, (int64_t)bt_width << bs_log2);
  if (plan.tiles > 65535) return NVAMD_EUNSUPPORTED;
  a.max_tiles = (int)plan.tiles;
  a.splits = 1;
  if (workspace != nullptr && plan.splits > 1) {
    if (workspace_bytes < plan.workspace) return NVAMD_EWORKSPACE;
    if (!aligned16(workspace)) return NVAMD_EINVAL;
    a.splits = plan.splits;
    a.partials = static_cast<float *>(workspace);
  }
  const dim3 grid(num_kv_heads * a.splits, a.max_tiles, n_seqs);
  if (plan.rows == kFewRows)
    hipLaunchKernelGGL(prefill_few_fp4_kernel, grid, dim3(kFewWaves * 64), 0, stream, a);
  else if (plan.rows == kStripRows)
    hipLaunchKernelGGL(prefill_strip_fp4_kernel, grid, dim3(kStripWaves * 64), 0, stream, a);
  else
    hipLaunchKernelGGL(prefill_fp4_kernel, grid, dim3(kWaves * 64), 0, stream, a);
  if (a.splits > 1) {
    const int st = launch_status();
    if (st != NVAMD_OK) return st;
    a.err = nullptr;  // the faults have been reported
    hipLaunchKernelGGL(prefill_join_fp4_kernel, dim3(num_kv_heads, a.max_tiles * (plan.rows / 8), n_seqs), dim3(256), 0,
                       stream, a, plan.rows);
  }
  return launch_status();
}
