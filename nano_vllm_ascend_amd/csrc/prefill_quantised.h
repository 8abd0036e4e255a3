// Causal prefill attention over a quantised paged cache: what the kernels of the 4-bit and of the 8-bit cache share -- a
// workgroup's rows and keys, the query, the ways out, the join of rows whose keys were cut, and which kernel a call takes.
//
// The queries are the last q_len positions of a context of kv_len, query row r sees keys 0 .. kv_len - q_len + r, all of
// them in the cache.  The G query heads of a kv head and the q_len tokens make q_len * G rows, R = token * G + head, that
// share the keys; a workgroup takes rows that follow one another, whatever G is.
#pragma once

#include "attention_tiles.h"

namespace nvamd {

template <typename Cache>
struct PrefillArgs {
  u16 *out;
  int64_t out_stride;
  const u16 *q;
  int64_t q_stride;
  Cache cache;
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
template <typename Args>
__device__ __forceinline__ bool find_rows(const Args &a, int per_group, int y, Rows &r) {
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
template <typename Args>
__device__ __forceinline__ Cut find_cut(const Args &a, const Rows &r, int per_group) {
  const int keys = max(min(r.kv_len, r.offset + (min(r.first + per_group, r.rows) - 1) / a.group + 1), 0);
  if (a.splits == 1) return {keys, keys, 1};
  const int length = max(ceil_div(ceil_div(keys, a.splits), kMinSplit), 1) * kMinSplit;
  return {keys, length, max(ceil_div(keys, length), 1)};
}
template <typename Args>
__device__ __forceinline__ float *record(const Args &a, int per_group, int g, int piece, int row) {
  const int64_t unit = ((int64_t)blockIdx.z * a.num_kv_heads + g) * a.splits + piece;
  return a.partials + (unit * (a.max_tiles * per_group) + row) * kRec;
}

// Index of the 16-token tile of the pool that holds a token whose page is `entry`.  (A pool has less than 2^31.)  WIDE: by
// way of the 64-bit index of the token, which the 4-bit cache's strips are scheduled better around (us, 32 / 64 bits: 8 x
// 1..64 on 1,040 13.2 / 13.0, 1 x 1,000 on 4,096 54.5 / 53.3), its tiles (701 / 708) and the 8-bit cache's strips (25.2 /
// 25.9) worse.
template <bool WIDE = false, typename Args>
__device__ __forceinline__ int tile_of(const Args &a, int entry, int token, int g, bool report) {
  if ((unsigned)entry >= (unsigned)a.num_blocks && report) flag_index_error(a.err, NVAMD_ERR_BLOCK);
  entry = min(max(entry, 0), a.num_blocks - 1);  // never leave the pool
  if constexpr (WIDE)
    return (int)(((((int64_t)entry * a.num_kv_heads + g) << a.bs_log2) + (token & ((1 << a.bs_log2) - 1))) >> 4);
  return (int)((((u32)entry * (u32)a.num_kv_heads + (u32)g) << (a.bs_log2 - 4)) + ((u32)(token & ((1 << a.bs_log2) - 1)) >> 4));
}

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0,
                                                 0, 0);
}
// A row's operands: dims 64 s + 16 half .. +15 and 64 s + 32 + 16 half .. +15, the scales of block 2 s + half.
template <typename Args>
__device__ __forceinline__ void load_query(const Args &a, const Rows &rows, int row, int g, int half,
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

// ------------------------------------------------------------------------------------------ tiles
constexpr int kBK = 32;  // keys per tile
constexpr int kTileWaves = 4;
constexpr int kTileRows = 32 * kTileWaves;
constexpr int kRowPad = kHeadDim + 8;  // elements of a row in the output's turn: 16 bytes of padding spread the banks

// The end of the tile kernel, where wave w has rows r0 .. r0 + 31 and a lane row `row`: register i of acc[db] is dim 32 db
// + 8 (i / 4) + 4 half + i % 4 of it.  s_mem: kTurnBytes that every wave is done with.
constexpr size_t kTurnBytes = (size_t)kTileWaves * 16 * kRowPad * sizeof(u16);
template <typename Args>
__device__ __forceinline__ void write_tile_rows(const Args &a, const Rows &rows, int g, int r0, int row, int w, int lane,
                                                f32x16 (&acc)[4], float l_run, u8 *s_mem) {
  constexpr int D = kHeadDim;
  const int half = lane >> 5, n = lane & 31;
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

// The end of a strip, or of a piece of its keys: registers i .. i + 3 (i % 4 = 0) of acc[db] are dims dim_of(db, i, half)
// .. + 3 of row n.
template <typename Args, typename Dim>
__device__ __forceinline__ void write_strip(const Args &a, const Rows &rows, const Cut &cut, int piece, int g, int w, int lane,
                                            f32x16 (&acc)[4], float neg_ref, float l_run,
                                            float (&s_o)[kStripWaves][kStripRows / 2][kRec],
                                            float (&s_m)[kStripWaves][kStripRows], float (&s_l)[kStripWaves][kStripRows],
                                            Dim &&dim_of) {
  constexpr int D = kHeadDim;
  const int half = lane >> 5, n = lane & 31;
  // The waves' results meet, 16 rows at a time.
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
          *reinterpret_cast<f32x4 *>(&s_o[w][n & 15][dim_of(db, i, half)]) =
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
template <typename Args>
__device__ __forceinline__ void write_quad(const Args &a, const Rows &rows, int g, int r, int dl, f32x4 num,
                                           float den) {
  const float inv = den > 0.f ? 1.f / den : 0.f;
  const int t = (rows.first + r) / a.group, h = g * a.group + rows.first + r - t * a.group;
  *reinterpret_cast<u32x2 *>(a.out + (int64_t)(rows.q_start + t) * a.out_stride + (int64_t)h * kHeadDim + 4 * dl) =
      u32x2{pack_bf16x2(num[0] * inv, num[1] * inv), pack_bf16x2(num[2] * inv, num[3] * inv)};
}

constexpr int kFewWaves = 8;
constexpr int kFewRows = 16;

// The end of a few rows, or of a piece of their keys.
template <typename Args>
__device__ __forceinline__ void write_few(const Args &a, const Rows &rows, const Cut &cut, int piece, int g, int w, int lane,
                                          f32x4 (&o)[8], float m, float l, float (&s_o)[kFewWaves][kFewRows * kRec],
                                          float (&s_m)[kFewWaves][kFewRows], float (&s_l)[kFewWaves][kFewRows]) {
  const int n = lane & 15, gq = lane >> 4;
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

template <typename Args>
__global__ void __launch_bounds__(256)
prefill_join_kernel(Args a, int per_group) {
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
// rows / strips / tiles, 4-bit cache, 16 query and 8 kv heads unless given:
//   1 x 20 rows on 4,096 cached   20 /  32 / 132        1 x 1,000 on 4,096    87 /  60 / 163
//   1 x 100 on 4,096              21 /  32 / 135        1 x 4,000 on none    171 /  96 / 151
//   the same, 40 and 8 heads      21 /  34 / 134        4 x 2,000 on 1,152     - / 194 / 194 (1,000 workgroups of tiles)
//   1 x 300 on none               10 / 8.7 /  16        3 x 3,000 on none      - / 163 / 146 (1,128)
//   8 x 64 on 1,040               19 /  15 /  41        16 x 2,000 on 1,152    - / 698 / 642 (4,096)
// The 8-bit cache has the same borders: 1 x 20 on 4,096 11.0 / 13.9, 8 x 64 on 1,040 20.3 / 14.0, 1 x 4,000 on none - / 85
// / 120, 4 x 2,000 on 1,152 (1,024) - / 172 / 172, 5 x 2,000 on 1,152 (1,280) - / 214 / 209, 3 x 3,000 on none - / 150 /
// 129, 8 x 2,000 on none (2,048) - / 207 / 166, 16 x 2,000 on 1,152 - / 695 / 584.
// Few rows: while one round over the CUs takes them all.  Tiles: from four workgroups a CU on; before, whole CUs wait
// for the longest rows.
constexpr int64_t kFewGroups = 256;
constexpr int64_t kStripGroups = 1024;  // of the tile kernel

// Where few rows or strips leave the card idle and contexts may be long, the keys are cut until the workgroups fill it
// once, at most kMaxSplits times, and a second kernel joins the pieces (some 3 us).  us, uncut / cut: 1 x 20 rows on
// 4,096 keys 20 / 12.4, 2 x 20 on 8,192 35 / 17.6, 1 x 300 on 8,192 61 / 44, 1 x 600 on 8,192 93 / 79.  Few rows take a
// CU each; of strips a CU holds STRIPS_ON_CU: three of the 4-bit cache's (cut for two: 45 and 93), two of the 8-bit
// cache's (cut for two / for three: 1 x 300 on 4,096 24.5 / 31.0, on 8,192 37.8 / 43.2, on 16,384 57.7 / 67.3; 3 x 100 on
// 4,096 25.8 / 33.6).
// Between one and two whole strips a CU, halves in a round and a half take less than one uneven round, but only of long
// contexts (8-bit cache, uncut / halves: 1 x 600 on 8,192 69.5 / 72.4, on 16,384 127.6 / 123.4, on 30,000 224.7 / 207.6).
constexpr int kSplitFrom = 4096;    // keys that the block tables hold
constexpr int kHalvesFrom = 16384;
constexpr int kMaxSplits = 32;

struct Plan {
  int rows;  // of a workgroup: kFewRows, kStripRows or kTileRows
  int64_t tiles;
  int splits;
  size_t workspace;
};
template <int STRIPS_ON_CU>
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
    slots = STRIPS_ON_CU * 256;
  } else {
    p.rows = kTileRows;
  }
  p.tiles = tiles_of(p.rows);
  const int64_t wanted = cap < kSplitFrom ? 1 : min(slots / (p.tiles * units), min(cap / kMinSplit, (int64_t)kMaxSplits));
  p.splits = (int)max(wanted, (int64_t)1);
  if (p.rows == kStripRows && cap >= kHalvesFrom && 2 * p.tiles * units <= 3 * 256) p.splits = max(p.splits, 2);
  p.workspace = p.splits == 1 ? 0 : (size_t)(units * p.splits * p.tiles * p.rows) * kRec * sizeof(float);
  return p;
}

// ------------------------------------------------------------------------------------------ a call
template <int STRIPS_ON_CU>
size_t prefill_workspace_bytes(int n_seqs, int max_q_len, int num_heads, int num_kv_heads, int block_size,
                                      int bt_width) {
  if (n_seqs <= 0 || max_q_len <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads || block_size <= 0 || bt_width <= 0)
    return 0;
  return plan_prefill<STRIPS_ON_CU>(n_seqs, (int64_t)max_q_len * (num_heads / num_kv_heads), num_kv_heads,
                      (int64_t)bt_width * block_size)
      .workspace;
}

// Checks and launches; few, strip and tiles are the kernels.
template <int STRIPS_ON_CU, typename Cache>
int prefill(void (*few)(PrefillArgs<Cache>), void (*strip)(PrefillArgs<Cache>), void (*tiles)(PrefillArgs<Cache>),
            const Cache &cache, bool cache_ok, void *out, int64_t out_stride, const void *q, int64_t q_stride,
            int num_blocks, int block_size, const int32_t *block_tables, int bt_stride, int bt_width,
            const int32_t *cu_seqlens_q, const int32_t *kv_lens, int n_seqs, int num_tokens, int max_q_len, int num_heads,
            int num_kv_heads, int head_dim, float scale, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (n_seqs == 0 || max_q_len == 0 || num_tokens == 0) return NVAMD_OK;
  const int bs_log2 = log2_exact(block_size);
  if (head_dim != kHeadDim || bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!(scale > 0.f)) return NVAMD_EINVAL;  // the softmax keeps its running max on raw scores
  if (!out || !q || !cache_ok || !block_tables || !cu_seqlens_q || !kv_lens ||
      n_seqs < 0 || num_tokens < 0 || max_q_len < 0 || num_blocks <= 0 || num_kv_heads <= 0 || num_heads <= 0 ||
      num_heads % num_kv_heads != 0 || bt_width <= 0 || bt_stride < bt_width || n_seqs > 65535 || !aligned16(q) ||
      !aligned16(out) || q_stride % 8 || out_stride % 8 || q_stride < (int64_t)num_heads * head_dim ||
      out_stride < (int64_t)num_heads * head_dim)
    return NVAMD_EINVAL;
  if (((int64_t)bt_width << bs_log2) > 1 << 30 || (((int64_t)num_blocks * num_kv_heads) << bs_log2) >> 4 > 0x7fffffff)
    return NVAMD_EUNSUPPORTED;
  using Args = PrefillArgs<Cache>;
  Args a = {};
  a.out = static_cast<u16 *>(out);
  a.out_stride = out_stride;
  a.q = static_cast<const u16 *>(q);
  a.q_stride = q_stride;
  a.cache = cache;
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
  const Plan plan = plan_prefill<STRIPS_ON_CU>(n_seqs, max_rows, num_kv_heads, (int64_t)bt_width << bs_log2);
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
    hipLaunchKernelGGL(few, grid, dim3(kFewWaves * 64), 0, stream, a);
  else if (plan.rows == kStripRows)
    hipLaunchKernelGGL(strip, grid, dim3(kStripWaves * 64), 0, stream, a);
  else
    hipLaunchKernelGGL(tiles, grid, dim3(kTileWaves * 64), 0, stream, a);
  if (a.splits > 1) {
    const int st = launch_status();
    if (st != NVAMD_OK) return st;
    a.err = nullptr;  // the faults have been reported
    hipLaunchKernelGGL(prefill_join_kernel<Args>, dim3(num_kv_heads, a.max_tiles * (plan.rows / 8), n_seqs), dim3(256), 0,
                       stream, a, plan.rows);
  }
  return launch_status();
}

}  // namespace nvamd
