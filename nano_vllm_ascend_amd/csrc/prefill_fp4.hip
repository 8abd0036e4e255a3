// Causal prefill attention over the 4-bit paged KV cache (the counterpart of prefill.hip's paged route): the queries are
// the last q_len positions of a context of kv_len, query row r sees keys 0 .. kv_len - q_len + r, all of them in the cache.
//
// Workgroup = 4 waves = one kv head, 1, 2 or 4 of its query heads, and 128 / heads query tokens; wave w owns 32 query rows of
// one head.  Per tile of 32 keys the workgroup expands K and V from 4 bits to bf16 once, into LDS, in the order in
// which the MFMA operands are read (every operand read is 64 lanes x 16 consecutive bytes: no bank conflicts, no
// swizzle), while the codes of the tile after the next are on their way into registers:
//   waves 0, 1: thread (quarter, row) expands 16 bytes of codes, one block of a K row under one scale, to four chunks of
//        8 dims;
//   waves 2, 3: thread (dim pair) of a 16-token tile expands 16 bytes, the tile's tokens of two dims, each under its token's
//        scale, and pairs tokens: four chunks of 8 keys of a dim.
// Then, as in prefill.hip:
//   S^T[32 keys x 32 queries] = K . Q^T        v_mfma_f32_32x32x16_bf16, Q in registers throughout;
//   O^T[128 dims x 32 queries] += V^T . P^T    with the k-slots in the order in which the S^T accumulator holds its rows,
//        so that P^T is a repack in registers.
// A block of values that reads as NaN must reach the rows that see its key and no others, though masked rows
// multiply it by a weight of zero: such values enter the products as zeros, and the rows that see
// the key get the NaN added afterwards (a branch that no other tile takes).
#include "fp4.h"

namespace nvamd {
namespace {

constexpr int kBK = 32;               // keys per tile
constexpr float kRescaleLog2 = 8.f;   // lazy-rescale threshold (log2 units)
constexpr u32 kBf16PairOne = 0x3F803F80u;
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;

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
  int max_q_tiles;
  int max_q_len;
  int num_tokens;
  float scale_log2e;
  int q_group;  // query heads of kv head g: q_group * g + q_head0 + (0 .. GQA-1)
  int q_head0;
  u32 *err;
};

__device__ __forceinline__ f32x16 mfma32(bf16x8v a, bf16x8v b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int B>
__device__ __forceinline__ float scale_of(u32 word) {
  return __uint_as_float(((word >> (8 * B)) & 0xffu) << 23);
}

// One stage: the operands of a tile, each 64 lanes x 16 bytes, and a bit per (block, token) whose values read as NaN.
struct Stage {
  u32x4 k[8][64];     // [16-dim step][lane]
  u32x4 v[2][4][64];  // [16-key step][32-dim block][lane]
  u16 nan[2][4];      // [16-key step][32-dim block]: bit per token
};

template <int GQA>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
prefill_fp4_kernel(PrefillFp4Args a) {
  constexpr int D = kHeadDim;
  constexpr int BQ = 32 * kWaves / GQA;  // query tokens per workgroup
  constexpr int WPH = kWaves / GQA;      // waves per query head
  __shared__ __attribute__((aligned(16))) Stage s_stage[2];

  const int g = blockIdx.x;
  const int qt = a.max_q_tiles - 1 - (int)blockIdx.y;
  const int s = blockIdx.z;
  const int q_start = a.cu_seqlens_q[s];
  const int q_end = a.cu_seqlens_q[s + 1];
  const int q_len = q_end - q_start;
  const int cap = a.bt_width << a.bs_log2;
  int kv_len = a.kv_lens[s];
  const bool rows_in = q_start >= 0 && q_len >= 0 && q_end <= a.num_tokens;  // else no row is touched
  if ((!rows_in || q_len > a.max_q_len || kv_len > cap || kv_len < q_len) && g == 0 && blockIdx.y == 0 &&
      threadIdx.x == 0)
    flag_index_error(a.err, NVAMD_ERR_CONTEXT);
  if (!rows_in || qt * BQ >= q_len) return;
  kv_len = min(kv_len, cap);
  const int offset = kv_len - q_len;  // query row r sees keys 0..offset+r

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5;
  const int n = lane & 31;  // this lane's query column
  const int head = g * a.q_group + a.q_head0 + w / WPH;
  const int r0 = qt * BQ + (w % WPH) * 32;  // first query row of this wave
  const int rq = r0 + n;

  bf16x8v qf[8];  // dims 16 kk + 8 hl .. +7 of the lane's query row
  {
    const u16 *qp = a.q + (int64_t)(q_start + min(rq, q_len - 1)) * a.q_stride + (int64_t)head * D + 8 * hl;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) qf[kk] = __builtin_bit_cast(bf16x8v, ld16(qp + 16 * kk));
  }
  f32x16 acc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
  float m_ref = -1e30f, m_thr = -1e30f, neg_ref = 1e30f, l_run = 0.f;

  // Keys this workgroup needs: up to the last visible key of its last valid row.
  const int kv_hi = min(kv_len, offset + min((qt + 1) * BQ, q_len));
  const int n_tiles = kv_hi > 0 ? ceil_div(kv_hi, kBK) : 0;
  const int wave_last_key = offset + min(r0 + 31, q_len - 1);  // beyond: fully masked for this wave

  const int32_t *bt_row = a.block_tables + (int64_t)s * a.bt_stride;
  const int bs_mask = (1 << a.bs_log2) - 1;
  // The 16-token tile of token t0 (the last one of the keys where t0 lies past them).
  auto tile_at = [&](int t0) {
    const int t = min(t0, (kv_len - 1) & ~15);
    const int e = bt_row[t >> a.bs_log2];
    if ((unsigned)e >= (unsigned)a.num_blocks && lane == 0) flag_index_error(a.err, NVAMD_ERR_BLOCK);
    return fp4_tile(min(max(e, 0), a.num_blocks - 1), t & bs_mask, g, a.num_kv_heads, a.bs_log2);
  };

  // What a thread expands: waves 0 and 1 row n of block 2w + hl of K, waves 2 and 3 the dim pair `lane` of tile w - 2.
  u32x4 codes, scales;
  auto fetch = [&](int t) {
    if (w < 2) {
      const int64_t t0 = tile_at(t * kBK), t1 = tile_at(t * kBK + 16);
      const int64_t tile = n < 16 ? t0 : t1;
      codes = *reinterpret_cast<const u32x4 *>(a.cache.k_codes + tile * kFp4TileBytes + (n & 15) * kFp4RowBytes +
                                               16 * (2 * w + hl));
      scales[0] = a.cache.k_scales[tile * kFp4TileScales + fp4_key_scale_at(n & 15, 2 * w + hl)];
    } else {
      const int64_t tile = tile_at(t * kBK + 16 * (w - 2));
      codes = *reinterpret_cast<const u32x4 *>(a.cache.v_codes + tile * kFp4TileBytes + 16 * lane);
      scales = *reinterpret_cast<const u32x4 *>(a.cache.v_scales + tile * kFp4TileScales + 16 * (lane >> 4));
    }
  };
  auto expand = [&](int t, Stage &st) {
    if (w < 2) {
      const float scale = fp4_scale(scales[0]);
      const int q = 2 * w + hl;
#pragma unroll
      for (int c = 0; c < 4; ++c) st.k[2 * q + (c >> 1)][32 * (c & 1) + n] = fp4_values(codes[c], scale);
    } else {
      // Blocks that read as NaN become zeros, and are noted where their token exists.
      u32 seen = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        // 0x80 in the bytes that are 255: only there do the low seven bits carry into a set top bit
        const u32 bad = ((scales[x] & 0x7f7f7f7fu) + 0x01010101u) & scales[x] & 0x80808080u;
        if (__builtin_expect(bad != 0, 0)) {
          scales[x] &= ~((bad >> 7) * 0xffu);
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if ((bad >> (8 * b + 7)) & 1) seen |= 1u << (4 * x + b);
        }
      }
      const int left = kv_len - t * kBK - 16 * (w - 2);
      if (left < 16) seen &= (1u << max(left, 0)) - 1u;
      if ((lane & 15) == 0) st.nan[w - 2][lane >> 4] = (u16)seen;
      u32x4 lo[2], hi[2];  // [k-slot half of the operand] of dims r and r + 16
#pragma unroll
      for (int x = 0; x < 4; ++x) {  // word x: tokens 4x .. 4x+3, which half x % 2 of the lanes takes at place x / 2
        const u32 v0 = fp4_pair<0>(codes[x], scale_of<0>(scales[x])), v1 = fp4_pair<1>(codes[x], scale_of<1>(scales[x]));
        const u32 v2 = fp4_pair<2>(codes[x], scale_of<2>(scales[x])), v3 = fp4_pair<3>(codes[x], scale_of<3>(scales[x]));
        lo[x & 1][2 * (x >> 1)] = pair_lo(v0, v1);
        lo[x & 1][2 * (x >> 1) + 1] = pair_lo(v2, v3);
        hi[x & 1][2 * (x >> 1)] = pair_hi(v0, v1);
        hi[x & 1][2 * (x >> 1) + 1] = pair_hi(v2, v3);
      }
      u32x4 *dst = st.v[w - 2][lane >> 4];
      const int r = lane & 15;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        dst[32 * h + r] = lo[h];
        dst[32 * h + 16 + r] = hi[h];
      }
    }
  };

  auto compute = [&](int t, const Stage &st) {
    const int base = t * kBK;
    if (r0 >= q_len || base > wave_last_key) return;
    f32x16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) sc = mfma32(__builtin_bit_cast(bf16x8v, st.k[kk][lane]), qf[kk], sc);
    // Key of register i: base + 8(i/4) + 4hl + i%4.
    const int lim = min(offset + rq, kv_len - 1) - base - 4 * hl;
    const bool need_mask = (base + kBK - 1 > offset + r0) || (base + kBK > kv_len);
    if (__builtin_expect(need_mask, 0)) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + (i % 4) > lim) sc[i] = -INFINITY;
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, sc[i]);
    tmax = max_xor32(tmax) * a.scale_log2e;
    if (__builtin_amdgcn_ballot_w64(tmax > m_thr) != 0) {
      const bool up = tmax > m_thr;
      const float alpha = up ? __builtin_amdgcn_exp2f(m_ref - tmax) : 1.f;
      if (up) {
        m_ref = tmax;
        m_thr = tmax + kRescaleLog2;
        neg_ref = -tmax;
      }
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
    }
    bf16x8v pf[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      u32x4 packed;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32 pr = pack_bf16x2(__builtin_amdgcn_exp2f(fmaf(sc[8 * hh + 2 * e], a.scale_log2e, neg_ref)),
                                   __builtin_amdgcn_exp2f(fmaf(sc[8 * hh + 2 * e + 1], a.scale_log2e, neg_ref)));
        l_run = dot2_bf16(pr, kBf16PairOne, l_run);  // both rounded values of the pair
        packed[e] = pr;
      }
      pf[hh] = __builtin_bit_cast(bf16x8v, packed);
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int db = 0; db < 4; ++db) acc[db] = mfma32(__builtin_bit_cast(bf16x8v, st.v[hh][db][lane]), pf[hh], acc[db]);
    const u32x4 nan = *reinterpret_cast<const u32x4 *>(&st.nan[0][0]);
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(nan[0] | nan[1] | nan[2] | nan[3]) != 0, 0)) {
      const int seen = min(offset + rq, kv_len - 1) - base;  // the last key of the tile that this lane's row sees
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const u32 bits = (u32)st.nan[0][db] | ((u32)st.nan[1][db] << 16);
        const bool hit = seen >= 0 && (bits & (seen >= 31 ? 0xffffffffu : (2u << seen) - 1u)) != 0;
        if (hit) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[db][i] = NAN;
        }
      }
    }
  };

  // Tile t is computed from stage t % 2 while the other stage takes tile t + 1, whose codes were fetched during tile t - 1.
  if (n_tiles > 0) {
    fetch(0);
    expand(0, s_stage[0]);
    if (n_tiles > 1) fetch(1);
  }
  __syncthreads();
  for (int t = 0; t < n_tiles; ++t) {
    if (t + 1 < n_tiles) {
      expand(t + 1, s_stage[(t + 1) & 1]);
      if (t + 2 < n_tiles) fetch(t + 2);
    }
    compute(t, s_stage[t & 1]);
    __syncthreads();
  }

  // Normalise and write: the wave turns its 32 rows around in LDS and stores whole 256-byte rows.
  const float l_tot = sum_xor32(l_run);
  const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;
  constexpr int kRow = D + 8;  // elements: 16 bytes of padding spread the rows over the banks
  static_assert(sizeof(s_stage) >= (size_t)kWaves * 16 * kRow * sizeof(u16), "16 rows of every wave");
  u16 *so = reinterpret_cast<u16 *>(&s_stage[0]) + w * 16 * kRow;
  const int rows = min(q_len - r0, 32);
#pragma unroll
  for (int half = 0; half < 2; ++half) {  // 16 query rows at a time
    __syncthreads();
    if ((n >> 4) == half) {
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          u32x2 pk;
          pk[0] = pack_bf16x2(acc[db][4 * i4] * inv, acc[db][4 * i4 + 1] * inv);
          pk[1] = pack_bf16x2(acc[db][4 * i4 + 2] * inv, acc[db][4 * i4 + 3] * inv);
          *reinterpret_cast<u32x2 *>(so + (n & 15) * kRow + 32 * db + 8 * i4 + 4 * hl) = pk;
        }
    }
    __syncthreads();
    u16 *op = a.out + (int64_t)(q_start + r0 + 16 * half) * a.out_stride + (int64_t)head * D + 8 * (lane & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + (lane >> 4);
      const u32x4 v = *reinterpret_cast<const u32x4 *>(so + r * kRow + 8 * (lane & 15));
      if (16 * half + r < rows) st16(op + (int64_t)r * a.out_stride, v);
    }
  }
}

template <int GQA>
int launch(const PrefillFp4Args &a, int n_seqs, hipStream_t stream) {
  hipLaunchKernelGGL((prefill_fp4_kernel<GQA>), dim3(a.num_kv_heads, a.max_q_tiles, n_seqs), dim3(kThreads), 0, stream,
                     a);
  return launch_status();
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" int nvamd_paged_prefill_fp4(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                       const void *k_codes, const void *k_scales, const void *v_codes,
                                       const void *v_scales, int num_blocks, int block_size,
                                       const int32_t *block_tables, int bt_stride, int bt_width,
                                       const int32_t *cu_seqlens_q, const int32_t *kv_lens, int n_seqs, int num_tokens,
                                       int max_q_len, int num_heads, int num_kv_heads, int head_dim, float scale, hipStream_t stream) {
  if (n_seqs == 0 || max_q_len == 0) return NVAMD_OK;
  const int bs_log2 = log2_exact(block_size);
  if (head_dim != kHeadDim || bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!(scale > 0.f)) return NVAMD_EINVAL;  // the softmax keeps its running max on raw scores
  if (!out || !q || !fp4_cache_ok(k_codes, k_scales, v_codes, v_scales) || !block_tables || !cu_seqlens_q || !kv_lens ||
      n_seqs < 0 || num_tokens < 0 || max_q_len < 0 || num_blocks <= 0 || num_kv_heads <= 0 || num_heads <= 0 ||
      num_heads % num_kv_heads != 0 || bt_width <= 0 || bt_stride < bt_width || n_seqs > 65535 || !aligned16(q) ||
      !aligned16(out) || q_stride % 8 || out_stride % 8 || q_stride < (int64_t)num_heads * head_dim ||
      out_stride < (int64_t)num_heads * head_dim)
    return NVAMD_EINVAL;
  if (((int64_t)bt_width << bs_log2) > 0x7fffffff) return NVAMD_EUNSUPPORTED;
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
  a.q_group = num_heads / num_kv_heads;
  // A workgroup takes 4, 2 or 1 heads of a group; other ratios run as consecutive launches over 4, then 2, then 1.
  for (int rest = a.q_group; rest > 0;) {
    const int sub = rest >= 4 ? 4 : rest >= 2 ? 2 : 1;
    a.q_head0 = a.q_group - rest;
    a.max_q_tiles = ceil_div(max_q_len, 32 * kWaves / sub);
    if (a.max_q_tiles > 65535) return NVAMD_EUNSUPPORTED;
    const int st = sub == 4 ? launch<4>(a, n_seqs, stream) : sub == 2 ? launch<2>(a, n_seqs, stream)
                                                                      : launch<1>(a, n_seqs, stream);
    if (st != NVAMD_OK) return st;
    rest -= sub;
  }
  return NVAMD_OK;
}
