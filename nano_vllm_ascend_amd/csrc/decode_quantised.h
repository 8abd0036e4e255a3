// Paged decode over a quantised cache: what the kernels of the 4-bit and of the 8-bit cache share -- how a call's contexts
// are cut into workgroups, the query, and how the results of waves and partitions meet.
//
// Work: a unit (sequence, kv head) is cut into partitions of equal length, a workgroup of WAVES waves each.  Every
// workgroup reads the context lengths and derives the same length from them (partition_tokens), so the cut follows the
// contexts themselves and not the bound that the launch was made with.  (A sequence of more than one step of the waves is
// so summed in an order that depends on the sequences beside it.)  A partition leaves (max, sum, numerator) per head in
// the workspace and counts its arrival; the last one of a unit joins them.
#pragma once

#include "attention_tiles.h"
#include "decode_workspace.h"
#include "norm_rope64.h"

#include <type_traits>

namespace nvamd {

constexpr int kCus = 256;
constexpr int kMaxHeads = 16;  // query heads of a kv head in one launch: the MFMA's columns
template <typename Cache>
struct DecodeArgs {
  u16 *out;
  int64_t out_stride;
  const u16 *q;
  int64_t q_stride;
  Cache cache;
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

// Cutting units of `tokens` tokens in all every `length` tokens ends in tokens / length + units / 2 partitions on
// average, and in a whole unit more than the quotient each at most.  The length is chosen for this quotient (share):
//   few units: partitions fill the card once, with one workgroup on each CU while that leaves two per unit, else two.
//     Anything between one and two workgroups per CU has half of the CUs do double the work;
//   many units: twice the mean context.  Units then go round by themselves, and only contexts far longer than the
//     others are cut.
// Measured (us, 4-bit cache): 4 x U[8192, 40960] at 8 kv heads 20.9 with one workgroup per CU, 22.8 with two, 25.8 where
// the length was the next power of two; 16 x U[512, 4096] at 8 groups of 8 heads 13.9 either way (16.4); 32 x U[256, 2304]
// at 8 kv heads 21.7 uncut, 16.0 with two (16.7); 100 x U[2048, 4096] 63 uncut, 76 cut in two.
__host__ __device__ constexpr int partition_share(int units) {
  const int slots = units * 2 <= kCus ? kCus : 2 * kCus;
  return slots - units / 2 > units / 2 ? slots - units / 2 : units / 2;
}
__device__ __forceinline__ int partition_tokens(u32 tokens, int units, int least) {  // a multiple of 64
  const u32 share = (u32)partition_share(units);
  const u32 len = (tokens + share - 1) / share;
  return max((int)((len + 63) & ~63u), least);
}
__host__ __device__ constexpr int max_partitions(int units) { return partition_share(units) + units; }

// A workgroup's partition.
struct Part {
  int b;        // sequence
  int g;        // kv head
  int p;        // partition of the unit
  int n_parts;  // of the unit
  int ctx;
  int tokens;  // of a partition
};
template <typename Args>
__device__ __forceinline__ bool find_part(const Args &a, int item, int lane, int least, u32 &err_bits, Part &part) {
  const int hkv = a.num_kv_heads;
  // The cut, and this workgroup's place in it.
  const int ctx_cap = min(a.max_ctx, a.bt_width << a.bs_log2);
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
  const int part_tokens = partition_tokens(total * (u32)hkv, a.batch * hkv, least);
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
  if (b < 0) return false;  // past the last partition
  b = __builtin_amdgcn_readfirstlane(b);
  // Head after head of a partition: with 8 kv heads each XCD (workgroups go round them) gets one head of every partition,
  // alike in length.  (Partition after partition of a head, full ones and last ones of two parts meet in different XCDs:
  // 32 x U[1000, 2000], 8-bit cache, 27.5 us, so 21.)
  const int rem = item - first * hkv;
  const int p = rem / hkv, g = rem - p * hkv;
  part = Part{b, g, p, n_parts, ctx, part_tokens};
  return true;
}

// The rows of a head's query that a lane of the products holds: dims 16 gq .. +15 and 64 + 16 gq .. +15 of head n
// (columns past the last head repeat it and are never read).
template <typename Args>
__device__ __forceinline__ void load_query(const Args &a, int b, int head0, int n, int gq, u32x4 (&x)[4]) {
  const u16 *qp = a.q + (int64_t)b * a.q_stride + (int64_t)(head0 + min(n, a.q_sub - 1)) * kHeadDim + 16 * gq;
  x[0] = ld16(qp);
  x[1] = ld16(qp + 8);
  x[2] = ld16(qp + 64);
  x[3] = ld16(qp + 72);
}

// The operand of the step's query, normed and rotated, for every wave of the workgroup.  One wave makes it for all (the
// 64-bit arithmetic of 8 waves at once takes 3 us more), others store the new row, in the workgroup whose partition ends
// the context: store(slot, row of the table), which waits until the workgroup's loads find what it has stored.
template <typename Args, typename Store>
__device__ __forceinline__ void step_query(const Args &a, const StepArgs &s, const Part &part, int head0, int w, int lane,
                                           u32x4 (&s_q)[4][64], u32 (&s_q_scale)[64], u32 &err_bits, i32x8 &q_hi,
                                           i32x8 &q_lo, u32 &q_scale, Store &&store) {
  const int n = lane & 15, gq = lane >> 4, b = part.b;
  int64_t pos = s.positions[b];
  if (pos < 0 || pos >= s.max_positions) {  // clamp and report
    err_bits |= NVAMD_ERR_POSITION;
    pos = pos < 0 ? 0 : s.max_positions - 1;
  }
  const float *row = s.cos_sin + pos * kHeadDim;
  if (w == 1) {
    u32x4 x[4];
    load_query(a, b, head0, n, gq, x);
    norm_rope_row(x, s.q_w, row, gq, (double)s.eps);
    s_q_scale[lane] = query_operand(x, gq, q_hi, q_lo);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s_q[j][lane] = u32x4{(u32)q_hi[4 * j], (u32)q_hi[4 * j + 1], (u32)q_hi[4 * j + 2], (u32)q_hi[4 * j + 3]};
      s_q[2 + j][lane] = u32x4{(u32)q_lo[4 * j], (u32)q_lo[4 * j + 1], (u32)q_lo[4 * j + 2], (u32)q_lo[4 * j + 3]};
    }
  } else if (part.p == part.n_parts - 1 && a.q_head0 == 0) {
    const int64_t slot = s.slots[b];
    if (slot < -1 || slot >= s.num_slots)
      err_bits |= NVAMD_ERR_SLOT;
    else if (slot >= 0)
      store(slot, row);
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
}

__device__ __forceinline__ void report(u32 *err, u32 bits, int lane) {  // a lane's own bits: any lane's count
#pragma unroll
  for (u32 bit = NVAMD_ERR_SLOT; bit <= NVAMD_ERR_BLOCK; bit <<= 1)
    if (__ballot(bits & bit) && lane == 0) flag_index_error(err, bit);
}

// The end of a partition: sums of its waves meet in LDS, those of a unit's partitions in the workspace.  Register i of
// o[e] is dim 16 e + 4 gq + i of head n; l is summed over the four lanes of a head here.
template <int WAVES, int GP, typename Args>
__device__ __forceinline__ void finish(const Args &a, const Part &part, int head0, int tid, int w, f32x4 (&o)[8], float m,
                                       float l, float (&s_o)[WAVES][GP * kPartFloats], float (&s_m)[WAVES][GP],
                                       float (&s_l)[WAVES][GP], int &s_last) {
  constexpr int HS = kPartFloats;
  constexpr int D = kHeadDim;
  constexpr int HALVES = 2 * WAVES, HALVES_LOG2 = HALVES == 16 ? 4 : 3;  // half-waves of the workgroup
  static_assert(HALVES == 1 << HALVES_LOG2 && WAVES * GP >= HALVES, "the shares of a join fit s_o");
  const int lane = tid & 63, n = lane & 15, gq = lane >> 4;
  const int hkv = a.num_kv_heads, G = a.q_sub;

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

  // The waves' results meet: a half-wave takes heads hw, hw + HALVES, its lane dims 4 dl .. 4 dl + 3.
  constexpr int HP = (GP + HALVES - 1) / HALVES;
  const int hw = tid >> 5, dl = lane & 31;
  f32x4 acc[HP];
  float mx[HP], ls[HP];
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = min(hw + HALVES * k, G - 1);
    float M = s_m[0][h];
#pragma unroll
    for (int x = 1; x < WAVES; ++x) M = fmaxf(M, s_m[x][h]);
    acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    ls[k] = 0.f;
#pragma unroll
    for (int x = 0; x < WAVES; ++x) {
      const float f = fast_exp2(s_m[x][h] - M);
      acc[k] += f * *reinterpret_cast<const f32x4 *>(&s_o[x][h * HS + 4 * dl]);
      ls[k] += f * s_l[x][h];
    }
    mx[k] = M;
  }
  auto write_out = [&](int h, f32x4 v, float den) {
    const float inv = den > 0.f ? 1.f / den : 0.f;
    *reinterpret_cast<u32x2 *>(a.out + (int64_t)part.b * a.out_stride + (int64_t)(head0 + h) * D + 4 * dl) =
        u32x2{pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv)};
  };
  if (part.n_parts == 1) {
#pragma unroll
    for (int k = 0; k < HP; ++k)
      if (hw + HALVES * k < G) write_out(hw + HALVES * k, acc[k], ls[k]);
    return;
  }

  // Publish this partition's record past the caches that are not coherent, then count it.
  const int rec_bytes = G * HS * (int)sizeof(float);
  float *base = a.partials + ((int64_t)part.b * hkv + part.g) * a.max_parts * (G * HS);
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(base, 0, part.n_parts * rec_bytes, kBufferRsrcWord3);
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = hw + HALVES * k;
    if (h < G) {
      const int off = part.p * rec_bytes + h * (HS * (int)sizeof(float));
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
    s_last = (int)__builtin_amdgcn_atomic_inc32(a.counters + (int64_t)part.b * hkv + part.g, (unsigned)(part.n_parts - 1),
                                                __ATOMIC_RELAXED, "agent");
  __syncthreads();
  if (s_last != part.n_parts - 1) return;

  // The last arriver joins the partitions.  The heads share out the half-waves: `split` of them take a head, each every
  // split-th run of kRun partitions, whose records it loads together; their shares meet in LDS, in order.
  constexpr int kRun = 8;
  const int slots_log2 = min(G <= 1 ? 0 : 32 - __builtin_clz(G - 1), HALVES_LOG2);
  const int split = HALVES >> slots_log2;
  const int sp = hw >> slots_log2;
  float *so = &s_o[0][0];  // free: every wave has passed two barriers since it read them
#pragma unroll 1
  for (int h = hw & ((1 << slots_log2) - 1); h < G; h += HALVES) {
    const int hoff = h * (HS * (int)sizeof(float));
    float M = kNoScore, den = 0.f;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int y0 = sp * kRun; y0 < part.n_parts; y0 += split * kRun) {
      u32x2 ml[kRun];
      u32x4 v[kRun];
#pragma unroll
      for (int y = 0; y < kRun; ++y) {  // past part.n_parts: zeros without a memory access
        ml[y] = __builtin_amdgcn_raw_buffer_load_b64(rsrc, (y0 + y) * rec_bytes + hoff, 0, kCachePolicyAgent);
        v[y] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (y0 + y) * rec_bytes + hoff + 16 + 16 * dl, 0,
                                                     kCachePolicyAgent);
      }
      float up = M;
#pragma unroll
      for (int y = 0; y < kRun; ++y)
        if (y0 + y < part.n_parts) up = fmaxf(up, __uint_as_float(ml[y][0]));
      const float f_old = fast_exp2(M - up);
      num *= f_old;
      den *= f_old;
#pragma unroll
      for (int y = 0; y < kRun; ++y) {
        const float f = y0 + y < part.n_parts ? fast_exp2(__uint_as_float(ml[y][0]) - up) : 0.f;
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

// Checks shared by the entry points; fills what they share.  LEAST: tokens of the smallest partition.
template <int LEAST, typename Cache>
int fill_decode_args(DecodeArgs<Cache> &a, void *out, int64_t out_stride, const void *q, int64_t q_stride, const Cache &cache,
                     bool cache_ok, int num_blocks, int block_size, const int32_t *block_tables, int bt_stride,
                     int bt_width, const int32_t *context_lens, int batch, int num_heads, int num_kv_heads, int head_dim,
                     float scale, int max_context_len, void *workspace, size_t workspace_bytes) {
  static_assert(LEAST >= kMinPart, "the workspace has records for these partitions");
  if (!out || !q || !cache_ok || !block_tables || !context_lens) return NVAMD_EINVAL;
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
  a.cache = cache;
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
  a.max_parts = ceil_div(max_context_len, LEAST);
  a.batch = batch;
  a.scale_log2e = scale * kLog2e;
  a.q_group = num_heads / num_kv_heads;
  a.err = index_error_word();
  return NVAMD_OK;
}

inline int fill_step_args(StepArgs &s, const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                          const void *q_weight, const void *k_weight, const int64_t *positions, const float *cos_sin,
                          int max_positions, float eps, const int64_t *slot_mapping, int num_blocks, int block_size,
                          int num_kv_heads) {
  const int64_t row = (int64_t)num_kv_heads * kHeadDim;
  if (!k || !v || !aligned16(k) || !aligned16(v) || k_stride % 8 || v_stride % 8 || k_stride < row || v_stride < row ||
      !q_weight || !k_weight || !aligned16(q_weight) || !aligned16(k_weight) || !positions || !cos_sin ||
      !aligned16(cos_sin) || max_positions <= 0 || !slot_mapping)
    return NVAMD_EINVAL;
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
  return NVAMD_OK;
}

// Workgroups that a launch can need at most; launch(GP) for each up to kMaxHeads query heads of a kv head, GP of 4, 8 or
// 16 the heads that registers and LDS are laid out for.
template <typename Args>
unsigned decode_items(const Args &a) {
  const int units = a.batch * a.num_kv_heads;  // <= kCounterSlots
  return (unsigned)min((int64_t)units * a.max_parts, (int64_t)max_partitions(units));
}
template <typename Args, typename Launch>
int launch_groups(Args &a, Launch &&launch) {
  for (a.q_head0 = 0; a.q_head0 < a.q_group; a.q_head0 += a.q_sub) {
    a.q_sub = min(a.q_group - a.q_head0, kMaxHeads);
    const int st = a.q_sub <= 4   ? launch(std::integral_constant<int, 4>{})
                   : a.q_sub <= 8 ? launch(std::integral_constant<int, 8>{})
                                  : launch(std::integral_constant<int, 16>{});
    if (st != NVAMD_OK) return st;
  }
  return NVAMD_OK;
}

}  // namespace nvamd
