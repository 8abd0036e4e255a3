// GQA paged decode attention over the 4-bit KV cache (the counterpart of paged_decode.hip).
//
// For a query token of each sequence and its heads h of kv head g: out = softmax(q . K^T * scale) V over the cached
// context, with K and V expanded from 4 bits on the way into the matrix cores (v_cvt_scalef32_pk_bf16_fp4: two values and
// their scale in one instruction, exact).
//
// Work: a unit (sequence, kv head) is cut into partitions of 256 * 2^shift tokens, a workgroup of 4 waves each.  Every
// workgroup reads the context lengths and derives the same shift: the least that leaves at most `target` partitions.  So
// the cut follows the contexts themselves and not the bound that the launch was made with.  A partition
// leaves (max, sum, numerator) per head in the workspace and counts its arrival; the last one of a unit
// joins them.
//
// A wave takes 64 tokens at a time, four 16-token tiles, one per 16 lanes (gq = lane / 16):
//   S^T = K . Q^T  v_mfma_f32_16x16x32_bf16, A = 16 rows of K, B = the heads as 16 columns.  The contraction runs over
//        dims 32 gq + 8 i + 0..7 in step i, so a lane's 16 bytes of codes are one block of a row, under one scale.
//        Row 4a + i of product t is token 4t + i of tile a: lane (h, gq) then finds the scores of tile gq's tokens
//        4t .. 4t+3 of head h in its accumulator of product t, that is of all 16 tokens in the four products;
//   O^T += V^T . P^T  A = 16 dims of V^T, B = P^T, whose 8 k-slots per lane are tokens 0..7 (8..15) of tile gq: just
//        what the lane holds.  The cache keeps V with 16 tokens of a dim pair in consecutive bytes, so the lane's
//        16 bytes give both products' operands of two dims: no lane movement anywhere.
// The score of a token past the context is replaced by -inf and the scales of its values by zero, whatever bytes it holds.
#include "fp4.h"

namespace nvamd {
namespace {

constexpr int kPartFloats = 132;  // a head's record: max, sum, 2 unused, 128 accumulators
constexpr int kCounterSlots = 16384;
constexpr size_t kCounterBytes = kCounterSlots * sizeof(int);
constexpr int kMaxContext = 131072;  // largest context bound of a call
constexpr int kMinPart = 256;        // tokens of the smallest partition: one 64-token chunk for each wave
constexpr int kWaves = 4;
constexpr int kTarget = 2048;  // partitions that a launch is cut into where the contexts allow
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

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0,
                                                 0, 0);
}

// Inclusive prefix sum over a wave (see paged_decode.hip).
__device__ __forceinline__ int wave_scan(int v, int lane) {
  v += __builtin_amdgcn_mov_dpp(v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x118, 0xF, 0xF, true);
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31);
  const int r2 = __builtin_amdgcn_readlane(v, 47);
  const int row = lane >> 4;
  return v + (row >= 1 ? r0 : 0) + (row >= 2 ? r1 : 0) + (row >= 3 ? r2 : 0);
}

// max / sum over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_over_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_xor32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_over_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum_xor32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

template <int B>
__device__ __forceinline__ float scale_of(u32 word) {
  return __uint_as_float(((word >> (8 * B)) & 0xffu) << 23);
}

// Keeps the first n bytes (0 .. 16) of 16.
__device__ __forceinline__ u32x4 keep_bytes(u32x4 v, int n) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int k = min(max(n - 4 * w, 0), 4);
    v[w] &= k == 4 ? 0xffffffffu : (1u << (8 * k)) - 1u;
  }
  return v;
}

template <int GP>
__global__ void __launch_bounds__(kWaves * 64)
paged_decode_fp4_kernel(DecodeFp4Args a) {
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
  int64_t total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int bi = b0 + lane;
    const int raw = bi < a.batch ? a.context_lens[bi] : 0;
    if (__ballot(raw < 0 || raw > ctx_cap)) err_bits |= NVAMD_ERR_CONTEXT;
    const int units = bi < a.batch ? max(ceil_div(min(max(raw, 0), ctx_cap), kMinPart), 1) : 0;
    total += __builtin_amdgcn_readlane(wave_scan(units, lane), 63);
  }
  int shift = 0;
  while ((total * hkv >> shift) > kTarget) ++shift;
  const int part_tokens = kMinPart << shift;
  int b = -1, n_parts = 0, first = 0, ctx = 0;
  for (int b0 = 0, base = 0; b0 < a.batch; b0 += 64) {
    const int bi = b0 + lane;
    const int ci = bi < a.batch ? min(max(a.context_lens[bi], 0), ctx_cap) : 0;
    const int np = bi < a.batch ? max(ceil_div(ci, part_tokens), 1) : 0;
    const int incl = wave_scan(np, lane);
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

  // Query operand: dims 32 gq + 8 i .. +7 of head n (columns past the last head repeat it and are never read).
  u32x4 qf[4];
  {
    const u16 *qp = a.q + (int64_t)b * a.q_stride + (int64_t)(head0 + min(n, G - 1)) * D + 32 * gq;
#pragma unroll
    for (int i = 0; i < 4; ++i) qf[i] = ld16(qp + 8 * i);
  }

  float m = -INFINITY, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int t_end = min((p + 1) * part_tokens, ctx);
  for (int t0 = p * part_tokens + 64 * w; t0 < t_end; t0 += 64 * kWaves) {
    // The tile of each 16 lanes, as row owners of K (a = n / 4) and as token owners of V (gq); tiles past the
    // context repeat its last one.
    const int last = (ctx - 1) & ~15;
    auto tile_at = [&](int i) {
      const int t = min(t0 + 16 * i, last);
      int blk = bt_row[t >> a.bs_log2];
      if ((unsigned)blk >= (unsigned)a.num_blocks) err_bits |= NVAMD_ERR_BLOCK;
      blk = min(max(blk, 0), a.num_blocks - 1);  // never leave the pool
      return fp4_tile(blk, t & bs_mask, g, hkv, a.bs_log2);
    };
    const int64_t kt = tile_at(n >> 2), vt = tile_at(gq);
    const u8 *kp = a.cache.k_codes + kt * kFp4TileBytes + (n & 3) * kFp4RowBytes + 16 * gq;
    const u8 *vp = a.cache.v_codes + vt * kFp4TileBytes + 16 * n;
    u32x4 kc[4], vc[4], vs[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) kc[t] = *reinterpret_cast<const u32x4 *>(kp + 4 * t * kFp4RowBytes);
    const u32 ks = *reinterpret_cast<const u32 *>(a.cache.k_scales + kt * kFp4TileScales + fp4_key_scale_at(n & 3, gq));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      vc[q] = *reinterpret_cast<const u32x4 *>(vp + 256 * q);
      vs[q] = *reinterpret_cast<const u32x4 *>(a.cache.v_scales + vt * kFp4TileScales + 16 * q);
    }

    f32x4 s[4];
    const float kscale[4] = {scale_of<0>(ks), scale_of<1>(ks), scale_of<2>(ks), scale_of<3>(ks)};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t] = mfma16(fp4_values(kc[t][i], kscale[t]), qf[i], s[t]);
    }

    // Online softmax: one reference per head and wave.
    const int live = t_end - t0 - 16 * gq;  // this lane's tokens that the partition holds
    float cm = m;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = 4 * t + i < live ? s[t][i] * a.scale_log2e : -INFINITY;
        cm = fmaxf(cm, s[t][i]);
      }
    cm = max_over_quarters(cm);
    const float ref = cm == -INFINITY ? 0.f : cm;
    const float alpha = fast_exp2(m - ref);
    m = cm;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= alpha;
    // P rounded to bf16 for the matrix cores; the sum takes the same rounded values.
    u32x4 pf[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32 pr = pack_bf16x2(fast_exp2(s[t][2 * i] - ref), fast_exp2(s[t][2 * i + 1] - ref));
        l = dot2_bf16(pr, 0x3F803F80u, l);
        pf[t >> 1][2 * (t & 1) + i] = pr;
      }

    if (t0 + 64 > t_end) {  // values past the partition's end weigh nothing, NaN scales of stale rows among them
#pragma unroll
      for (int q = 0; q < 4; ++q) vs[q] = keep_bytes(vs[q], live);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 lo, hi;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const u32 c = vc[q][2 * h + x], sc = vs[q][2 * h + x];
          const u32 v0 = fp4_pair<0>(c, scale_of<0>(sc)), v1 = fp4_pair<1>(c, scale_of<1>(sc));
          const u32 v2 = fp4_pair<2>(c, scale_of<2>(sc)), v3 = fp4_pair<3>(c, scale_of<3>(sc));
          lo[2 * x] = pair_lo(v0, v1);
          lo[2 * x + 1] = pair_lo(v2, v3);
          hi[2 * x] = pair_hi(v0, v1);
          hi[2 * x + 1] = pair_hi(v2, v3);
        }
        o[2 * q] = mfma16(lo, pf[h], o[2 * q]);
        o[2 * q + 1] = mfma16(hi, pf[h], o[2 * q + 1]);
      }
  }

  {
    u32 bits = err_bits;  // a lane's own bits: any lane's count
#pragma unroll
    for (u32 bit = NVAMD_ERR_SLOT; bit <= NVAMD_ERR_BLOCK; bit <<= 1)
      if (__ballot(bits & bit) && lane == 0) flag_index_error(a.err, bit);
  }

  // Register i of o[e] is dim 16 e + 4 gq + i of head n.
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

  // The waves' results meet: a half-wave takes heads hw, hw + 8, its lane dims 4 dl .. 4 dl + 3.
  constexpr int HP = (GP + 7) / 8;
  const int hw = tid >> 5, dl = lane & 31;
  f32x4 acc[HP];
  float mx[HP], ls[HP];
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = min(hw + 8 * k, G - 1);
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) M = fmaxf(M, s_m[x][h]);
    acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    ls[k] = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      const float f = s_m[x][h] == -INFINITY ? 0.f : fast_exp2(s_m[x][h] - M);
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
      if (hw + 8 * k < G) write_out(hw + 8 * k, acc[k], ls[k]);
    return;
  }

  // Publish this partition's record past the caches that are not coherent, then count it.
  const int rec_bytes = G * HS * (int)sizeof(float);
  float *base = a.partials + ((int64_t)b * hkv + g) * a.max_parts * (G * HS);
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(base, 0, n_parts * rec_bytes, kBufferRsrcWord3);
#pragma unroll
  for (int k = 0; k < HP; ++k) {
    const int h = hw + 8 * k;
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

  // The last arriver joins the partitions, in their order.
#pragma unroll 1
  for (int h = hw; h < G; h += 8) {
    const int hoff = h * (HS * (int)sizeof(float));
    float M = -INFINITY, den = 0.f;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int y = 0; y < n_parts; ++y) {
      const u32x2 ml = __builtin_amdgcn_raw_buffer_load_b64(rsrc, y * rec_bytes + hoff, 0, kCachePolicyAgent);
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, y * rec_bytes + hoff + 16 + 16 * dl, 0,
                                                            kCachePolicyAgent);
      const float pm = __uint_as_float(ml[0]);
      const float up = fmaxf(M, pm);
      const float f_old = M == -INFINITY ? 0.f : fast_exp2(M - up), f_new = pm == -INFINITY ? 0.f : fast_exp2(pm - up);
      num = num * f_old + f_new * __builtin_bit_cast(f32x4, v);
      den = den * f_old + f_new * __uint_as_float(ml[1]);
      M = up;
    }
    write_out(h, num, den);
  }
}

template <int GP>
int launch(const DecodeFp4Args &a, hipStream_t stream) {
  const int64_t units = (int64_t)a.batch * a.num_kv_heads;
  // partitions: one per unit at least, kTarget in all besides, and no more than the bound allows
  const int64_t items = min(units * a.max_parts, units + kTarget);
  hipLaunchKernelGGL((paged_decode_fp4_kernel<GP>), dim3((unsigned)items), dim3(kWaves * 64), 0, stream, a);
  return launch_status();
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
      ((int64_t)bt_width << bs_log2) > 0x7fffffff)
    return NVAMD_EUNSUPPORTED;
  if (!workspace ||
      workspace_bytes < nvamd_paged_decode_workspace_size(batch, num_heads, num_kv_heads, max_context_len))
    return NVAMD_EWORKSPACE;
  if (!aligned16(workspace)) return NVAMD_EINVAL;

  DecodeFp4Args a = {};
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
  a.max_parts = ceil_div(max_context_len, kMinPart);
  a.batch = batch;
  a.scale_log2e = scale * kLog2e;
  a.q_group = num_heads / num_kv_heads;
  a.err = index_error_word();
  for (a.q_head0 = 0; a.q_head0 < a.q_group; a.q_head0 += a.q_sub) {
    a.q_sub = min(a.q_group - a.q_head0, kMaxHeads);
    const int st = a.q_sub <= 4 ? launch<4>(a, stream) : a.q_sub <= 8 ? launch<8>(a, stream) : launch<16>(a, stream);
    if (st != NVAMD_OK) return st;
  }
  return NVAMD_OK;
}
