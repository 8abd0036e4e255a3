// Attention over the 8-bit paged KV cache, one wave for each query row and head: the formula as it stands.
//
// 16 keys (a tile) at a time: lane (t, part) takes 32 dims of key t, the four parts meet by exchanges, the softmax keeps
// a running maximum and sum in 32 bits, and a lane adds up two dims of the values.
#include "attention_tiles.h"
#include "fp8.h"

namespace nvamd {
namespace {

struct AttentionArgs {
  u16 *out;
  int64_t out_stride;
  const u16 *q;
  int64_t q_stride;
  Fp8Cache cache;
  const int32_t *block_tables;
  const int32_t *cu_seqlens_q;  // or null: one row a sequence
  const int32_t *kv_lens;
  int bt_stride;
  int bt_width;
  int num_blocks;
  int bs_log2;
  int num_kv_heads;
  int group;  // query heads of a kv head
  int max_q_len;
  int num_tokens;
  int max_ctx;
  float scale;
  u32 *err;
};

__device__ __forceinline__ float code_value(const u8 *p, int64_t at, float scale) {
  return bf16_lo(fp8_pair<false>((u32)p[at], scale));
}

__global__ void __launch_bounds__(64)
attention_fp8_kernel(AttentionArgs a) {
  const int s = blockIdx.z, head = blockIdx.x, lane = threadIdx.x;
  const int g = head / a.group;
  const int q_start = a.cu_seqlens_q ? a.cu_seqlens_q[s] : s;
  const int q_end = a.cu_seqlens_q ? a.cu_seqlens_q[s + 1] : s + 1;
  const int q_len = (int)((unsigned)q_end - (unsigned)q_start);
  const bool rows_in = q_start >= 0 && q_start <= q_end && q_end <= a.num_tokens;  // else no row is touched
  const int cap = min(a.max_ctx, a.bt_width << a.bs_log2);
  const int raw = a.kv_lens[s];
  const bool short_of_rows = a.cu_seqlens_q != nullptr && raw < q_len;
  if ((!rows_in || q_len > a.max_q_len || raw > cap || raw < 0 || short_of_rows) && head == 0 && blockIdx.y == 0 && lane == 0)
    flag_index_error(a.err, NVAMD_ERR_CONTEXT);
  const int token = blockIdx.y;
  if (!rows_in || token >= q_len || token >= a.max_q_len) return;
  const int kv_len = min(max(raw, 0), cap);
  const int keys = a.cu_seqlens_q ? min(kv_len, kv_len - q_len + token + 1) : kv_len;  // that the row sees
  const int t = lane & 15, part = lane >> 4;
  float q[32];
  const u16 *qp = a.q + (int64_t)(q_start + token) * a.q_stride + (int64_t)head * kHeadDim;
#pragma unroll
  for (int d = 0; d < 32; ++d) q[d] = bf16_to_f32(qp[32 * part + d]);
  float m = kNoScore, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int t0 = 0; t0 < keys; t0 += kFp8Tile) {
    int entry = a.block_tables[(int64_t)s * a.bt_stride + (t0 >> a.bs_log2)];
    if ((unsigned)entry >= (unsigned)a.num_blocks && lane == 0) flag_index_error(a.err, NVAMD_ERR_BLOCK);
    entry = min(max(entry, 0), a.num_blocks - 1);  // never leave the pool
    const int64_t tile = fp8_tile(entry, t0 & ((1 << a.bs_log2) - 1), g, a.num_kv_heads, a.bs_log2);
    const u8 *kc = a.cache.k_codes + tile * kFp8TileBytes, *vc = a.cache.v_codes + tile * kFp8TileBytes;
    const float ks = fp8_scale(a.cache.k_scales[tile]), vs = fp8_scale(a.cache.v_scales[tile]);
    float score = 0.f;
#pragma unroll
    for (int d = 0; d < 32; ++d) score += q[d] * code_value(kc, fp8_key_at(t, 32 * part + d), ks);
    score += __shfl_xor(score, 16);
    score += __shfl_xor(score, 32);
    score = t0 + t < keys ? score * a.scale * kLog2e : -INFINITY;
    float top = score;
    for (int x = 1; x < 16; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    const float up = fmaxf(m, top), alpha = fast_exp2(m - up), p = fast_exp2(score - up);
    float sum = p;
    for (int x = 1; x < 16; x *= 2) sum += __shfl_xor(sum, x);
    l = l * alpha + sum;
    o0 *= alpha;
    o1 *= alpha;
    m = up;
    for (int i = 0; i < kFp8Tile && t0 + i < keys; ++i) {
      const float w = __shfl(p, i);
      o0 += w * code_value(vc, fp8_value_at(i, 2 * lane), vs);
      o1 += w * code_value(vc, fp8_value_at(i, 2 * lane + 1), vs);
    }
  }
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // no key: zeros; a NaN stays one
  reinterpret_cast<u32 *>(a.out + (int64_t)(q_start + token) * a.out_stride + (int64_t)head * kHeadDim)[lane] =
      pack_bf16x2(o0 * inv, o1 * inv);
}

int fill_args(AttentionArgs &a, void *out, int64_t out_stride, const void *q, int64_t q_stride, const void *k_codes,
              const void *k_scales, const void *v_codes, const void *v_scales, int num_blocks, int block_size,
              const int32_t *block_tables, int bt_stride, int bt_width, const int32_t *kv_lens, int num_heads,
              int num_kv_heads, int head_dim, float scale) {
  const int bs_log2 = log2_exact(block_size);
  if (head_dim != kHeadDim || bs_log2 < 4) return NVAMD_EUNSUPPORTED;
  if (!out || !q || !fp8_cache_ok(k_codes, k_scales, v_codes, v_scales) || !block_tables || !kv_lens || num_blocks <= 0 ||
      num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || bt_width <= 0 || bt_stride < bt_width ||
      !aligned16(q) || !aligned16(out) || q_stride % 8 || out_stride % 8 || q_stride < (int64_t)num_heads * head_dim ||
      out_stride < (int64_t)num_heads * head_dim)
    return NVAMD_EINVAL;
  if (((int64_t)bt_width << bs_log2) > 1 << 30 || (((int64_t)num_blocks * num_kv_heads) << bs_log2) >> 4 > 0x7fffffff)
    return NVAMD_EUNSUPPORTED;
  a = {};
  a.out = static_cast<u16 *>(out);
  a.out_stride = out_stride;
  a.q = static_cast<const u16 *>(q);
  a.q_stride = q_stride;
  a.cache = Fp8Cache{const_cast<u8 *>(static_cast<const u8 *>(k_codes)),
                     const_cast<u8 *>(static_cast<const u8 *>(k_scales)),
                     const_cast<u8 *>(static_cast<const u8 *>(v_codes)),
                     const_cast<u8 *>(static_cast<const u8 *>(v_scales))};
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.bt_width = bt_width;
  a.num_blocks = num_blocks;
  a.bs_log2 = bs_log2;
  a.kv_lens = kv_lens;
  a.num_kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.scale = scale;
  a.err = index_error_word();
  return NVAMD_OK;
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" size_t nvamd_paged_prefill_fp8_workspace_size(int n_seqs, int max_q_len, int num_heads, int num_kv_heads,
                                                         int block_size, int bt_width) {
  return 0;
}

extern "C" int nvamd_paged_prefill_fp8(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                       const void *k_codes, const void *k_scales, const void *v_codes,
                                       const void *v_scales, int num_blocks, int block_size,
                                       const int32_t *block_tables, int bt_stride, int bt_width,
                                       const int32_t *cu_seqlens_q, const int32_t *kv_lens, int n_seqs, int num_tokens,
                                       int max_q_len, int num_heads, int num_kv_heads, int head_dim, float scale,
                                       void *workspace, size_t workspace_bytes, hipStream_t stream) {
  if (n_seqs == 0 || max_q_len == 0 || num_tokens == 0) return NVAMD_OK;
  AttentionArgs a;
  const int st = fill_args(a, out, out_stride, q, q_stride, k_codes, k_scales, v_codes, v_scales, num_blocks, block_size,
                           block_tables, bt_stride, bt_width, kv_lens, num_heads, num_kv_heads, head_dim, scale);
  if (st != NVAMD_OK) return st;
  if (!(scale > 0.f) || !cu_seqlens_q || n_seqs < 0 || num_tokens < 0 || max_q_len < 0 || n_seqs > 65535)
    return NVAMD_EINVAL;
  if (max_q_len > 65535) return NVAMD_EUNSUPPORTED;
  a.cu_seqlens_q = cu_seqlens_q;
  a.max_q_len = max_q_len;
  a.num_tokens = num_tokens;
  a.max_ctx = 0x7fffffff;
  hipLaunchKernelGGL(attention_fp8_kernel, dim3(num_heads, max_q_len, n_seqs), dim3(64), 0, stream, a);
  return launch_status();
}
