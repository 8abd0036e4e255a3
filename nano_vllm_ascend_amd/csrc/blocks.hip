// Copies of blocks inside a cache's pools: what a request that branches, or that is moved to other blocks, needs.
//
// pool[layer][target[i]] = pool[layer][source[i]] for every layer of every pool, in one launch.  Bound by memory: each
// byte is read once and written once.  A workgroup copies 16 KiB of a block's layer, a lane 64 bytes whose loads are on
// their way together; the stores pass the caches by.  One block of 128 tokens of 8 heads in 28 layers of the 8-bit cache
// (15 MB read and written): 3.0 us from a graph (4.1 to 4.4 eager, where the launch takes the host 3.6), 4.0 with ordinary
// stores, one load at a time; 8 blocks 21.8 us (5.4 TB/s), 26.2; 48 blocks of the bf16 cache, 1.4 GB, 268 to 271 us (5.2
// TB/s, the rate of one large copy), 272.  Pieces of 8 KiB: 4.1, 24.5 and 262 us, of 32: 3.3, 23.0 and 267.
#include "common.h"

namespace nvamd {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPools = 8;
constexpr int kPiece = 16384;  // bytes of a block that a workgroup copies

struct CopyArgs {
  uint8_t *pools[kMaxPools];
  int64_t block_bytes[kMaxPools];
  int pieces[kMaxPools + 1];  // of a block: those of pool p are pieces[p] .. pieces[p + 1] - 1
  const int32_t *sources;
  const int32_t *targets;
  int num_blocks;
  u32 *err;
};

template <typename T>
__device__ __forceinline__ void copy_bytes(uint8_t *dst, const uint8_t *src, int bytes, int tid) {
  constexpr int kBatch = 4;  // loads of a lane that are on their way together
  T *to = reinterpret_cast<T *>(dst);
  const T *from = reinterpret_cast<const T *>(src);
  const int n = bytes / (int)sizeof(T);
  int i = tid;
  for (; i + (kBatch - 1) * kThreads < n; i += kBatch * kThreads) {
    T x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) x[j] = from[i + j * kThreads];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) __builtin_nontemporal_store(x[j], to + i + j * kThreads);
  }
  for (; i < n; i += kThreads) to[i] = from[i];
}

__global__ void __launch_bounds__(kThreads)
copy_blocks_kernel(CopyArgs a) {
  const int source = a.sources[blockIdx.y], target = a.targets[blockIdx.y];
  if ((unsigned)source >= (unsigned)a.num_blocks || (unsigned)target >= (unsigned)a.num_blocks) {
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) flag_index_error(a.err, NVAMD_ERR_BLOCK);
    return;
  }
  if (source == target) return;
  int p = 0;
  while ((int)blockIdx.x >= a.pieces[p + 1]) ++p;
  const int64_t size = a.block_bytes[p], at = (int64_t)((int)blockIdx.x - a.pieces[p]) * kPiece;
  uint8_t *layer = a.pools[p] + (int64_t)blockIdx.z * a.num_blocks * size;
  uint8_t *dst = layer + target * size + at;
  const uint8_t *src = layer + source * size + at;
  const int bytes = (int)min(size - at, (int64_t)kPiece);
  if (((reinterpret_cast<uintptr_t>(a.pools[p]) | (uintptr_t)size) & 15) == 0)
    copy_bytes<u32x4>(dst, src, bytes, threadIdx.x);
  else
    copy_bytes<uint8_t>(dst, src, bytes, threadIdx.x);
}

}  // namespace
}  // namespace nvamd

using namespace nvamd;

extern "C" int nvamd_copy_blocks(void *const *pools, const int64_t *block_bytes, int num_pools, int num_layers,
                                 int num_blocks, const int32_t *sources, const int32_t *targets, int count,
                                 hipStream_t stream) {
  if (count == 0 || num_layers == 0) return NVAMD_OK;
  if (!pools || !block_bytes || num_pools <= 0 || num_layers < 0 || num_blocks <= 0 || !sources || !targets || count < 0)
    return NVAMD_EINVAL;
  if (num_pools > kMaxPools || num_layers > 65535 || count > 65535) return NVAMD_EUNSUPPORTED;
  CopyArgs a = {};
  for (int p = 0; p < num_pools; ++p) {
    if (!pools[p] || block_bytes[p] <= 0) return NVAMD_EINVAL;
    if (block_bytes[p] > (int64_t)1 << 32) return NVAMD_EUNSUPPORTED;
    a.pools[p] = static_cast<uint8_t *>(pools[p]);
    a.block_bytes[p] = block_bytes[p];
    a.pieces[p + 1] = a.pieces[p] + (int)((block_bytes[p] + kPiece - 1) / kPiece);
  }
  a.sources = sources;
  a.targets = targets;
  a.num_blocks = num_blocks;
  a.err = index_error_word();
  hipLaunchKernelGGL(copy_blocks_kernel, dim3(a.pieces[num_pools], count, num_layers), dim3(kThreads), 0, stream, a);
  return launch_status();
}
