// The workspace of paged decode, which the bf16 and the 4-bit kernels share: an arrival counter for each unit (sequence,
// kv head), then for each unit the records of its partitions, kPartFloats floats for each query head of the kv head.
#pragma once

#include "common.h"

namespace nvamd {

constexpr int kPartFloats = kHeadDim + 4;  // a head's record: max, sum, accumulators, 2 unused (16-byte rows)
// Arrival counters live in a fixed-size region at the front of the workspace so
// calls with different batch sizes or context bounds never place partial
// results where another call expects a zero counter.
constexpr int kCounterSlots = 16384;
constexpr size_t kCounterBytes = kCounterSlots * sizeof(int);
constexpr int kMaxContext = 131072;  // largest context bound of a call
// Tokens of the smallest partition that the workspace has records for.  A kernel whose partitions are no shorter, and
// whose context bound gives `parts` of them, fits: its records take units * parts * (heads of a kv head) of kPartFloats.
constexpr int kMinPart = 256;

inline size_t decode_workspace_bytes(int batch, int num_heads, int num_kv_heads, int max_context_len) {
  const size_t parts = (size_t)ceil_div(max_context_len, kMinPart);
  const size_t units = (size_t)batch * num_kv_heads;
  return kCounterBytes + units * parts * (num_heads / num_kv_heads) * kPartFloats * sizeof(float);
}

// Inclusive prefix sum over the 64 lanes of a wave, in registers: a Hillis-Steele scan inside
// each 16-lane row by DPP row shifts (lanes shifted in from outside the row read 0), then each
// row adds the totals of the rows before it (lane 15 of each row, read into scalar registers).
__device__ __forceinline__ int wave_incl_scan(int v, int lane) {
  v += __builtin_amdgcn_mov_dpp(v, 0x111, 0xF, 0xF, true);  // row_shr:1
  v += __builtin_amdgcn_mov_dpp(v, 0x112, 0xF, 0xF, true);  // row_shr:2
  v += __builtin_amdgcn_mov_dpp(v, 0x114, 0xF, 0xF, true);  // row_shr:4
  v += __builtin_amdgcn_mov_dpp(v, 0x118, 0xF, 0xF, true);  // row_shr:8
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31);
  const int r2 = __builtin_amdgcn_readlane(v, 47);
  const int row = lane >> 4;
  return v + (row >= 1 ? r0 : 0) + (row >= 2 ? r1 : 0) + (row >= 3 ? r2 : 0);
}

}  // namespace nvamd
