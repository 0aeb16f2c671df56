// Device-side view of a paged batch: rows to sequences, positions to pages.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"

namespace b200ar {
namespace paged {

// First row of sequence s. No offset leads outside the inputs, whatever q_start holds.
__device__ __forceinline__ int q_begin(const Batch& b, int s) {
  return b.q_start ? min(max(__ldg(b.q_start + s), 0), b.rows) : s;
}

// Sequence of input row `row` (the last s with q_start[s] <= row), or -1 for a
// row behind the last sequence. Called by whole warps: each step compares
// against 32 offsets at once, so two steps serve 1024 sequences.
__device__ __forceinline__ int sequence_of_row(const Batch& b, int row) {
  if (!b.q_start) return row < b.seqs ? row : -1;
  const int lane = threadIdx.x & 31;
  int lo = 0, n = b.seqs + 1;  // q_start[lo] <= row, and the answer's index is in [lo, lo + n)
  if (__ldg(b.q_start) > row) return -1;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i = lo + lane * step;
    const bool le = lane * step < n && __ldg(b.q_start + i) <= row;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, le));
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo < b.seqs ? lo : -1;
}

// Page of position `pos` of sequence s, or -1 if it has none in the pool.
__device__ __forceinline__ int page_of(const Batch& b, int s, int page_index, int num_pages) {
  if (page_index < 0 || page_index >= b.max_pages) return -1;
  const int page = __ldg(b.page_table + s * b.table_stride + page_index);
  return page >= 0 && page < num_pages ? page : -1;
}

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t w);
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace paged
}  // namespace b200ar
