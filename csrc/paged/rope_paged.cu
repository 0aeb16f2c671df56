// Norms of queries and keys for each head, the rotary embedding and the write
// into a paged KV cache, in one pass over the qkv projection:
//
//   x'     = x * rsqrt(mean(x^2) + eps) * gamma         (heads of q and k; optional)
//   (a, b) -> (a cos - b sin, b cos + a sin)             a = x'[i], b = x'[i + d/2]
//   q to q_out, k and v to slot p % page_size of page page_table[s][p / page_size]
//
// d / 16 lanes share a head: a lane holds 8 elements of its first half and the
// 8 partners of its second half, two 16-byte loads and two 16-byte stores, so
// the rotation needs no exchange and the mean takes log2(d / 16) shuffles.
// Everything between the loads and the stores is fp32; each output is rounded
// once. A lane's 8 angles are the same for every head of a token and are
// loaded once for all the heads that it handles.
//
// Every value is read once and written once, so memory bounds the large calls
// and one chain of loads (length, offset, page, value) the small ones: five
// prompts with 64 + 2 x 8 heads of 128 (279 MB) take 58 us, 4.8 TB/s, and one or
// 64 tokens 2 us. (Prompts: DRAM 49 % of its nominal rate, issue slots 59 %. A block
// serves one row, so the chain is walked for each and its loads do not run beside
// the stores of the row before.)
#include <algorithm>

#include "../common/check.h"
#include "../common/pdl.h"
#include "../common/trace.h"
#include "batch.cuh"

namespace b200ar {
namespace paged {

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float* v) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = to_float2<T>(u[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

// Grid (rows, head chunks); a block handles kIters * kGroups consecutive heads
// of [q heads | k heads | v heads] of one row.
template <typename T, int D, int kIters>
__global__ void __launch_bounds__(kThreads) rope_paged_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kLanes = D / 16;              // lanes of a head
  constexpr int kGroups = kThreads / kLanes;  // heads in flight in a block
  const int row = blockIdx.x;
  const int lane = threadIdx.x % kLanes;
  const int h0 = blockIdx.y * (kIters * kGroups) + threadIdx.x / kLanes;
  const int heads = a.hq + 2 * a.hkv;
  pdl_wait();
  pdl_trigger();
  // The values first: their loads run beside the chain of loads that finds the page.
  uint4 w0[kIters], w1[kIters];
  const T* in = static_cast<const T*>(a.qkv) + row * a.qkv_stride + lane * 8;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    w0[i] = w1[i] = make_uint4(0u, 0u, 0u, 0u);
    if (h0 + i * kGroups < heads) {
      w0[i] = *reinterpret_cast<const uint4*>(in + (h0 + i * kGroups) * D);
      w1[i] = *reinterpret_cast<const uint4*>(in + (h0 + i * kGroups) * D + D / 2);
    }
  }
  const int s = sequence_of_row(a.batch, row);
  if (s < 0) return;
  const int first = q_begin(a.batch, s), n = q_begin(a.batch, s + 1) - first;
  const int pos = __ldg(a.batch.kv_len + s) - n + (row - first);
  if (pos < 0 || pos >= a.positions) {
    if (threadIdx.x == 0) atomicExch(a.err, kErrPosition);
    return;
  }
  const int page = page_of(a.batch, s, pos / a.page_size, a.num_pages);
  const int slot = pos % a.page_size;
  if (page < 0) {
    if (threadIdx.x == 0) atomicExch(a.err, kErrPage);
    return;
  }
  float c[8], sn[8];
  {
    const int64_t off = static_cast<int64_t>(pos) * (D / 2) + lane * 8;
    const float4* cp = reinterpret_cast<const float4*>(a.cos_t + off);
    const float4* sp = reinterpret_cast<const float4*>(a.sin_t + off);
    *reinterpret_cast<float4*>(c) = __ldg(cp);
    *reinterpret_cast<float4*>(c + 4) = __ldg(cp + 1);
    *reinterpret_cast<float4*>(sn) = __ldg(sp);
    *reinterpret_cast<float4*>(sn + 4) = __ldg(sp + 1);
  }
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = h0 + i * kGroups;
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
    float x0[8], x1[8];
    unpack8<T>(w0[i], x0);
    unpack8<T>(w1[i], x1);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x0[e] * x0[e] + x1[e] * x1[e];
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (h >= heads) continue;
    T* dst;
    if (is_q) {
      dst = static_cast<T*>(a.q_out) + row * a.q_tok + h * a.q_head;
    } else {
      const Pool& p = is_v ? a.v : a.k;
      dst = static_cast<T*>(p.base) + page * p.page + slot * p.tok + (h - a.hq - (is_v ? a.hkv : 0)) * p.head;
    }
    dst += lane * 8;
    if (is_v) {
      *reinterpret_cast<uint4*>(dst) = w0[i];
      *reinterpret_cast<uint4*>(dst + D / 2) = w1[i];
      continue;
    }
    const T* gamma = static_cast<const T*>(is_q ? a.q_gamma : a.k_gamma);
    if (gamma) {
      const float inv = rsqrtf(ss * (1.f / D) + a.eps);
      float g0[8], g1[8];
      unpack8<T>(__ldg(reinterpret_cast<const uint4*>(gamma + lane * 8)), g0);
      unpack8<T>(__ldg(reinterpret_cast<const uint4*>(gamma + D / 2 + lane * 8)), g1);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x0[e] = x0[e] * inv * g0[e];
        x1[e] = x1[e] * inv * g1[e];
      }
    }
    float y0[8], y1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y0[e] = x0[e] * c[e] - x1[e] * sn[e];
      y1[e] = x1[e] * c[e] + x0[e] * sn[e];
    }
    *reinterpret_cast<uint4*>(dst) = pack8<T>(y0);
    *reinterpret_cast<uint4*>(dst + D / 2) = pack8<T>(y1);
  }
}

template <typename T, int D, int kIters>
void launch_iters(const RopeArgs& a, cudaStream_t s) {
  constexpr int kHeads = kIters * (kThreads / (D / 16));  // heads of a block
  const int heads = a.hq + 2 * a.hkv;
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>((heads + kHeads - 1) / kHeads));
  launch_pdl(rope_paged_kernel<T, D, kIters>, grid, dim3(kThreads), 0, s, 1, a);
}

template <typename T, int D>
void launch(const RopeArgs& a, cudaStream_t s) {
  constexpr int kGroups = kThreads / (D / 16);
  const int heads = a.hq + 2 * a.hkv;
  // Many rows: up to three heads a thread, so that a block's fixed chain of loads serves more values. Few rows:
  // one, so that more SMs share the call.
  if (a.rows < 512 || heads <= kGroups)
    launch_iters<T, D, 1>(a, s);
  else if (heads <= 2 * kGroups)
    launch_iters<T, D, 2>(a, s);
  else
    launch_iters<T, D, 3>(a, s);
}

}  // namespace

void qk_norm_rope_paged(const RopeArgs& a, int d, Half type, cudaStream_t s) {
  const TraceRange trace("b200ar::qk_norm_rope_paged");
  B200AR_CHECK(d == 64 || d == 128, "qk_norm_rope_paged is built for heads of 64 and 128");
  if (a.rows == 0 || a.batch.seqs == 0) return;
  if (type == Half::kBf16)
    d == 64 ? launch<__nv_bfloat16, 64>(a, s) : launch<__nv_bfloat16, 128>(a, s);
  else
    d == 64 ? launch<__half, 64>(a, s) : launch<__half, 128>(a, s);
}

}  // namespace paged
}  // namespace b200ar
