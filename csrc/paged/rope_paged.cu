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
// and one chain of loads (length, offset, page, value) the small ones.
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

// Grid (rows, head chunks); a block handles `per_block` consecutive heads of
// [q heads | k heads | v heads] of one row.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rope_paged_kernel(const RopeArgs a, int per_block) {
  constexpr int kLanes = D / 16;             // lanes of a head
  constexpr int kGroups = kThreads / kLanes;  // heads in flight in a block
  const int row = blockIdx.x;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  pdl_wait();
  pdl_trigger();
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
  const T* in = static_cast<const T*>(a.qkv) + row * a.qkv_stride;
  const int heads = a.hq + 2 * a.hkv;
  const int h_end = min(heads, (static_cast<int>(blockIdx.y) + 1) * per_block);
  // Uniform trip count: the shuffles below need every lane of the warp.
  for (int h0 = blockIdx.y * per_block; h0 < h_end; h0 += kGroups) {
    const int h = h0 + group;
    const bool on = h < h_end;
    float x0[8], x1[8];
    uint4 w0 = make_uint4(0u, 0u, 0u, 0u), w1 = w0;
    if (on) {
      const T* src = in + h * D + lane * 8;
      w0 = *reinterpret_cast<const uint4*>(src);
      w1 = *reinterpret_cast<const uint4*>(src + D / 2);
    }
    unpack8<T>(w0, x0);
    unpack8<T>(w1, x1);
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
    const T* gamma = static_cast<const T*>(is_q ? a.q_gamma : a.k_gamma);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x0[i] * x0[i] + x1[i] * x1[i];
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!on) continue;
    T* dst;
    if (is_q) {
      dst = static_cast<T*>(a.q_out) + row * a.q_tok + h * a.q_head;
    } else {
      const Pool& p = is_v ? a.v : a.k;
      const int kh = h - a.hq - (is_v ? a.hkv : 0);
      dst = static_cast<T*>(p.base) + page * p.page + slot * p.tok + kh * p.head;
    }
    dst += lane * 8;
    if (is_v) {
      *reinterpret_cast<uint4*>(dst) = w0;
      *reinterpret_cast<uint4*>(dst + D / 2) = w1;
      continue;
    }
    if (gamma) {
      const float inv = rsqrtf(ss * (1.f / D) + a.eps);
      float g0[8], g1[8];
      unpack8<T>(__ldg(reinterpret_cast<const uint4*>(gamma + lane * 8)), g0);
      unpack8<T>(__ldg(reinterpret_cast<const uint4*>(gamma + D / 2 + lane * 8)), g1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x0[i] = x0[i] * inv * g0[i];
        x1[i] = x1[i] * inv * g1[i];
      }
    }
    float y0[8], y1[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y0[i] = x0[i] * c[i] - x1[i] * sn[i];
      y1[i] = x1[i] * c[i] + x0[i] * sn[i];
    }
    *reinterpret_cast<uint4*>(dst) = pack8<T>(y0);
    *reinterpret_cast<uint4*>(dst + D / 2) = pack8<T>(y1);
  }
}

template <typename T, int D>
void launch(const RopeArgs& a, cudaStream_t s) {
  constexpr int kGroups = kThreads / (D / 16);
  const int heads = a.hq + 2 * a.hkv;
  // Few rows: one pass of the block over its heads, so that more SMs share the call.
  const int per_block = kGroups;
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>((heads + per_block - 1) / per_block));
  launch_pdl(rope_paged_kernel<T, D>, grid, dim3(kThreads), 0, s, 1, a, per_block);
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
