// Attention of new tokens over a paged KV cache.
//
//   o[i] = sum_p softmax_p(scale q[i] . k[p]) v[p]  over the positions p that row i sees
//
// The simplest form: one warp for each (row, query head) walks the positions
// with a running maximum and sum.
#include "../common/check.h"
#include "../common/pdl.h"
#include "../common/trace.h"
#include "batch.cuh"

namespace b200ar {
namespace paged {

namespace {

template <typename T, int D>
__global__ void __launch_bounds__(128) attention_simple_kernel(const AttnArgs a) {
  constexpr int kPairs = D / 64;  // pairs of elements that a lane holds
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  pdl_wait();
  pdl_trigger();
  if (item >= static_cast<int64_t>(a.rows) * a.hq) return;
  const int row = static_cast<int>(item / a.hq), h = static_cast<int>(item % a.hq);
  const int s = sequence_of_row(a.batch, row);
  if (s < 0) return;
  const int first = q_begin(a.batch, s), n = q_begin(a.batch, s + 1) - first;
  const int len = __ldg(a.batch.kv_len + s);
  const int pos = len - n + (row - first);
  const int end = a.causal ? pos + 1 : len;
  const int begin = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int kh = h / (a.hq / a.hkv);
  float2 q[kPairs], o[kPairs];
  const T* qp = static_cast<const T*>(a.q) + row * a.q_tok + h * a.q_head;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    q[i] = to_float2<T>(*reinterpret_cast<const uint32_t*>(qp + i * 64 + lane * 2));
    o[i] = make_float2(0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
  for (int p = begin; p < end; ++p) {
    const int page = page_of(a.batch, s, p / a.page_size, a.num_pages);
    if (page < 0) {
      if (lane == 0) atomicExch(a.err, kErrPage);
      continue;
    }
    const int slot = p % a.page_size;
    const T* kp = static_cast<const T*>(a.k.base) + page * a.k.page + slot * a.k.tok + kh * a.k.head;
    const T* vp = static_cast<const T*>(a.v.base) + page * a.v.page + slot * a.v.tok + kh * a.v.head;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 k = to_float2<T>(*reinterpret_cast<const uint32_t*>(kp + i * 64 + lane * 2));
      dot += q[i].x * k.x + q[i].y * k.y;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    const float x = dot * a.scale * 1.4426950408889634f;
    const float mn = fmaxf(m, x);
    const float f = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float e = exp2f(x - mn);
    m = mn;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 v = to_float2<T>(*reinterpret_cast<const uint32_t*>(vp + i * 64 + lane * 2));
      o[i].x = o[i].x * f + e * v.x;
      o[i].y = o[i].y * f + e * v.y;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* op = static_cast<T*>(a.out) + row * a.o_tok + h * a.o_head;
#pragma unroll
  for (int i = 0; i < kPairs; ++i)
    *reinterpret_cast<uint32_t*>(op + i * 64 + lane * 2) = pack2<T>(o[i].x * inv, o[i].y * inv);
}

template <typename T, int D>
void launch(const AttnArgs& a, cudaStream_t s) {
  const int64_t items = static_cast<int64_t>(a.rows) * a.hq;
  launch_pdl(attention_simple_kernel<T, D>, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(128), 0, s, 1, a);
}

}  // namespace

void paged_attention(const AttnArgs& a, int d, Half type, cudaStream_t s) {
  const TraceRange trace("b200ar::paged_attention");
  B200AR_CHECK(d == 64 || d == 128, "paged_attention is built for heads of 64 and 128");
  if (a.rows == 0 || a.batch.seqs == 0) return;
  if (type == Half::kBf16)
    d == 64 ? launch<__nv_bfloat16, 64>(a, s) : launch<__nv_bfloat16, 128>(a, s);
  else
    d == 64 ? launch<__half, 64>(a, s) : launch<__half, 128>(a, s);
}

}  // namespace paged
}  // namespace b200ar
