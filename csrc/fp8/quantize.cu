// Quantization to e4m3 with one scale for each block of 128.
//
//   scale = amax / 448 (1 where that is 0),  q = e4m3(x / scale)
//
// Both quotients are the correctly rounded fp32 ones, so the codes are those
// of the formula and not an approximation of it. (The products with a number
// just below and one just above 1 / scale enclose the quotient: only where their
// codes differ the division is made.) The maximum is taken over the
// bit patterns of |x|, in which NaN is above infinity: a block that holds a
// NaN gets the scale NaN, one that holds an infinity the scale infinity, and
// either reaches the outputs of its row.
//
// Each value is read once and its code written once, 3 bytes: 4096 x 8192 values
// take 28 us (100 MB, 15 us at the copy rate) and a weight of 7168 x 8192 41 us.
// What bounds it is the number of instructions, two conversions of each value
// among them: issue slots 84 % of the active cycles, DRAM 29 %. (With a test of
// every product for the middle between two codes it took nearly twice as long.)
#include "../common/check.h"
#include "../common/pdl.h"
#include "../common/trace.h"
#include "encode.cuh"
#include "fp8.h"

namespace b200ar {
namespace fp8 {

namespace {

constexpr int kThreads = 256;

// Sixteen lanes share a block of 128 values; grid (groups of kRows rows, 16 blocks of them).
template <typename T, int kRows>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, float* __restrict__ scale,
                    int64_t lds, int64_t M, int K, unsigned* __restrict__ zero, int64_t zeros) {
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int lane = threadIdx.x & 15;
  const int b = blockIdx.y * (kThreads / 16) + (threadIdx.x >> 4);
  const int k = b * kBlock + lane * 8;
  Eight<T> v[kRows];
  pdl_wait();
  pdl_trigger();
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y) * kThreads + threadIdx.x; i < zeros;
       i += static_cast<int64_t>(gridDim.x) * gridDim.y * kThreads)
    zero[i] = 0u;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    v[r].zero();
    if (k < K && m0 + r < M) v[r].load(x + (m0 + r) * ldx + k);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    unsigned amax = v[r].amax();
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = Eight<T>::larger(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (k >= K || m0 + r >= M) continue;
    const Scale s(Eight<T>::fp32(amax));
    float f[8];
    v[r].get(f);
    *reinterpret_cast<uint2*>(q + (m0 + r) * K + k) = encode8(f, s);
    if (lane == 0) scale[b * lds + m0 + r] = s.scale;
  }
}

// One CTA for each 128 x 128 block: 16 lanes on a row, 8 rows a thread.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    quantize_weight_kernel(const T* __restrict__ w, int64_t ldw, uint8_t* __restrict__ q, float* __restrict__ scale,
                           int64_t N, int K) {
  __shared__ unsigned part[kThreads / 32];
  const int lane = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int k = blockIdx.x * kBlock + lane * 8;
  const int64_t n0 = static_cast<int64_t>(blockIdx.y) * kBlock;
  Eight<T> v[8];
  unsigned amax = 0;
  pdl_wait();
  pdl_trigger();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = n0 + r0 + 16 * i;
    v[i].zero();
    if (n < N && k < K) v[i].load(w + n * ldw + k);
    amax = Eight<T>::larger(amax, v[i].amax());
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = Eight<T>::larger(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) amax = Eight<T>::larger(amax, part[i]);
  const Scale s(Eight<T>::fp32(amax));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = n0 + r0 + 16 * i;
    if (n >= N || k >= K) continue;
    float f[8];
    v[i].get(f);
    *reinterpret_cast<uint2*>(q + n * K + k) = encode8(f, s);
  }
  if (threadIdx.x == 0) scale[blockIdx.y * static_cast<int64_t>(gridDim.x) + blockIdx.x] = s.scale;
}

template <typename T>
void launch_rows(const void* x, int64_t ldx, uint8_t* q, float* scale, int64_t lds, int64_t M, int64_t K,
                 unsigned* zero, int64_t zeros, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>(((K + kBlock - 1) / kBlock + kThreads / 16 - 1) / (kThreads / 16));
  const T* xt = static_cast<const T*>(x);
  // Many rows: four loads of a thread under way at once.
  if (M >= 512)
    launch_pdl(quantize_kernel<T, 4>, dim3(static_cast<unsigned>((M + 3) / 4), blocks), dim3(kThreads), 0, s, 1, xt,
               ldx, q, scale, lds, M, static_cast<int>(K), zero, zeros);
  else
    launch_pdl(quantize_kernel<T, 1>, dim3(static_cast<unsigned>(M), blocks), dim3(kThreads), 0, s, 1, xt, ldx, q,
               scale, lds, M, static_cast<int>(K), zero, zeros);
}
template <typename T>
void launch_weight(const void* w, int64_t ldw, uint8_t* q, float* scale, int64_t N, int64_t K, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((K + kBlock - 1) / kBlock), static_cast<unsigned>((N + kBlock - 1) / kBlock));
  launch_pdl(quantize_weight_kernel<T>, grid, dim3(kThreads), 0, s, 1, static_cast<const T*>(w), ldw, q, scale, N,
             static_cast<int>(K));
}

void check_shape(int64_t rows, int64_t K) {
  B200AR_CHECK(rows >= 0 && rows < (1ll << 31) && K > 0 && K < (1ll << 30), "bad shape for quantization");
  B200AR_CHECK(K % 16 == 0, "K must be a multiple of 16");
}

}  // namespace

void quantize(const void* x, int64_t ldx, uint8_t* q, float* scale, int64_t lds, int64_t M, int64_t K, Type type,
              unsigned* zero, int64_t zeros, cudaStream_t s) {
  const TraceRange trace("b200ar::quantize_fp8");
  check_shape(M, K);
  if (M == 0) return;
  switch (type) {
    case Type::kBf16: return launch_rows<__nv_bfloat16>(x, ldx, q, scale, lds, M, K, zero, zeros, s);
    case Type::kFp16: return launch_rows<__half>(x, ldx, q, scale, lds, M, K, zero, zeros, s);
    case Type::kFp32: return launch_rows<float>(x, ldx, q, scale, lds, M, K, zero, zeros, s);
  }
}

void quantize_weight(const void* w, int64_t ldw, uint8_t* q, float* scale, int64_t N, int64_t K, Type type,
                     cudaStream_t s) {
  const TraceRange trace("b200ar::quantize_fp8_weight");
  check_shape(N, K);
  B200AR_CHECK(N <= 65535ll * kBlock, "weights of at most 65535 * 128 rows");
  if (N == 0) return;
  switch (type) {
    case Type::kBf16: return launch_weight<__nv_bfloat16>(w, ldw, q, scale, N, K, s);
    case Type::kFp16: return launch_weight<__half>(w, ldw, q, scale, N, K, s);
    case Type::kFp32: return launch_weight<float>(w, ldw, q, scale, N, K, s);
  }
}

}  // namespace fp8
}  // namespace b200ar
