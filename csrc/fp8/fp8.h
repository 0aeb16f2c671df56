// Host API of the 8-bit linear layer (quantize.cu, linear_fp8.cu).
//
// e4m3 values with one fp32 scale for each block of 128 along K: activations
// have a scale for each row and block, weights one for each 128 x 128 block.
// A block's scale is amax / 448 (1 where that is zero), a value's code
// is x / scale rounded to the nearest e4m3 number.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace b200ar {
namespace fp8 {

constexpr int kBlock = 128;

enum class Type { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

// x [M, K] (row stride ldx elements) to q [M, K] (contiguous) and scale
// [blocks, M]: the scales of a block for all rows are contiguous, row stride lds.
// `zero` (or null): `zeros` words that are set to zero on the way.
void quantize(const void* x, int64_t ldx, uint8_t* q, float* scale, int64_t lds, int64_t M, int64_t K, Type type,
              unsigned* zero, int64_t zeros, cudaStream_t s);

// w [N, K] (row stride ldw) to q [N, K] and scale [ceil(N / 128), ceil(K / 128)].
void quantize_weight(const void* w, int64_t ldw, uint8_t* q, float* scale, int64_t N, int64_t K, Type type,
                     cudaStream_t s);

struct LinearArgs {
  // x as codes [M, K] with scales [ceil(K / 128), M], row stride lds; or raw: [M, K] of the output's type, row
  // stride ldx, quantized here.
  const uint8_t* x;
  const float* sx;
  int64_t lds;
  const void* raw;
  int64_t ldx;
  const uint8_t* w;   // [N, K]
  const float* sw;    // [ceil(N / 128), ceil(K / 128)]
  void* out;          // [M, N], row stride ldo
  int64_t ldo;
  int64_t M, N, K;
  int* err;
  float* workspace;    // set by linear()
  unsigned* counters;
};
// Whether a call of these sizes on the current device takes the kernel for many rows.
bool linear_takes_pairs(int64_t M, int64_t N, int64_t K);
// Bytes of scratch of a call; not kept from call to call.
int64_t linear_scratch(const LinearArgs& a);
// out = sum over blocks b of sx[b, m] sw[n / 128, b] (x[m, b] . w[n, b])
void linear(const LinearArgs& a, Type out, void* scratch, cudaStream_t s);

}  // namespace fp8
}  // namespace b200ar
