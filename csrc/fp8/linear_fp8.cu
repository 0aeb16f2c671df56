// Matrix product of e4m3 operands with block scales:
//
//   out[m, n] = sum_b sx[b, m] sw[n / 128, b] sum_{k in block b} x[m, k] w[n, k]
//
// The simplest form: 64 x 64 output tiles, operands widened to fp32 in shared
// memory, sums in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../common/check.h"
#include "../common/pdl.h"
#include "../common/trace.h"
#include "fp8.h"

namespace b200ar {
namespace fp8 {

namespace {

__device__ __forceinline__ float decode(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

template <typename T>
__global__ void __launch_bounds__(256) linear_simple_kernel(const LinearArgs a) {
  __shared__ float sx[16][65], sw[16][65];
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * 64, n0 = static_cast<int64_t>(blockIdx.y) * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t kblocks = (a.K + kBlock - 1) / kBlock;
  float acc[4][4] = {};
  pdl_wait();
  pdl_trigger();
  for (int64_t b = 0; b < kblocks; ++b) {
    float part[4][4] = {};
    for (int64_t k0 = b * kBlock; k0 < min((b + 1) * kBlock, a.K); k0 += 16) {
      __syncthreads();
      for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int r = i >> 4, c = i & 15;
        sx[c][r] = m0 + r < a.M ? decode(a.x[(m0 + r) * a.K + k0 + c]) : 0.f;
        sw[c][r] = n0 + r < a.N ? decode(a.w[(n0 + r) * a.K + k0 + c]) : 0.f;
      }
      __syncthreads();
      for (int c = 0; c < 16; ++c)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) part[i][j] += sx[c][ty + 16 * i] * sw[c][tx + 16 * j];
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
        if (m < a.M && n < a.N) acc[i][j] += part[i][j] * a.sx[b * a.lds + m] * a.sw[(n / kBlock) * kblocks + b];
      }
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < a.M && n < a.N) put(static_cast<T*>(a.out) + m * a.ldo + n, acc[i][j]);
    }
}

}  // namespace

void linear(const LinearArgs& a, Type out, cudaStream_t s) {
  const TraceRange trace("b200ar::linear_fp8");
  B200AR_CHECK(a.M >= 0 && a.M < (1ll << 30) && a.N > 0 && a.N < (1ll << 21) && a.K > 0 && a.K < (1ll << 30),
               "bad shape for linear_fp8");
  B200AR_CHECK(a.K % 16 == 0 && a.N % 8 == 0, "K must be a multiple of 16 and N of 8");
  if (a.M == 0) return;
  const dim3 grid(static_cast<unsigned>((a.M + 63) / 64), static_cast<unsigned>((a.N + 63) / 64));
  if (out == Type::kBf16)
    launch_pdl(linear_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, 1, a);
  else
    launch_pdl(linear_simple_kernel<__half>, grid, dim3(256), 0, s, 1, a);
}

}  // namespace fp8
}  // namespace b200ar
