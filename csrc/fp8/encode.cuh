// Values to e4m3 codes with the scale of their block (fp8.h), for the kernels that quantize.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace b200ar {
namespace fp8 {

constexpr float kMax = 448.f;

// Eight 16-bit values as fp32.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float* v);
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& w, float* v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void unpack8<__half>(const uint4& w, float* v) {
  const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// Eight consecutive values as fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  unpack8<T>(*reinterpret_cast<const uint4*>(p), v);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* v) {
  *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
  *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(p + 4);
}

__device__ __forceinline__ unsigned abs_max8(const float* v) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ float scale_of(unsigned amax_bits) {
  return amax_bits == 0u ? 1.f : __fdiv_rn(__uint_as_float(amax_bits), kMax);
}
// `inverse` is 1 / scale, or NaN where that is not a normal number.
__device__ __forceinline__ float inverse_of(float scale) {
  return scale >= 0x1p-120f ? __frcp_rn(scale) : __uint_as_float(0x7fffffffu);
}
__device__ __forceinline__ uint2 encode8(const float* v, float scale, float inverse) {
  float y[8];
  bool near = !(inverse == inverse);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = v[i] * inverse;
    const uint32_t u = __float_as_uint(y[i]);
    // Three bits of the mantissa stay: the middle is a one behind them, then zeros. Zero itself has the code zero.
    near |= ((u & 0xfffffu) - 0x7fffcu <= 8u) | (fabsf(y[i]) < 0x1p-5f && v[i] != 0.f);
  }
  if (near)
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(v[i], scale);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

}  // namespace fp8
}  // namespace b200ar
