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
// Eight consecutive values as they are loaded, and the maximum of their absolute values as a bit pattern: fp32, or
// for the 16-bit types a pair of them, since a max of two 16-bit integers is one instruction.
template <typename T>
struct Eight {
  uint4 w;
  __device__ __forceinline__ void zero() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ unsigned amax() const {
    constexpr unsigned kAbs = 0x7fff7fffu;
    return larger(larger(w.x & kAbs, w.y & kAbs), larger(w.z & kAbs, w.w & kAbs));
  }
  static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return __vmaxu2(a, b); }
  static __device__ __forceinline__ unsigned fp32(unsigned m) {  // the pair's maximum as fp32 bits
    float v[8];
    unpack8<T>(make_uint4(max(m & 0xffffu, m >> 16), 0u, 0u, 0u), v);
    return __float_as_uint(v[0]);
  }
  __device__ __forceinline__ void get(float* v) const { unpack8<T>(w, v); }
};
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ unsigned amax() const {
    float v[8];
    get(v);
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  static __device__ __forceinline__ unsigned larger(unsigned x, unsigned y) { return max(x, y); }
  static __device__ __forceinline__ unsigned fp32(unsigned m) { return m; }
  __device__ __forceinline__ void get(float* v) const {
    *reinterpret_cast<float4*>(v) = a;
    *reinterpret_cast<float4*>(v + 4) = b;
  }
};

// A block's scale, and factors just below and above 1 / scale. With inverse = rn(1 / scale), each of the two and their
// products with a value are off by at most three roundings of 2^-24, less than the 2^-21 they were moved by: so
// v low <= rn(v / scale) <= v high in magnitude, and where both have one code it is the quotient's.
struct Scale {
  float scale, low, high;
  bool divide;  // 1 / scale may not be a normal number
  __device__ __forceinline__ explicit Scale(unsigned amax_bits) {
    scale = __fdiv_rn(__uint_as_float(amax_bits), kMax);
    if (scale == 0.f) scale = 1.f;  // a block of zeros, or of fp32 values up to 224 2^-149: all codes are 0
    const float inverse = __frcp_rn(scale);
    low = inverse * (1.f - 0x1p-21f);
    high = inverse * (1.f + 0x1p-21f);
    divide = scale < 0x1p-120f;
  }
};
__device__ __forceinline__ uint32_t code2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 encode8(const float* v, const Scale& s) {
  uint32_t lo[4], hi[4], differ = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = code2(v[2 * i] * s.low, v[2 * i + 1] * s.low);
    hi[i] = code2(v[2 * i] * s.high, v[2 * i + 1] * s.high);
    differ |= lo[i] ^ hi[i];
  }
  if (differ != 0u || s.divide)
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = code2(__fdiv_rn(v[2 * i], s.scale), __fdiv_rn(v[2 * i + 1], s.scale));
  return make_uint2(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16));
}

}  // namespace fp8
}  // namespace b200ar
