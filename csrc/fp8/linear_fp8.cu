// Matrix product of e4m3 operands with block scales on the 5th-generation tensor cores:
//
//   out[m, n] = sum_b sx[b, m] sw[n / 128, b] sum_{k in block b} x[m, k] w[n, k]
//
// A block of 128 values of K is one 128-byte row of a swizzled tile and four
// tcgen05.mma (kind::f8f6f4, K = 32). Scales differ from block to block, so the
// tensor core sums one block at a time into tensor memory; four or eight warps
// take it from there, scale it and add it in fp32 registers while the next
// block is multiplied. Two kernels:
//
// rows_kernel (few rows of x). The weights' 128 rows are the product's M, the
//   rows of x (16 to 128) its N, so a product moves each weight once whatever
//   the number of rows. The K blocks are split over the CTAs of a cluster,
//   which add their sums through distributed shared memory: no workspace. The
//   weights' first tiles are on their way before the kernel waits for the
//   quantization of x. Bound by the stream of the weights behind two launches:
//   1 x 7168 x 8192 takes 15.5 us with the quantization (59 MB, 9.0 us at the
//   copy rate), 48 x 8192 x 3584 12.7 us (30 MB, 4.7 us). With 65 to 128 rows one
//   CTA fits an SM (254 registers a thread) and 7168 x 8192 takes 36 to 38 us.
// pair_kernel (many rows). CTA pairs (cta_group::2) compute 256 x 256 tiles. A K
//   block's sums go to one of two buffers in tensor memory, each in two halves
//   of 128 columns with a warpgroup and barriers of its own: handing a buffer
//   over and back takes about as long as its products (signals between the CTAs
//   included), so four half buffers keep more of them in flight than two whole
//   ones. Two warps read the scales four K blocks ahead and hand their products
//   over through shared memory: read by those that need them they made every
//   block wait. All tiles' K blocks form
//   one line that is cut into equal parts for the pairs, so no pair idles in a
//   last partial wave. A tile that a cut falls into is finished by the pair that
//   arrives last, which adds the parts in the order of K. Bound by the way of
//   every block's sums out of tensor memory (tensor core 44 % of the active cycles,
//   issue slots 41 %, DRAM 23 %): 4093 x 7168 x 8192 with the quantization takes 306
//   us in a short run, 1570 TFLOP/s, and 360 us in a long one, at the power limit.
//
// Every wait is bounded: on expiry the error word is set and all roles run
// down without waiting.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "../common/check.h"
#include "../common/pdl.h"
#include "../common/trace.h"
#include "../gemm/tcgen05.cuh"
#include "fp8.h"

namespace b200ar {
namespace fp8 {

namespace {

constexpr int kErrTimeout = 5;  // in the error word that other operators share; a bounded wait expired

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

// D fp32, A and B e4m3, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_e4m3_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Four bytes to shared memory, and the arrival on a barrier once all of the thread's copies so far are there.
__device__ __forceinline__ void cp_async4(void* smem, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sm100::smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ uint64_t pack64(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void unpack64(uint64_t v, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  lo = __uint_as_float(a);
  hi = __uint_as_float(b);
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t both(float x) { return pack64(__float_as_uint(x), __float_as_uint(x)); }

__device__ __forceinline__ bool normal(float x) { return fabsf(x) >= 0x1p-126f && fabsf(x) < INFINITY; }

// A block's sum r (0, or from 2^-18 to 2^25) times two scales a and b, as (r first) b second: whatever the scales, a
// product on the way is out of range only if the result is. (r a is a normal number for a between 2^-100 and 2^100;
// outside, a power of two of a's is left for the end.)
__device__ __forceinline__ void around(float a, float& first, float& second) {
  const bool high = fabsf(a) > 0x1p100f, low = fabsf(a) < 0x1p-100f;
  first = high ? 0x1p64f : low ? 0x1p-64f : a;
  second = high ? a * 0x1p-64f : low ? a * 0x1p64f : 1.f;
}

struct Args {
  const float* sx;  // [kblocks, M], row stride lds
  const float* sw;  // [ceil(N / 128), kblocks]
  void* out;        // [M, N], row stride ldo
  int64_t lds, ldo;
  int M, N, kblocks;
  int* err;
};

// ------------------------------------------------------------------ few rows
template <int MP>  // rows of x in a tile
struct RowsCfg {
  static constexpr int kThreads = 224;
  static constexpr uint32_t kW = 128 * 128, kX = MP * 128, kStage = kW + kX;
  // Two CTAs fit an SM, or one at 128 rows: their sums take 254 registers a thread (and the ring's space at the end).
  static constexpr int kStages = (100 * 1024) / kStage;
  static constexpr int kBufs = MP == 128 ? 2 : 4;  // accumulators in tensor memory
  static constexpr uint32_t kCols = kBufs * MP;    // a power of two from 64 to 256
  static constexpr int kScales = 8;                // ring of K blocks' scales: of the rows of x, of those of W
  static constexpr int kScaleFloats = MP + 4;
  static constexpr size_t kSmem = 1024 + kStages * kStage + kScales * kScaleFloats * 4 + 512;
  static_assert(MP * 128 * 4 <= kStages * kStage, "the sums of a CTA reuse the ring");
};

// Grid: clusters of `splits` CTAs along x; cluster (x / splits) has 128 rows of W, y 128 or fewer rows of x.
template <typename T, int MP>
__global__ void __launch_bounds__(RowsCfg<MP>::kThreads)
    rows_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx, const Args a,
                int splits, int early) {
  using C = RowsCfg<MP>;
  extern __shared__ __align__(1024) uint8_t rows_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(rows_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = smem + C::kStages * C::kW;
  float* scales = reinterpret_cast<float*>(smem + C::kStages * C::kStage);  // [kScales][kScaleFloats]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + C::kScales * C::kScaleFloats);
  uint64_t* empty = full + C::kStages;
  uint64_t* tfull = empty + C::kStages;
  uint64_t* tempty = tfull + C::kBufs;
  uint64_t* sfull = tempty + C::kBufs;
  uint64_t* sempty = sfull + C::kScales;
  uint64_t* drained = sempty + C::kScales;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* s_err = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * C::kStages + 2 * C::kBufs + 2 * C::kScales + 2) * 8 <= 512, "barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int block = blockIdx.x / splits, rank = blockIdx.x % splits;
  const int m0 = blockIdx.y * MP;
  const int kb0 = a.kblocks * rank / splits, kb1 = a.kblocks * (rank + 1) / splits, nkb = kb1 - kb0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      sm100::mbar_init(&full[i], 1);
      sm100::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::kBufs; ++i) {
      sm100::mbar_init(&tfull[i], 1);
      sm100::mbar_init(&tempty[i], 4);
    }
    for (int i = 0; i < C::kScales; ++i) {
      sm100::mbar_init(&sfull[i], 32);
      sm100::mbar_init(&sempty[i], 4);
    }
    sm100::mbar_init(drained, 1);
    *s_err = 0;
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&tw);
    sm100::prefetch_tmap(&tx);
  }
  if (warp == 1) {
    sm100::tmem_alloc(tmem_slot, C::kCols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* b, uint32_t parity) {
    if (sm100::mbar_try_wait(b, parity)) return;
    if (!*s_err && !sm100::mbar_wait(b, parity)) *s_err = 1;
  };

  uint64_t acc[MP / 2];  // pairs of rows of x
#pragma unroll
  for (int i = 0; i < MP / 2; ++i) acc[i] = 0;

  if (warp == 0) {
    if (sm100::elect_one()) {
      // With `early` the kernel before is the quantization of x, which started after everything before it was
      // done: the weights are there, and the first ring of them is requested while x is still being written.
      const int pre = early ? min(nkb, C::kStages) : 0;
      for (int i = 0; i < pre; ++i) {
        sm100::mbar_arrive_expect_tx(&full[i], C::kStage);
        sm100::tma_load_2d(sW + i * C::kW, &tw, &full[i], (kb0 + i) * kBlock, block * 128);
      }
      pdl_wait();
      for (int i = 0; i < pre; ++i) sm100::tma_load_2d(sX + i * C::kX, &tx, &full[i], (kb0 + i) * kBlock, m0);
      int issued = pre;
      for (; issued < nkb; ++issued) {
        const int st = issued % C::kStages;
        wait(&empty[st], ((issued / C::kStages) & 1) ^ 1);
        if (*s_err) break;
        sm100::mbar_arrive_expect_tx(&full[st], C::kStage);
        sm100::tma_load_2d(sW + st * C::kW, &tw, &full[st], (kb0 + issued) * kBlock, block * 128);
        sm100::tma_load_2d(sX + st * C::kX, &tx, &full[st], (kb0 + issued) * kBlock, m0);
      }
      // Never leave while a copy into this CTA's shared memory is in flight.
      for (int i = max(0, issued - C::kStages); i < issued; ++i)
        sm100::mbar_wait(&full[i % C::kStages], (i / C::kStages) & 1);
    }
    __syncwarp();
    pdl_wait();
  } else if (warp == 1) {
    if (sm100::elect_one()) {
      for (int i = 0; i < nkb && !*s_err; ++i) {
        const int st = i % C::kStages, bf = i % C::kBufs;
        wait(&tempty[bf], ((i / C::kBufs) & 1) ^ 1);
        wait(&full[st], (i / C::kStages) & 1);
        if (*s_err) break;
        sm100::tc_fence_after();
        const uint64_t dw = sm100::smem_desc_sw128(sW + st * C::kW);
        const uint64_t dx = sm100::smem_desc_sw128(sX + st * C::kX);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_e4m3(tmem + bf * MP, dw + 2 * k, dx + 2 * k, idesc_e4m3(128, MP), k > 0 ? 1u : 0u);
        sm100::mma_commit(&empty[st]);
        sm100::mma_commit(&tfull[bf]);
      }
      sm100::mma_commit(drained);
      if (!sm100::mbar_wait(drained, 0)) *s_err = 1;
    }
    __syncwarp();
    pdl_wait();
  } else if (warp == 6) {
    // Scales, up to eight K blocks ahead: read straight from global memory by the warps below they would be waited
    // for with every block.
    pdl_wait();
    const float* sw = a.sw + static_cast<int64_t>(block) * a.kblocks + kb0;
    for (int i = 0; i < nkb; ++i) {
      const int sl = i % C::kScales;
      wait(&sempty[sl], ((i / C::kScales) & 1) ^ 1);
      float* dst = scales + sl * C::kScaleFloats;
      const float* sx = a.sx + (kb0 + i) * a.lds + m0;
#pragma unroll
      for (int m = lane; m < MP; m += 32) cp_async4(dst + m, sx + min(m, a.M - 1 - m0));
      if (lane == 0) cp_async4(dst + MP, sw + i);
      cp_async_arrive(&sfull[sl]);
    }
    cp_async_wait_all();
  } else {
    // Thread = row of W.
    pdl_wait();
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    for (int i = 0; i < nkb; ++i) {
      const int bf = i % C::kBufs, sl = i % C::kScales;
      wait(&sfull[sl], (i / C::kScales) & 1);
      const float* sc = scales + sl * C::kScaleFloats;
      const float sw = sc[MP];
      wait(&tfull[bf], (i / C::kBufs) & 1);
      sm100::tc_fence_after();
      constexpr int kStep = MP < 32 ? MP : 32;
      float first, second;
      around(sw, first, second);
      const uint64_t first2 = both(first), second2 = both(second);
#pragma unroll
      for (int c = 0; c < MP; c += kStep) {
        uint32_t r[kStep];
        if constexpr (kStep == 16)
          sm100::tmem_ld_32x32b_x16(tmem + lanes + bf * MP + c, r);
        else
          sm100::tmem_ld_32x32b_x32(tmem + lanes + bf * MP + c, r);
        sm100::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < kStep; e += 4) {
          const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(sc + c + e);  // scales of four rows
          uint64_t* sum = acc + (c + e) / 2;
          sum[0] = fma2(mul2(mul2(pack64(r[e], r[e + 1]), first2), s.x), second2, sum[0]);
          sum[1] = fma2(mul2(mul2(pack64(r[e + 2], r[e + 3]), first2), s.y), second2, sum[1]);
        }
      }
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        sm100::mbar_arrive(&tempty[bf]);
        sm100::mbar_arrive(&sempty[sl]);
      }
    }
  }
  pdl_trigger();
  sm100::tc_fence_before();
  __syncthreads();  // copies and products are done: the ring is free
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, C::kCols);
  }
  // Sums of the cluster: [row of x][row of W] in each CTA, added in the order of K.
  float* sums = reinterpret_cast<float*>(smem);
  if (warp >= 2 && warp < 6) {
    const int id = (warp & 3) * 32 + lane;
#pragma unroll
    for (int i = 0; i < MP; i += 2) {
      float x, y;
      unpack64(acc[i / 2], x, y);
      if (m0 + i < a.M) sums[i * 128 + id] = x;
      if (m0 + i + 1 < a.M) sums[(i + 1) * 128 + id] = y;
    }
  }
  if (splits > 1)
    sm100::cluster_sync();
  else
    __syncthreads();
  const int rows = min(MP, a.M - m0);
  const uint32_t base = sm100::smem_u32(sums);
  // Four columns of a row a thread; this CTA has every splits-th group of them.
  for (int i = rank * C::kThreads + threadIdx.x; i < rows * 32; i += splits * C::kThreads) {
    const int r = i >> 5, c = (i & 31) * 4, n = block * 128 + c;
    if (n >= a.N) continue;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < splits; ++p) {
      const uint32_t addr = splits > 1 ? sm100::mapa_shared(base, p) + (r * 128 + c) * 4 : 0;
      float4 v;
      if (splits > 1)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                     : "r"(addr)
                     : "memory");
      else
        v = *reinterpret_cast<const float4*>(sums + r * 128 + c);
      y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
    }
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (m0 + r) * a.ldo + n) =
        make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
  }
  if (splits > 1) sm100::cluster_sync();  // no CTA leaves while another reads its sums
  if (threadIdx.x == 0 && *s_err) atomicExch(a.err, kErrTimeout);
}

// ------------------------------------------------------------------ many rows
namespace pair {

constexpr int BM = 256, BN = 256;
constexpr int kStages = 6;
constexpr int kThreads = 384;  // three warpgroups of 168 registers a thread: 56 and twice 224 after the split
constexpr uint32_t kA = 128 * 128, kB = 128 * 128, kStage = kA + kB;  // a CTA's halves
constexpr int kScales = 8;           // ring of K blocks' factors (products of two scales): [2 halves][128 rows]
constexpr int kScaleFloats = 260;    // and a mark of each warp that made them
constexpr size_t kSmem = 1024 + kStages * kStage + kScales * kScaleFloats * 4 + 512;
constexpr uint32_t kCols = 512;      // [2 buffers][2 halves of the tile's columns][128]
constexpr int64_t kPartFloats = 128 * 256;  // a CTA's sums of a tile

struct Line {
  int tiles_m, tiles;
  int64_t units;  // tiles * kblocks
  int pairs;
  float* parts;    // [pairs][2][2 CTAs][kPartFloats]
  unsigned* done;  // [tiles][2], zero
  __device__ __forceinline__ int64_t start(int p) const { return units * p / pairs; }
  // The pair whose part holds a unit.
  __device__ __forceinline__ int owner(int64_t u) const { return static_cast<int>((pairs * (u + 1) - 1) / units); }
  __device__ __forceinline__ float* part(int p, int which, int rank) const {
    return parts + (static_cast<int64_t>(p * 2 + which) * 2 + rank) * kPartFloats;
  }
};

__device__ __forceinline__ void sum_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// Multiplies 128 columns of the calling warp's sums in tensor memory.
__device__ __forceinline__ void scale_sums(uint32_t at, float first, float second) {
#pragma unroll 1
  for (int c = 0; c < 128; c += 16) {
    uint32_t r[16];
    sm100::tmem_ld_32x32b_x16(at + c, r);
    sm100::tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * first * second);
    sm100::tmem_st_32x32b_x16(at + c, r);
  }
  sm100::tmem_st_wait();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, const Args a,
                const Line line) {
  extern __shared__ __align__(1024) uint8_t pair_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pair_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + kStages * kA;
  float* scales = reinterpret_cast<float*>(smem + kStages * kStage);  // [kScales][kScaleFloats]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + kScales * kScaleFloats);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;  // [2 buffers][2 halves]
  uint64_t* tempty = tfull + 4;       // the same (the leader's: four warps of each CTA)
  uint64_t* sfull = tempty + 4;       // [kScales]
  uint64_t* sempty = sfull + kScales;
  uint64_t* drained = sempty + kScales;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* s_err = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_last = const_cast<int*>(s_err) + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = sm100::cluster_ctarank();
  const bool leader = rank == 0;
  const int p = blockIdx.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      sm100::mbar_init(&full[i], 1);
      sm100::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      sm100::mbar_init(&tfull[i], 1);
      sm100::mbar_init(&tempty[i], 8);
    }
    for (int i = 0; i < kScales; ++i) {
      sm100::mbar_init(&sfull[i], 64);
      sm100::mbar_init(&sempty[i], 8);
    }
    sm100::mbar_init(drained, 1);
    *s_err = 0;
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&tx);
    sm100::prefetch_tmap(&tw);
  }
  if (warp == 9) {
    sm100::tmem_alloc_pair(tmem_slot, kCols);
    sm100::tmem_relinquish_pair();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();  // both CTAs' barriers exist before any signal between them
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* b, uint32_t parity) {
    if (sm100::mbar_try_wait(b, parity)) return;
    if (!*s_err && !sm100::mbar_wait(b, parity)) *s_err = 1;
  };
  pdl_wait();
  pdl_trigger();
  const int64_t u0 = line.start(p), u1 = line.start(p + 1);
  const int count = static_cast<int>(u1 - u0);

  if (warp >= 8) {
    sm100::reg_give<56>();
    int tile = static_cast<int>(u0 / a.kblocks), kb = static_cast<int>(u0 - int64_t(tile) * a.kblocks);
    if (warp == 8 && sm100::elect_one()) {
      // -------------------------------------------------------- TMA producer
      int st = 0, n = 0;
      uint32_t phase = 0;
      const uint32_t fbar = sm100::mapa_shared(sm100::smem_u32(full), 0);
      for (; n < count; ++n) {
        const int ym = tile % line.tiles_m * BM + static_cast<int>(rank) * 128;
        const int yn = tile / line.tiles_m * BN + static_cast<int>(rank) * 64;
        wait(&empty[st], phase ^ 1u);
        if (*s_err) break;
        if (leader) sm100::mbar_arrive_expect_tx(&full[st], 2 * kStage);  // both CTAs' bytes
        sm100::tma_load_2d_pair(sA + st * kA, &tx, fbar + st * 8, kb * kBlock, ym);
        // Half of each half of the tile's columns: a product of one half reads 64 rows of W from either CTA.
        sm100::tma_load_2d_pair(sB + st * kB, &tw, fbar + st * 8, kb * kBlock, yn);
        sm100::tma_load_2d_pair(sB + st * kB + kB / 2, &tw, fbar + st * 8, kb * kBlock, yn + 128);
        if (++st == kStages) st = 0, phase ^= 1u;
        if (++kb == a.kblocks) kb = 0, ++tile;
      }
      if (leader)
        for (int i = max(0, n - kStages); i < n; ++i) sm100::mbar_wait(&full[i % kStages], (i / kStages) & 1);
    }
    if (warp == 9 && leader && sm100::elect_one()) {
      // -------------------------------------------------------- MMA issue (leader)
      int st = 0;
      uint32_t phase = 0;
      uint32_t empty_at[2], tfull_at[2];
      for (uint32_t r = 0; r < 2; ++r) {
        empty_at[r] = sm100::mapa_shared(sm100::smem_u32(empty), r);
        tfull_at[r] = sm100::mapa_shared(sm100::smem_u32(tfull), r);
      }
      const uint64_t da0 = sm100::smem_desc_sw128(sA), db0 = sm100::smem_desc_sw128(sB);
      for (int i = 0; i < count && !*s_err; ++i) {
        const int bf = i & 1;
        const uint64_t da = da0 + st * (kA >> 4);
        wait(&full[st], phase);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          wait(&tempty[bf * 2 + h], ((i >> 1) & 1u) ^ 1u);
          if (*s_err) break;
          sm100::tc_fence_after();
          const uint64_t db = db0 + st * (kB >> 4) + h * (kB >> 5);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_e4m3_pair(tmem + bf * 256 + h * 128, da + 2 * k, db + 2 * k, idesc_e4m3(BM, 128), k > 0 ? 1u : 0u);
          sm100::mma_commit_pair(tfull_at[0] + (bf * 2 + h) * 8);
          sm100::mma_commit_pair(tfull_at[1] + (bf * 2 + h) * 8);
        }
        sm100::mma_commit_pair(empty_at[0] + st * 8);
        sm100::mma_commit_pair(empty_at[1] + st * 8);
        if (++st == kStages) st = 0, phase ^= 1u;
      }
      sm100::mma_commit_pair(sm100::mapa_shared(sm100::smem_u32(drained), 0));
      if (!sm100::mbar_wait(drained, 0)) *s_err = 1;
    }
    if (warp >= 10) {
      // -------------------------------------------------------- factors: two rows a lane, four K blocks ahead
      constexpr int kAhead = 4;
      const int id = (warp - 10) * 32 + lane, nblocks = (a.N + kBlock - 1) / kBlock;
      float x[kAhead][2], w[kAhead][2];
      auto load = [&](float* xs, float* ws) {
        const int m = tile % line.tiles_m * BM + static_cast<int>(rank) * 128 + id, nb = tile / line.tiles_m * 2;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          xs[h] = __ldg(a.sx + kb * a.lds + min(m + 64 * h, a.M - 1));
          ws[h] = __ldg(a.sw + static_cast<int64_t>(min(nb + h, nblocks - 1)) * a.kblocks + kb);
        }
        if (++kb == a.kblocks) kb = 0, ++tile;
      };
#pragma unroll
      for (int e = 0; e < kAhead; ++e)
        if (e < count) load(x[e], w[e]);
#pragma unroll 1
      for (int i = 0; i < count; i += kAhead) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
          if (i + e >= count) break;
          const int sl = (i + e) % kScales;
          wait(&sempty[sl], (((i + e) / kScales) & 1u) ^ 1u);
          float* dst = scales + sl * kScaleFloats;
          bool all = true;
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float f = x[e][h] * w[e][g];
              dst[g * 128 + id + 64 * h] = f;
              all = all && normal(f);
            }
          const unsigned odd = __ballot_sync(0xffffffffu, !all);
          if (lane == 0) reinterpret_cast<unsigned*>(dst)[256 + warp - 10] = odd;
          sm100::mbar_arrive(&sfull[sl]);
          if (i + e + kAhead < count) load(x[e], w[e]);
        }
      }
    }
  } else {
    // ---------------------------------------------------------- scale, add, store: 8 warps
    sm100::reg_take<224>();
    const int g = warp >> 2, row = (warp & 3) * 32 + lane;  // half of the tile's columns, row of the CTA
    const uint32_t td = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + g * 128;
    const uint32_t free_bar[2] = {sm100::mapa_shared(sm100::smem_u32(&tempty[g]), 0),
                                  sm100::mapa_shared(sm100::smem_u32(&tempty[2 + g]), 0)};
    unsigned n = 0;
    for (int64_t u = u0; u < u1;) {
      const int tile = static_cast<int>(u / a.kblocks), k0 = static_cast<int>(u - int64_t(tile) * a.kblocks);
      const int k1 = static_cast<int>(min(static_cast<int64_t>(a.kblocks), k0 + u1 - u));
      const int tm = tile % line.tiles_m, tn = tile / line.tiles_m;
      const int m = tm * BM + static_cast<int>(rank) * 128 + row, n0 = tn * BN + g * 128;
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      for (int kb = k0; kb < k1; ++kb, ++n) {
        const int bf = n & 1, sl = n % kScales;
        wait(&sfull[sl], (n / kScales) & 1u);
        float sf = scales[sl * kScaleFloats + g * 128 + row];
        const uint2 odd = *reinterpret_cast<const uint2*>(scales + sl * kScaleFloats + 256);
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&sempty[sl]);
        wait(&tfull[bf * 2 + g], (n >> 1) & 1u);
        sm100::tc_fence_after();
        // Where a factor of the block is not a normal number, two of three (around()) are multiplied into the row's sums
        // in tensor memory first; other rows' stay as they are. (Measured for 4093 x 7168 x 8192, this kernel alone:
        // with one product for every block, right or not, 266 us; this way 270; tested here 275; with a second form of
        // the loop below 314.)
        if ((odd.x | odd.y) != 0u) {
          float first = 1.f, sx = 1.f;
          if (!normal(sf)) {
            sx = __ldg(a.sx + kb * a.lds + min(m, a.M - 1));
            const int64_t nb = min(tn * 2 + g, (a.N + kBlock - 1) / kBlock - 1);
            around(__ldg(a.sw + nb * a.kblocks + kb), first, sf);
          }
          scale_sums(td + bf * BN, first, sx);
        }
        const uint64_t s = both(sf);
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          uint32_t r[32];
          sm100::tmem_ld_32x32b_x32(td + bf * BN + c, r);
          sm100::tmem_ld_wait();
          if (c == 96) {  // the half buffer is read: the next block but one may overwrite it
            sm100::tc_fence_before();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive_remote(free_bar[bf]);
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) acc[(c + e) / 2] = fma2(pack64(r[e], r[e + 1]), s, acc[(c + e) / 2]);
        }
      }
      u += k1 - k0;

      if (k1 - k0 < a.kblocks) {
        // A cut tile: whoever arrives last has all parts and adds them in the order of K. (Of two parts it adds the
        // other to its own: the sum of two numbers has no order.) Each CTA of the pair has its own rows.
        const int first = line.owner(int64_t(tile) * a.kblocks);
        const int last = line.owner(int64_t(tile + 1) * a.kblocks - 1);
        const unsigned others = static_cast<unsigned>(last - first);
        unsigned* done = line.done + tile * 2 + rank;
        volatile int* is_last = s_last;
        if (threadIdx.x == 0) *is_last = others == 1 && atomicAdd(done, 0u) == others;
        sum_sync();
        if (!*is_last) {
          float4* dst = reinterpret_cast<float4*>(line.part(p, k0 > 0 ? 0 : 1, rank)) + g * 32 * 128 + row;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float4 v;
            unpack64(acc[2 * i], v.x, v.y);
            unpack64(acc[2 * i + 1], v.z, v.w);
            __stcg(dst + i * 128, v);
          }
          __threadfence();
          sum_sync();
          if (threadIdx.x == 0) *is_last = atomicAdd(done, 1u) == others;
          sum_sync();
        }
        const bool finish = *is_last != 0;
        __threadfence();
        sum_sync();  // s_last may be written again
        if (!finish) continue;
        if (others > 1) {
#pragma unroll
          for (int i = 0; i < 64; ++i) acc[i] = 0;
        }
        for (int o = first; o <= last; ++o) {
          if (others == 1 && o == p) continue;
          const float4* src = reinterpret_cast<const float4*>(line.part(o, o > first ? 0 : 1, rank)) + g * 32 * 128 + row;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {  // eight loads under way
            float4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __ldcg(src + (i + e) * 128);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float x, y;
              unpack64(acc[2 * (i + e)], x, y);
              acc[2 * (i + e)] = pack64(__float_as_uint(x + v[e].x), __float_as_uint(y + v[e].y));
              unpack64(acc[2 * (i + e) + 1], x, y);
              acc[2 * (i + e) + 1] = pack64(__float_as_uint(x + v[e].z), __float_as_uint(y + v[e].w));
            }
          }
        }
      }
      T* out = static_cast<T*>(a.out) + static_cast<int64_t>(m) * a.ldo + n0;
#pragma unroll
      for (int c = 0; c < 128; c += 8) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) unpack64(acc[c / 2 + e], y[2 * e], y[2 * e + 1]);
        if (m < a.M && n0 + c < a.N)  // N is a multiple of 8
          *reinterpret_cast<uint4*>(out + c) =
              make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
      }
    }
  }

  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();  // neither CTA leaves while the pair's products or signals may touch it
  if (warp == 9) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc_pair(tmem, kCols);
  }
  if (threadIdx.x == 0 && *s_err) atomicExch(a.err, kErrTimeout);
}

}  // namespace pair

// ------------------------------------------------------------------ host side
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode() {
  static EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    B200AR_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q));
    if (q != cudaDriverEntryPointSuccess || !ptr) throw std::runtime_error("cuTensorMapEncodeTiled unavailable");
    return reinterpret_cast<EncodeFn>(ptr);
  }();
  return fn;
}

// Codes [rows, K], box of box_rows x 128.
CUtensorMap codes_map(const void* base, int64_t rows, int64_t K, int box_rows) {
  CUtensorMap m;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(K)};
  const cuuint32_t box[2] = {kBlock, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = encode()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled (e4m3) failed: " + std::to_string(r));
  return m;
}

int sm_count() {
  int dev = 0, n = 0;
  B200AR_CUDA(cudaGetDevice(&dev));
  B200AR_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
  return n;
}

template <typename T, int MP>
void launch_rows(const LinearArgs& l, const Args& a, int splits, cudaStream_t s) {
  using C = RowsCfg<MP>;
  const CUtensorMap tw = codes_map(l.w, l.N, l.K, 128), tx = codes_map(l.x, l.M, l.K, MP);
  auto kern = rows_kernel<T, MP>;
  static PerDeviceOnce attr;
  attr([&] {
    B200AR_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem)));
  });
  const dim3 grid(static_cast<unsigned>((l.N + 127) / 128 * splits), static_cast<unsigned>((l.M + MP - 1) / MP));
  launch_pdl(kern, grid, dim3(C::kThreads), C::kSmem, s, splits, tw, tx, a, splits, l.raw ? 1 : 0);
}

// K blocks of a pair's part at least: shorter parts take longer to add than to compute.
constexpr int64_t kPartUnits = 12;

int64_t pair_tiles(const LinearArgs& l) {
  return (l.M + pair::BM - 1) / pair::BM * ((l.N + pair::BN - 1) / pair::BN);
}
int64_t pair_units(const LinearArgs& l) { return pair_tiles(l) * ((l.K + kBlock - 1) / kBlock); }
int pairs_of(const LinearArgs& l) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count() / 2, pair_units(l) / kPartUnits)));
}

// Whether pair_kernel takes a call: above one tile of rows_kernel, if there is a part for every pair (888 K blocks of
// tiles on 148 SMs). Measured (rows_kernel, pair_kernel): 128 x 7168 x 8192 43, 45 us; 256 x 7168 x 8192 67, 45 us (1792
// K blocks of tiles); 512 x 1280 x 8192 41, 39 us (640), which the rule leaves to the slower by 2 us; 300 x 4096 x 2048
// 29, 35 us (512); 333 x 1288 x 1040 14, 27 us (108).
bool many_rows(const LinearArgs& l) {
  return l.M > 128 && (pair_units(l) >= sm_count() / 2 * kPartUnits || l.M > 65535 * 128);
}

template <typename T>
void launch_pair(const LinearArgs& l, const Args& a, cudaStream_t s) {
  const CUtensorMap tx = codes_map(l.x, l.M, l.K, 128), tw = codes_map(l.w, l.N, l.K, 64);
  pair::Line line{};
  line.tiles_m = static_cast<int>((l.M + pair::BM - 1) / pair::BM);
  line.tiles = static_cast<int>(pair_tiles(l));
  line.units = pair_units(l);
  line.pairs = pairs_of(l);
  line.parts = l.workspace;
  line.done = l.counters;
  auto kern = pair::pair_kernel<T>;
  static PerDeviceOnce attr;
  attr([&] {
    B200AR_CUDA(
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(pair::kSmem)));
  });
  launch_pdl(kern, dim3(static_cast<unsigned>(2 * line.pairs)), dim3(pair::kThreads), pair::kSmem, s, 2, tx, tw, a,
             line);
}

template <typename T, int MP>
void dispatch_rows(const LinearArgs& l, const Args& a, cudaStream_t s) {
  // Cluster size: the most CTAs that two to an SM hold, with two K blocks each at least.
  const int64_t ctas = (l.N + 127) / 128 * ((l.M + MP - 1) / MP);
  int splits = 1;
  while (splits < 8 && ctas * splits * 2 <= 2 * sm_count() && a.kblocks >= splits * 4) splits *= 2;
  launch_rows<T, MP>(l, a, splits, s);
}

template <typename T>
void dispatch(const LinearArgs& l, const Args& a, cudaStream_t s) {
  if (many_rows(l)) return launch_pair<T>(l, a, s);
  if (l.M <= 16) return dispatch_rows<T, 16>(l, a, s);
  if (l.M <= 32) return dispatch_rows<T, 32>(l, a, s);
  if (l.M <= 64) return dispatch_rows<T, 64>(l, a, s);
  dispatch_rows<T, 128>(l, a, s);
}

void check(const LinearArgs& l) {
  B200AR_CHECK(l.M >= 0 && l.M < (1ll << 30) && l.N > 0 && l.N < (1ll << 21) && l.K > 0 && l.K < (1ll << 30),
               "bad shape for linear_fp8");
  B200AR_CHECK(l.K % 16 == 0 && l.N % 8 == 0, "K must be a multiple of 16 and N of 8");
}

}  // namespace

namespace {

// Places of a call's scratch, in bytes: parts of cut tiles, their counters, codes and scales of x.
struct Layout {
  int64_t counters, zeros, codes, scales, bytes;
};
Layout layout(const LinearArgs& l) {
  const auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  Layout o{};
  if (many_rows(l)) {
    o.counters = up(pairs_of(l) * 4 * pair::kPartFloats * 4);
    o.zeros = 2 * pair_tiles(l);
  }
  o.codes = o.counters + up(o.zeros * 4);
  o.scales = o.codes;
  o.bytes = o.codes;
  if (l.raw) {
    o.scales += up(l.M * l.K);
    o.bytes = o.scales + (l.K + kBlock - 1) / kBlock * l.M * 4;
  }
  return o;
}

}  // namespace

bool linear_takes_pairs(int64_t M, int64_t N, int64_t K) {
  LinearArgs l{};
  l.M = M, l.N = N, l.K = K;
  check(l);
  return many_rows(l);
}

int64_t linear_scratch(const LinearArgs& l) {
  check(l);
  return l.M == 0 ? 0 : layout(l).bytes;
}

void linear(const LinearArgs& args, Type out, void* scratch, cudaStream_t s) {
  const TraceRange trace("b200ar::linear_fp8");
  LinearArgs l = args;
  check(l);
  if (l.M == 0) return;
  const Layout at = layout(l);
  uint8_t* mem = static_cast<uint8_t*>(scratch);
  l.workspace = reinterpret_cast<float*>(mem);
  l.counters = reinterpret_cast<unsigned*>(mem + at.counters);
  if (l.raw) {
    float* scales = reinterpret_cast<float*>(mem + at.scales);
    quantize(l.raw, l.ldx, mem + at.codes, scales, l.M, l.M, l.K, out, l.counters, at.zeros, s);
    l.x = mem + at.codes;
    l.sx = scales;
    l.lds = l.M;
  } else if (at.zeros) {
    B200AR_CUDA(cudaMemsetAsync(l.counters, 0, at.zeros * 4, s));
  }
  Args a{};
  a.sx = l.sx;
  a.sw = l.sw;
  a.out = l.out;
  a.lds = l.lds;
  a.ldo = l.ldo;
  a.M = static_cast<int>(l.M);
  a.N = static_cast<int>(l.N);
  a.kblocks = static_cast<int>((l.K + kBlock - 1) / kBlock);
  a.err = l.err;
  if (out == Type::kBf16)
    dispatch<__nv_bfloat16>(l, a, s);
  else
    dispatch<__half>(l, a, s);
}

}  // namespace fp8
}  // namespace b200ar
