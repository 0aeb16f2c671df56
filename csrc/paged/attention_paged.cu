// Attention of new tokens over a paged KV cache, on the 5th-generation tensor cores.
//
//   o[i] = sum_p w[i, p] v[p] / sum_p w[i, p],   w[i, p] = exp(scale q[i] . k[p])
//
// over the positions p that row i sees. The G query heads of a KV head share
// keys and values, so the rows of a product are (token, head) pairs: a block
// is 256 of them (schedule.cuh), and for each tile of 128 tokens
//
//   S [128 rows x 128 tokens] = Q K^T   (tcgen05.mma, Q and K in shared memory)
//   O [128 rows x d]         += P V     (tcgen05.mma, P in tensor memory)
//
// with P = exp2(scale log2(e) S - m) rounded to the type of V, m a running
// bound on the row's maximum and the sum of P kept in fp32.
//
//   warps 0-3, 4-7  softmax: group t owns S_t, P_t (in the columns of S_t) and
//                   O_t in tensor memory; a thread owns one row
//   warps 8, 11     TMA producers of K and of V
//   warp 9          TMEM allocation and MMA issue (one thread)
//   warp 10         walks the CTA's items and hands them to the others; clears positions of V (see below)
//
// Steps alternate between the two groups, so that one's products run during
// the other's softmax. What the groups work on depends on the block's rows:
//   over 128   group t has rows 128 t .. 128 t + 127; both use every tile
//   33 to 128  both have the same rows; group t takes the tiles t, t + 2, ...
//   up to 32   as before, and the 32 rows are held four times: warp w of a
//              group takes the tokens 32 w .. 32 w + 31 of a tile. The products
//              cost the same, the softmax of a tile a quarter
// and the states of a row (its maximum, sum and O) are joined at the end. Calls
// with one token for each sequence and at most 32 heads to a KV head have only
// the last kind: they run an instance of the kernel without the others' code
// (kTokens), which a short call fetches faster.
//
// P takes the place of S; S of a group's next step is issued behind its P V, in
// which order the tensor core works. (Measured: steps of 64 tokens with two
// buffers for S, which hide the products of the step before, take 873 us where
// whole tiles take 723, for 4096 tokens over 4096 with 64 heads of 128: S of 64
// columns takes the tensor core nearly as long as of 128. With heads of 64: 764
// and 714 us.) O is rescaled only when the row's maximum has grown by 2^8 or more
// over the bound m in use (2^6 for fp16, whose P has a factor 2^8 to keep small
// weights out of the subnormals; bf16's has 2^-8, so that P is at most 1), after
// the product before is done: P stays in the type's range, and numerator and
// denominator have the same factor.
//
// What bounds it: with many rows the way of a tile through a group, S, maximum,
// exponentials, P, product, which the other group does not cover. By count the
// exponentials (8 clocks for a warp's 32) take the time of both products, and for
// 4096 tokens over 8192 the exponential unit is in use for 55 % of the active
// cycles, the tensor core for 54 % and the issue slots for 35 %: none is full.
// With single tokens over long caches it is the stream of K and V (64 tokens over
// 1 to 4095 with 8 KV heads of 128: 100 us for 0.5 GB), and over short ones the way
// of a block through the pipeline, about 3 us.
//
// Pages are read by TMA boxes of the largest power of two of tokens (8 to
// 128) that divides the page size. Runs that no row sees are not looked up:
// their boxes lie outside the pool and read as zeros. What a row must not see is
// masked in S; in V, where a zero weight does not hide a NaN,
//   - positions that no row of the block sees (behind the last row's, before the first row's window) become zeros;
//   - of those that some rows see and others do not (at most 255 at either end of the block's range, in its first
//     and last tiles) the infinities and NaN become zeros, and their outputs are settled at the end, row by row;
//   - what all rows see stays, so it reaches only rows that it belongs to.
// A row with a NaN score is NaN. Other outputs that are not finite, and rows of a block whose V had to be cleared,
// follow from the values of V alone: a column is inf, -inf or NaN as the sum of what the row sees in it that is not
// finite (settle, settle_columns). That reads V once more for each warp with such rows, whatever their number: one NaN
// that 256 tokens over 4096 with 8 heads of 128 see makes 0.14 ms of 0.06. (Rows computed again one by one took 13.)
//
// Every wait is bounded: on expiry the error word is set and all roles run
// down without waiting.
#include <cuda.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "../common/check.h"
#include "../common/pdl.h"
#include "../common/trace.h"
#include "../gemm/tcgen05.cuh"
#include "schedule.cuh"

namespace b200ar {
namespace paged {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// 1 / l for a row's sum of weights. A sum of zero is a row that sees nothing, whose output is zero (the factor 0
// stands for that), or one whose scores are all -inf: NaN, as exp(-inf - max) is.
__device__ __forceinline__ float inverse(float l, bool sees) {
  return l != 0.f ? 1.f / l : (sees ? __int_as_float(0x7fffffff) : 0.f);
}

// ------------------------------------------------------------------ infinities and NaN
// A pair of 16-bit values without the ones that are not finite.
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  return w & ~__vcmpeq2(w & kExp, kExp);
}

// The largest absolute values of both halves, as bit patterns.
__device__ __forceinline__ uint32_t largest2(const uint4& w) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(w.x & kAbs, w.y & kAbs), __vmaxu2(w.z & kAbs, w.w & kAbs));
}

// Settles the columns that are not finite in rows whose weights are numbers (bits of `rows`, from row `first` of the
// block on; the calling warp sees their stored outputs). Every weight counts as positive, as in the formula: a column
// in which a row sees +inf, -inf or both, or a NaN, is that, -that or NaN. `all`: look at what every row sees, too;
// `some`: at what not every row sees.
template <typename T, int D>
__device__ __noinline__ void settle(const AttnArgs& a, const Item& it, int group, int first, unsigned rows, bool all,
                                    bool some) {
  constexpr int kPairs = D / 64;  // pairs of columns that a lane looks at
  constexpr unsigned kPlus = 1, kMinus = 2, kNan = 4;
  const int lane = threadIdx.x & 31;
  // Which of the three appear in this lane's columns at positions [from, to): three bits for each column.
  auto scan = [&](int from, int to) {
    unsigned seen = 0;
#pragma unroll 1
    for (int p = from; p < to;) {
      const int index = p / a.page_size, page = page_of(a.batch, it.s, index, a.num_pages);
      const int stop = min(to, (index + 1) * a.page_size);
      if (page >= 0) {
        const T* vp = static_cast<const T*>(a.v.base) + page * a.v.page + it.h * a.v.head + lane * 2;
#pragma unroll 1
        for (; p < stop; p += 8) {  // eight positions under way
          uint32_t w[8][kPairs];
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < kPairs; ++i)
              w[e][i] = p + e < stop ? *reinterpret_cast<const uint32_t*>(vp + (p + e - index * a.page_size) * a.v.tok +
                                                                          i * 64)
                                     : 0u;
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < kPairs; ++i)
              if (finite2<T>(w[e][i]) != w[e][i]) {
                const float2 v = to_float2<T>(w[e][i]);
                seen |= (v.x != v.x ? kNan : v.x == INFINITY ? kPlus : v.x == -INFINITY ? kMinus : 0u) << (6 * i);
                seen |= (v.y != v.y ? kNan : v.y == INFINITY ? kPlus : v.y == -INFINITY ? kMinus : 0u) << (6 * i + 3);
              }
        }
      }
      p = stop;
    }
    return seen;
  };
  const bool common = it.see0 < it.hide0;
  const unsigned every = all && common ? scan(it.see0, it.hide0) : 0u;
#pragma unroll 1
  for (; rows; rows &= rows - 1) {
    const int x = it.row0 + first + __ffs(rows) - 1, tok = x / group, pos = it.len - it.n + tok;
    unsigned seen = every;
    if (some) {
      const int lo = a.window > 0 ? max(it.begin, pos - a.window + 1) : it.begin, hi = a.causal ? pos + 1 : it.end;
      seen |= scan(lo, min(hi, common ? it.see0 : it.end));
      if (common) seen |= scan(it.hide0, min(hi, it.end));
    }
    T* out = static_cast<T*>(a.out) + (it.q0 + tok) * a.o_tok + (it.h * group + x % group) * a.o_head + lane * 2;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      auto value = [&](unsigned bits, float old) {
        return bits == 0 ? old : bits == kPlus ? INFINITY : bits == kMinus ? -INFINITY : __int_as_float(0x7fffffff);
      };
      uint32_t* at = reinterpret_cast<uint32_t*>(out + i * 64);
      const float2 old = to_float2<T>(*reinterpret_cast<volatile uint32_t*>(at));
      const unsigned x3 = seen >> (6 * i) & 7u, y3 = seen >> (6 * i + 3) & 7u;
      if (x3 | y3) *at = pack2<T>(value(x3, old.x), value(y3, old.y));
    }
  }
}

// ------------------------------------------------------------------ workspace
// CTA c leaves at most two parts of blocks that others work on too: its first
// and its last item (slots 2 c and 2 c + 1).
struct PartDesc {
  int s, h, b;
  short rows, cleared;    // cleared: of the item
  int t0, t1, tiles, q0;  // q0 < 0: not used
};

struct Workspace {
  PartDesc* desc;  // [2 CTAs]
  float* ml;       // [2 CTAs][row_cap][2]: bound on the maximum (log2 units), sum
  float* acc;      // [2 CTAs][d / 4][row_cap][4]
  int row_cap;
};

// ------------------------------------------------------------------ shared memory
template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;                    // 128-byte wide halves of a row
  static constexpr uint32_t kGroupBytes = kHalves * 1024;   // 8 tokens of K or V: [half][token][128 bytes]
  static constexpr uint32_t kHalfBytes = 128 * 128;         // 128 rows x 128 bytes
  static constexpr uint32_t kTileBytes = kHalves * kHalfBytes;
  static constexpr int kSlots = D == 128 ? 5 : 8;           // ring of K and V tiles
  static constexpr uint32_t kQ = 0;                         // two tiles of queries
  static constexpr uint32_t kRing = 2 * kTileBytes;
  static constexpr uint32_t kMisc = kRing + kSlots * kTileBytes;
  static constexpr size_t kSmem = 1024 + kMisc + 1536;
};

constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;  // S_0, S_1 at columns 0 and 128 O_0, O_1 at 256 and 384

struct Barriers {
  uint64_t full[8], empty[8];  // ring slots
  uint64_t qready[2];          // queries of tile t written
  uint64_t sfull[2];           // S of group t computed
  uint64_t pready[2];          // P written in its place, O_t rescaled if need be
  uint64_t odone[2];           // a product P V of group t done
  uint64_t ofull[2];           // the last one in a block
  uint64_t gsync, gfree;       // the eight softmax warps: states written; their memory read
  uint64_t ifull[4], iempty[4];  // ring of items
  uint64_t vcut[8], vclear[8];   // ring slots: V with positions to clear is on its way; is cleared
  uint64_t drained;
};
constexpr int kItems = 4;
struct Misc {
  Barriers bar;
  Item item[kItems];  // rows == 0: no more
  int64_t red[33];
  Part part;
  uint32_t tmem;
  int err;
  unsigned bad;      // rows of a 32-row block with outputs that are not finite, but for those of NaN weights
  float inv[32];     // factors of such a block's rows (inverse())
  int last[2][8];    // last load of K and of V into each slot of the ring, or -1
};
static_assert(sizeof(Misc) <= 1536, "miscellaneous shared memory");

// exp2 of the arguments that a softmax makes: 0 below the normal numbers.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pack64(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(__float_as_uint(lo)), "r"(__float_as_uint(hi)));
  return r;
}
__device__ __forceinline__ float2 unpack64(uint64_t v) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <typename T>
struct Weights;
template <>
struct Weights<__nv_bfloat16> {
  // No weight above 1: sums of weights times large values stay in range where those with the row's maximum do.
  static constexpr float kBias = -8.f, kSlack = 8.f;
  static constexpr uint32_t kFormat = 1, kInf = 0x7f80u;
};
template <>
struct Weights<__half> {
  static constexpr float kBias = 8.f, kSlack = 6.f;
  static constexpr uint32_t kFormat = 0, kInf = 0x7c00u;
};

// Products with shared-memory descriptors given by their low words: the high word of a layout is a constant, and
// the issuing thread, whose pace bounds the kernel otherwise, has one register to hand over instead of two.
constexpr uint32_t desc_high(uint32_t stride_bytes) { return (stride_bytes >> 4) | 1u << 14 | 2u << 29; }
__device__ __forceinline__ uint32_t desc_low(const void* tile, uint32_t lead_bytes) {
  return ((sm100::smem_u32(tile) >> 4) & 0x3fffu) | (lead_bytes >> 4) << 16;
}
template <uint32_t kHighA, uint32_t kHighB, uint32_t kIdesc>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %6, p;\n\t}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(static_cast<uint32_t>(accumulate)), "n"(kHighA), "n"(kHighB), "n"(kIdesc)
      : "memory");
}
template <uint32_t kHighB, uint32_t kIdesc>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_low, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %5, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_low), "r"(static_cast<uint32_t>(accumulate)), "n"(kHighB), "n"(kIdesc)
      : "memory");
}

// Instruction descriptor: D fp32, A and B of type T, shape 128 x n; B MN-major if `bt`.
template <typename T>
constexpr uint32_t idesc(int n, bool bt) {
  return (1u << 4) | (Weights<T>::kFormat << 7) | (Weights<T>::kFormat << 10) | (bt ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (128u >> 4 << 24);
}

// Steps of an item: step k belongs to group k & 1 and takes a tile.
template <bool kTokens>
struct Steps {
  bool wide;  // over 128 rows: both groups use every tile, else every other one
  int nt;     // tiles
  __device__ __forceinline__ Steps(const Item& it) : wide(!kTokens && it.rows > 128), nt(it.t1 - it.t0) {}
  __device__ __forceinline__ int count() const { return wide ? 2 * nt : nt; }
  __device__ __forceinline__ int tile(int k) const { return wide ? k / 2 : k; }
  // Place of tile j's K and V in the ring's order of loads: the order of first use.
  __device__ __forceinline__ int k_at(int j) const { return wide ? 2 * j : (j == 0 ? 0 : 2 * j - 1); }
  __device__ __forceinline__ int v_at(int j) const { return wide ? 2 * j + 1 : (j + 1 < nt ? 2 * j + 2 : 2 * nt - 1); }
};

// Clears the tile of V from position c0 on, by one warp: zeros where no row of the block sees the position, and in
// place of what is not finite where only some do, which is marked. (A call, so that this rare work lies outside of
// the kernel's loops: inlined, it made them 3 to 5 % slower.)
template <typename T, int kHalves, uint32_t kGroupBytes>
__device__ __noinline__ void clear_hidden(uint8_t* tile, Item& it, int c0) {
  const int lane = threadIdx.x & 31, see0 = it.see0, hide0 = it.hide0, begin = it.begin, end = it.end;
  uint8_t* v = tile + (lane & 7) * 16;  // eight lanes on 128 bytes of a row
  uint32_t top = 0;
#pragma unroll 2
  for (int r = lane >> 3; r < kTile; r += 4) {
    const int p = c0 + r;
    const bool none = p >= end || p < begin;
    if (!none && p < hide0 && p >= see0) continue;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      uint4* w = reinterpret_cast<uint4*>(v + (r >> 3) * kGroupBytes + h * 1024 + (r & 7) * 128);
      if (none)
        *w = make_uint4(0u, 0u, 0u, 0u);
      else
        top = __vmaxu2(top, largest2(*w));
    }
  }
  if (!__any_sync(0xffffffffu, max(top >> 16, top & 0xffffu) >= Weights<T>::kInf)) return;
  if (lane == 0) *static_cast<volatile int*>(&it.cleared) = 1;
#pragma unroll 1
  for (int r = lane >> 3; r < kTile; r += 4) {
    if (c0 + r < hide0 && c0 + r >= see0) continue;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      uint4* w = reinterpret_cast<uint4*>(v + (r >> 3) * kGroupBytes + h * 1024 + (r & 7) * 128);
      const uint4 x = *w;
      *w = make_uint4(finite2<T>(x.x), finite2<T>(x.y), finite2<T>(x.z), finite2<T>(x.w));
    }
  }
}

template <typename T, int D, bool kTokens>
__global__ void __launch_bounds__(kThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ AttnArgs a, const Workspace ws, int group, int box, float q_sign,
                     float scale_log2) {
  using C = Cfg<D>;
  constexpr int kSlots = C::kSlots;
  extern __shared__ __align__(1024) uint8_t attention_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(attention_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + C::kRing;
  Misc& misc = *reinterpret_cast<Misc*>(smem + C::kMisc);
  Barriers& bar = misc.bar;
  volatile int* s_err = &misc.err;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  PartDesc* desc = ws.desc + 2 * blockIdx.x;  // thread 0 writes them
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      sm100::mbar_init(&bar.full[i], 1);
      sm100::mbar_init(&bar.empty[i], 1);
      sm100::mbar_init(&bar.vcut[i], 1);
      sm100::mbar_init(&bar.vclear[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&bar.qready[i], 4);
      sm100::mbar_init(&bar.sfull[i], 1);
      sm100::mbar_init(&bar.pready[i], 4);
      sm100::mbar_init(&bar.odone[i], 1);
      sm100::mbar_init(&bar.ofull[i], 1);
    }
    for (int i = 0; i < kItems; ++i) {
      sm100::mbar_init(&bar.ifull[i], 1);
      sm100::mbar_init(&bar.iempty[i], 11);  // two producers, MMA issue, eight softmax warps
    }
    sm100::mbar_init(&bar.gsync, 8);
    sm100::mbar_init(&bar.gfree, 8);
    sm100::mbar_init(&bar.drained, 1);
    misc.err = 0;
    misc.bad = 0;
    for (int i = 0; i < 8; ++i) misc.last[0][i] = misc.last[1][i] = -1;
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&tk);
    sm100::prefetch_tmap(&tv);
  }
  if (warp == 9) {
    sm100::tmem_alloc(&misc.tmem, kTmemCols);
    sm100::tmem_relinquish();
  }
  pdl_wait();  // lengths, offsets, pages, queries and the cache may come from the kernel before
  if (threadIdx.x == 0) desc[0].q0 = desc[1].q0 = -1;
  find_part<kThreads, kTokens>(a, group, misc.red, &misc.part);
  pdl_trigger();  // after a barrier: this CTA holds its tensor memory
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = misc.tmem;
  // A wait that ends early once any role of the CTA has given up. A failed try is suspended for a microsecond or
  // two, so the limit is seconds (and a tenth of one if it never were). Small on purpose: it is inlined at many
  // places, and code that does not stay in the instruction cache is what a short call spends its time on.
  auto wait = [&](uint64_t* b, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; !sm100::mbar_try_wait(b, parity); ++i)
      if ((i & 63) == 63 && (*s_err || i > (1 << 22))) {
        *s_err = 1;
        break;
      }
  };
  // 168 registers a thread at launch: 72 for the last warpgroup and 216 for the two of the softmax.
  if (warp >= 8) {
    if constexpr (!kTokens) sm100::reg_give<72>();
    if (warp == 10) {
      // ------------------------------------------------------------ items, and V where rows differ in what they see
      Walk<kTokens> walk;
      if (lane == 0) walk.start(a, group, misc.part);
      bool more = lane == 0;
      unsigned base = 0;   // loads of the items before, K and V
      uint32_t phase = 0;  // parity of the next vcut[slot] (bit slot)
#pragma unroll 1
      for (unsigned i = 0;; ++i) {
        if (more) {
          Item it;
          more = walk.next(a, group, it) && !*s_err;
          if (!more) it.rows = 0;
          wait(&bar.iempty[i % kItems], ((i / kItems) & 1u) ^ 1u);
          misc.item[i % kItems] = it;
          sm100::mbar_arrive(&bar.ifull[i % kItems]);
        }
        if constexpr (kTokens) {
          if (!__any_sync(0xffffffffu, more)) break;
        } else {
          // Then the item two before that one: the ring's place was free as soon as this item's turn came.
          __syncwarp();
          if (i < 2) continue;
          Item& it = misc.item[(i - 2) % kItems];
          if (__any_sync(0xffffffffu, *s_err || it.rows == 0)) break;
          const Steps<kTokens> st(it);
          const int first = (it.tile0 + it.t0) * kTile;
#pragma unroll 1
          for (int j = 0; j < st.nt; ++j) {
            if (!it.cut(first + j * kTile)) continue;
            const unsigned n = base + st.v_at(j), sl = n % kSlots;
            wait(&bar.vcut[sl], phase >> sl & 1u);
            phase ^= 1u << sl;
            wait(&bar.full[sl], (n / kSlots) & 1u);
            clear_hidden<T, C::kHalves, C::kGroupBytes>(ring + sl * C::kTileBytes, it, first + j * kTile);
            sm100::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&bar.vclear[sl]);
          }
          base += 2 * st.nt;
        }
      }
    } else if (warp == 8 || warp == 11) {
      // ------------------------------------------------------------ TMA producers
      const bool is_v = warp == 11;
      const CUtensorMap* map = is_v ? &tv : &tk;
      const int boxes = kTile / box;  // page runs of a tile
      const int ahead = 32 / boxes;   // tiles whose runs the warp's lanes look up together
      const int unit = is_v ? a.unit_v : a.unit_k;  // of 64 values from head to head
      unsigned base = 0;              // loads of the items before, K and V
#pragma unroll 1
      for (unsigned item = 0;; ++item) {
        wait(&bar.ifull[item % kItems], (item / kItems) & 1u);
        const Item& it = misc.item[item % kItems];
        if (__any_sync(0xffffffffu, *s_err || it.rows == 0)) break;
        const Steps<kTokens> st(it);
        const int first = (it.tile0 + it.t0) * kTile, nt = st.nt, s = it.s, begin = it.begin, end = it.end;
        const int head = it.h * unit;
        if (it.over && lane == 0) atomicExch(a.err, kErrPage);
        // Page and token of this lane's run in the tiles [ahead g, ahead (g + 1)). Runs that no row sees lie
        // outside the pool: zeros.
        auto look_up = [&](int g) {
          const int j = g * ahead + lane / boxes, pos = first + j * kTile + lane % boxes * box;
          int2 at = make_int2(a.num_pages, 0);
          if (j < nt && pos + box > begin && pos < end) {
            at.x = page_of(a.batch, s, pos / a.page_size, a.num_pages);
            at.y = pos % a.page_size / 8;
            if (at.x < 0) {
              atomicExch(a.err, kErrPage);
              at.x = a.num_pages;
            }
          }
          return at;
        };
        int2 cur = make_int2(0, 0), next = look_up(0);
#pragma unroll 1
        for (int j = 0; j < nt; ++j) {
          if (j % ahead == 0) {
            cur = next;
            next = look_up(j / ahead + 1);
          }
          const unsigned n = base + (is_v ? st.v_at(j) : st.k_at(j)), sl = n % kSlots, ph = (n / kSlots) & 1u;
          wait(&bar.empty[sl], ph ^ 1u);
          if (__any_sync(0xffffffffu, *s_err)) break;
          if (lane == 0) sm100::mbar_arrive_expect_tx(&bar.full[sl], C::kTileBytes);
          uint8_t* dst = ring + sl * C::kTileBytes;
#pragma unroll 1
          for (int run = 0; run < boxes; ++run) {
            const int page = __shfl_sync(0xffffffffu, cur.x, j % ahead * boxes + run);
            const int tok8 = __shfl_sync(0xffffffffu, cur.y, j % ahead * boxes + run);
            if (lane == 0)
              sm100::tma_load_5d(dst + run * (box / 8) * C::kGroupBytes, map, &bar.full[sl], 0, 0, head, tok8, page);
          }
          if (lane == 0) misc.last[is_v][sl] = static_cast<int>(n);
          if constexpr (!kTokens)
            if (lane == 0 && is_v && it.cut(first + j * kTile)) sm100::mbar_arrive(&bar.vcut[sl]);
        }
        base += 2 * nt;
        if (lane == 0) sm100::mbar_arrive(&bar.iempty[item % kItems]);
      }
    } else {
      // ------------------------------------------------------------ MMA issue
      if (sm100::elect_one()) {
        constexpr uint32_t kHighQ = desc_high(1024), kHighKV = desc_high(C::kGroupBytes);
        unsigned base = 0;                // loads of the items before
        uint32_t qphase = 0, pphase = 0;  // parity of the next qready[tile] (bit tile), pready[t] (bit t)
        uint32_t cphase = 0;              // of the next vclear[slot]
        int qt = 0;                       // tile of the queries of an item of at most 128 rows
        bool narrow_before = false;
#pragma unroll 1
        for (unsigned item = 0;; ++item) {
          wait(&bar.ifull[item % kItems], (item / kItems) & 1u);
          const Item& it = misc.item[item % kItems];
          if (*s_err || it.rows == 0) break;
          const Steps<kTokens> st(it);
          // Positions before `low` and from `high` on, counted from the first tile, are cleared in V.
          const int first = (it.tile0 + it.t0) * kTile, low = it.see0 - first, high = it.hide0 - first;
          sm100::mbar_arrive(&bar.iempty[item % kItems]);
          const bool wide = st.wide;
          const int steps = st.count();
          qt = !wide && narrow_before ? qt ^ 1 : 0;
          narrow_before = !wide;
          wait(&bar.qready[qt], qphase >> qt & 1u);
          qphase ^= 1u << qt;
          if (wide) {
            wait(&bar.qready[1], qphase >> 1 & 1u);
            qphase ^= 2u;
          }
          const uint32_t q_low = desc_low(smem + C::kQ, 16), ring_low = desc_low(ring, 0);
          // S of step k. With `wide` both groups use a tile: the first waits for it and the second frees it.
          auto scores = [&](int k) {
            const int t = k & 1;
            const unsigned n = base + st.k_at(st.tile(k)), sl = n % kSlots;
            if (!wide || t == 0) wait(&bar.full[sl], (n / kSlots) & 1u);
            sm100::tc_fence_after();
            const uint32_t q = q_low + (wide ? t : qt) * (C::kTileBytes >> 4);
            const uint32_t kk = ring_low + sl * (C::kTileBytes >> 4) + (1u << 16);  // leading byte offset, unused
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
              mma_ss<kHighQ, kHighKV, idesc<T>(kTile, false)>(
                  tmem + t * 128, q + (i >> 2) * (C::kHalfBytes >> 4) + 2 * (i & 3),
                  kk + (i >> 2) * (1024 >> 4) + 2 * (i & 3), i > 0);
            sm100::mma_commit(&bar.sfull[t]);
            if (!wide || t == 1) sm100::mma_commit(&bar.empty[sl]);
          };
#pragma unroll 1
          for (int k = 0; k < 2 && k < steps; ++k) scores(k);
#pragma unroll 1
          for (int k = 0; k < steps && !*s_err; ++k) {
            const int t = k & 1;
            const unsigned n = base + st.v_at(st.tile(k)), sl = n % kSlots;
            if (!wide || t == 0) {
              const int c = st.tile(k) * kTile;
              const bool cut = !kTokens && (c < low || c + kTile > high);  // Item::cut()
              wait(cut ? &bar.vclear[sl] : &bar.full[sl], cut ? cphase >> sl & 1u : (n / kSlots) & 1u);
              if (cut) cphase ^= 1u << sl;
            }
            // Leading byte offset: to the second half.
            const uint32_t v = ring_low + sl * (C::kTileBytes >> 4) + ((1024u >> 4) << 16);
            wait(&bar.pready[t], pphase >> t & 1u);
            pphase ^= 1u << t;
            sm100::tc_fence_after();
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)  // 16 tokens: two groups further in V, 8 columns in P
              mma_ts<kHighKV, idesc<T>(D, true)>(tmem + kColO + t * 128, tmem + t * 128 + i * 8,
                                                 v + i * (2 * C::kGroupBytes >> 4), k > 1 || i > 0);
            sm100::mma_commit(&bar.odone[t]);
            if (!wide || t == 1) sm100::mma_commit(&bar.empty[sl]);
            if (k + 2 < steps)
              scores(k + 2);
            else
              sm100::mma_commit(&bar.ofull[t]);
          }
          base += 2 * st.nt;
        }
        // Tensor memory is freed only after every product is done.
        sm100::mma_commit(&bar.drained);
        if (!sm100::mbar_wait(&bar.drained, 0)) *s_err = 1;
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax
    if constexpr (!kTokens) sm100::reg_take<216>();
    const int t = warp >> 2, w4 = warp & 3;
    const int row = w4 * 32 + lane;  // row of the group's tile
    const uint32_t lanes = static_cast<uint32_t>(w4 * 32) << 16;
    const uint32_t tS = tmem + lanes + t * 128, tO = tmem + lanes + kColO + t * 128;
    unsigned no = 0, nb = 0, ng = 0, nf = 0, base = 0;  // products P V, blocks, joins, frees and loads so far
    bool q_loaded = false, narrow_before = false;
    int qt = 0;  // tile of the queries of an item of at most 128 rows
    // All softmax warps (not a barrier that a warp which gave up would leave the others at).
    auto group_sync = [&] {
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&bar.gsync);
      wait(&bar.gsync, ng++ & 1u);
    };
    auto more = [&](unsigned i) {
      wait(&bar.ifull[i % kItems], (i / kItems) & 1u);
      return !__any_sync(0xffffffffu, *s_err || misc.item[i % kItems].rows == 0);
    };

    // Hands this warp's part of tensor memory to the MMA issue.
    auto arrive = [&](uint64_t* b) {
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(b);
    };
    // Writes the queries of an item into a tile: those of this group's 128 rows, or all of an item of at most 128.
    // D / 8 lanes read a row, so that a load touches whole lines.
    auto load_q = [&](const Item& i, int tile) {
      constexpr int kLanes = D / 8, kRows = 32 / kLanes;
      const int chunk = lane % kLanes;
      const int first = !kTokens && i.rows > 128 ? t * 128 + w4 * 32 : (kTokens || i.rows <= 32 ? 0 : w4 * 32);
      uint8_t* dst = smem + C::kQ + tile * C::kTileBytes + (chunk >> 3) * C::kHalfBytes + w4 * 32 * 128;
      int r = first + lane / kLanes;
      int tok = (i.row0 + r) / group, g = (i.row0 + r) % group;
      const T* q = static_cast<const T*>(a.q) + i.q0 * a.q_tok + i.h * group * a.q_head + chunk * 8;
      const int rows = i.rows;
      // Four loads under way; a short loop, since code that runs once per block is fetched anew each time.
#pragma unroll 1
      for (int j = 0; j < kLanes; j += 4) {
        uint4 v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = make_uint4(0u, 0u, 0u, 0u);
          if (r < rows) v[e] = __ldg(reinterpret_cast<const uint4*>(q + tok * a.q_tok + g * a.q_head));
          r += kRows;
#pragma unroll 1
          for (g += kRows; g >= group; g -= group) ++tok;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (q_sign != 1.f) {  // a negative or zero scale moves into the queries
            uint32_t* u = reinterpret_cast<uint32_t*>(&v[e]);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float2 f = to_float2<T>(u[x]);
              u[x] = pack2<T>(f.x * q_sign, f.y * q_sign);
            }
          }
          const int lr = (j + e) * kRows + lane / kLanes;
          *reinterpret_cast<uint4*>(dst + lr * 128 + (((chunk & 7) ^ (lr & 7)) << 4)) = v[e];
        }
      }
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&bar.qready[tile]);
    };

#pragma unroll 1
    for (unsigned item = 0; more(item); ++item) {
      Item& it = misc.item[item % kItems];
      const Steps<kTokens> st(it);
      const bool wide = st.wide, quad = kTokens || it.rows <= 32;
      // The queries of a narrow item alternate between the tiles, so that those of the next are loaded now; the
      // item's own tile takes the joining of its states at the end.
      if (narrow_before) wait(&bar.gfree, nf++ & 1u);  // the memory of the item before is read
      qt = !wide && narrow_before ? qt ^ 1 : 0;
      narrow_before = !wide;
      if (!q_loaded && (wide || t == 1)) load_q(it, wide ? t : qt);
      const bool next_narrow = !wide && more(item + 1) && misc.item[(item + 1) % kItems].rows <= 128;
      if (next_narrow && t == 1) load_q(misc.item[(item + 1) % kItems], qt ^ 1);
      q_loaded = next_narrow;
      // This thread's row of the block and what it sees.
      const int r = wide ? t * 128 + row : (quad ? lane : row);
      const bool valid = r < it.rows;
      const int rr = it.row0 + min(r, it.rows - 1);
      const int pos = it.len - it.n + rr / group;
      const int hi = valid ? (a.causal ? pos + 1 : it.len) : 0x7fffffff;  // rows that are not there hide nothing
      const int lo = a.window > 0 && valid ? pos - a.window + 1 : 0;
      const bool idle = __all_sync(0xffffffffu, !valid);
      const int hi_all = __reduce_min_sync(0xffffffffu, hi), lo_all = __reduce_max_sync(0xffffffffu, lo);
      const int first_pos = (it.tile0 + it.t0) * kTile, see0 = it.see0, hide0 = it.hide0;
      float m = -INFINITY, l = 0.f;  // bound on the maximum, in units of S; sum of P
      const int steps = st.count();
      int mine = 0;  // steps of this group
#pragma unroll 1
      for (int k = t; k < steps; k += 2, ++mine, ++no) {
        const int j = st.tile(k), c0 = first_pos + j * kTile;
        wait(&bar.sfull[t], no & 1u);
        sm100::tc_fence_after();
        // Single tokens, whose rows all see the same: the rest becomes zeros in V here, since zero times NaN is NaN.
        // (After S of the step: what the slot of V held before is consumed or still waited for by this load.)
        if constexpr (kTokens)
          if (c0 + kTile > hide0 || c0 < see0) {
            const unsigned at = base + st.v_at(j);
            wait(&bar.full[at % kSlots], (at / kSlots) & 1u);
            if (c0 + row >= hide0 || c0 + row < see0) {
              uint8_t* vt = ring + (at % kSlots) * C::kTileBytes + (row >> 3) * C::kGroupBytes + (row & 7) * 128;
              // From a part of its own on for each of eight rows: their banks differ.
#pragma unroll
              for (int c = 0; c < 8 * C::kHalves; ++c)
                *reinterpret_cast<uint4*>(vt + (c >> 3) * 1024 + ((c + row) & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            sm100::fence_proxy_async_smem();
          }
        if (!idle) {
          // Columns of this thread: all, or the warp's quarter.
          auto softmax = [&](auto cols_tag) {
            constexpr int kCols = decltype(cols_tag)::value;
            const int first = kCols == kTile ? 0 : w4 * kCols;
            uint32_t x[kCols];
#pragma unroll
            for (int c = 0; c < kCols; c += 32) sm100::tmem_ld_32x32b_x32(tS + first + c, x + c);
            sm100::tmem_ld_wait();
            // Hidden columns become -inf, in the tiles where a row of the warp has some.
            if (kCols < kTile || c0 + kTile > hi_all) {
              const int to = hi - c0 - first;
#pragma unroll
              for (int c = 0; c < kCols; ++c) x[c] = c < to ? x[c] : 0xff800000u;
            }
            if (c0 < lo_all) {
              const int from = lo - c0 - first;
#pragma unroll
              for (int c = 0; c < kCols; ++c) x[c] = c >= from ? x[c] : 0xff800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kCols; c += 4)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(x[c + e]));
            const float top = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
            // -inf minus -inf is NaN, which is not above the slack: such a row keeps its bound.
            if (__any_sync(0xffffffffu, (top - m) * scale_log2 > Weights<T>::kSlack)) {
              const float f = m == -INFINITY ? 0.f : fast_exp2((m - top) * scale_log2);
              m = top;
              l *= f;
              if (mine > 0) {
                wait(&bar.odone[t], (no - 1) & 1u);  // the product of the step before; those before it are done
                sm100::tc_fence_after();
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                  uint32_t o[32];
                  sm100::tmem_ld_32x32b_x32(tO + c, o);
                  sm100::tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                  sm100::tmem_st_32x32b_x32(tO + c, o);
                }
                sm100::tmem_st_wait();
              }
            }
            const float shift = m == -INFINITY ? 0.f : Weights<T>::kBias - m * scale_log2;
            const uint64_t scale2 = pack64(scale_log2, scale_log2), shift2 = pack64(shift, shift);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < kCols; c += 32) {  // P of columns c .. goes where S was
              uint32_t p[32 / 2];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 y = unpack64(
                    fma2(pack64(__uint_as_float(x[c + e]), __uint_as_float(x[c + e + 1])), scale2, shift2));
                const float2 w = make_float2(fast_exp2(y.x), fast_exp2(y.y));
                sum[(e / 2) & 1] = add2(sum[(e / 2) & 1], pack64(w.x, w.y));
                p[e / 2] = pack2<T>(w.x, w.y);
              }
              sm100::tmem_st_32x32b_x16(tS + (first + c) / 2, p);
            }
            const float2 all = unpack64(add2(sum[0], sum[1]));
            l += all.x + all.y;
            if constexpr (kCols < kTile) {
              // The other quarters' tokens have no weight in this warp's rows.
              const uint32_t zero[16] = {};
#pragma unroll
              for (int q = 1; q < 4; ++q) sm100::tmem_st_32x32b_x16(tS + ((w4 + q) & 3) * 16, zero);
            }
            sm100::tmem_st_wait();
          };
          if constexpr (kTokens) {
            softmax(std::integral_constant<int, kTile / 4>{});
          } else if (quad) {
            softmax(std::integral_constant<int, kTile / 4>{});
          } else {
            softmax(std::integral_constant<int, kTile>{});
          }
        }
        arrive(&bar.pready[t]);
      }
      base += 2 * st.nt;

      // ---------------------------------------------------------- end of the block's part
      if (wide && more(item + 1)) {  // this group's last S is done: its queries are free
        const Item& next = misc.item[(item + 1) % kItems];
        if (next.rows > 128 || t == 0) load_q(next, t);
        q_loaded = true;
      }
      if (mine > 0) {
        wait(&bar.ofull[t], nb++ & 1u);
        sm100::tc_fence_after();
      }
      const bool whole = it.whole();
      // The first item of a CTA may continue a block, the last may leave one; one that does both is the first.
      const int which = it.t0 > 0 ? 0 : 1, slot = 2 * blockIdx.x + which;
      float* acc = ws.acc + static_cast<int64_t>(slot) * ws.row_cap * D;
      float* ml = ws.ml + static_cast<int64_t>(slot) * ws.row_cap * 2;
      auto cleared = [&] { return *static_cast<volatile int*>(&it.cleared) != 0; };
      auto describe = [&] {
        if (!whole && threadIdx.x == 0)
          desc[which] =
              PartDesc{it.s, it.h, it.b, static_cast<short>(it.rows), cleared(), it.t0, it.t1, it.tiles, it.q0};
      };
      if (wide) describe();
      auto out_of = [&](int r2) {
        const int x = it.row0 + r2;
        return static_cast<T*>(a.out) + (it.q0 + x / group) * a.o_tok + (it.h * group + x % group) * a.o_head;
      };
      // Stores 32 columns of each of the warp's rows. As fp32 to the workspace: float4 c of row r at place
      // c row_cap + r, so that lanes write side by side. Or rounded with the factor inv: four lanes exchange their
      // 16-byte parts, so that each store writes 64 bytes of a row.
      const int64_t my_out = out_of(min(r, it.rows - 1)) - static_cast<T*>(a.out);
      auto store32 = [&](int c, const float* o, float inv, float& odd) {
        if (!whole) {
          if (!valid) return;
          float4* dst = reinterpret_cast<float4*>(acc) + static_cast<int64_t>(c / 4) * ws.row_cap + r;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[static_cast<int64_t>(e) * ws.row_cap] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          return;
        }
        uint4 part[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] = inv == 0.f ? 0.f : o[8 * e + i] * inv;
            odd += y[i] * 0.f;  // NaN if any is not finite
          }
          part[e] = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
        }
        auto exchange = [&](uint4& keep_low, uint4& keep_high, int mask) {
          const bool high = lane & mask;
          const uint4 send = high ? keep_low : keep_high;
          uint4 got;
          got.x = __shfl_xor_sync(0xffffffffu, send.x, mask);
          got.y = __shfl_xor_sync(0xffffffffu, send.y, mask);
          got.z = __shfl_xor_sync(0xffffffffu, send.z, mask);
          got.w = __shfl_xor_sync(0xffffffffu, send.w, mask);
          if (high)
            keep_low = got;
          else
            keep_high = got;
        };
        exchange(part[0], part[1], 1);
        exchange(part[2], part[3], 1);
        exchange(part[0], part[2], 2);
        exchange(part[1], part[3], 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // part e of this lane: columns 8 (lane & 3) of row 4 (lane / 4) + e of the warp
          const int from = (lane & ~3) + e;
          const int64_t off = __shfl_sync(0xffffffffu, my_out, from);
          if (__shfl_sync(0xffffffffu, static_cast<int>(valid), from))
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + off + c + (lane & 3) * 8) = part[e];
        }
      };
      const float m2 = m == -INFINITY ? -INFINITY : m * scale_log2;

      // Rows computed by one thread each: 128 of a wide block by each group, or a narrow block's by group 0, which
      // adds the state of group 1: the same rows in the same lanes of tensor memory.
      auto finish_rows = [&](float mj, float lj, float f0, float f1, bool add) {
        const float inv = inverse(lj, valid && hi > max(lo, 0));
        float odd = 0.f;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          sm100::tmem_ld_32x32b_x32(tO + c, o);
          sm100::tmem_ld_wait();
          float y[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = __uint_as_float(o[e]) * f0;
          if (add) {
            sm100::tmem_ld_32x32b_x32(tO + 128 + c, o);
            sm100::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) y[e] += __uint_as_float(o[e]) * f1;
          }
          store32(c, y, inv, odd);
        }
        if (!whole && valid) *reinterpret_cast<float2*>(ml + r * 2) = make_float2(mj, lj);
        if (whole) {
          const bool some = cleared(), counts = valid && inv == inv && inv != 0.f;
          const unsigned not_finite = __ballot_sync(0xffffffffu, counts && odd != 0.f);
          const unsigned rows = __ballot_sync(0xffffffffu, counts && (odd != 0.f || some));
          __syncwarp();  // the rows are stored
          if (rows) settle<T, D>(a, it, group, (wide ? t * 128 : 0) + w4 * 32, rows, not_finite != 0, some);
        }
      };
      float* buf = reinterpret_cast<float*>(smem + C::kQ + qt * C::kTileBytes);
      float mj = m2, lj = l, f0 = 1.f, f1 = 0.f;  // the joined state of this thread's row and the factors of both
      bool joins = false;
      auto factor = [](float mm, float top) { return mm == -INFINITY ? 0.f : fast_exp2(mm - top); };
      // The states of all warps, through the memory of the item's queries: every S is done, since it was issued
      // before the last but one product with V, which each group with a step has waited for.
      float2* sml = reinterpret_cast<float2*>(buf);  // [8 warps][32 lanes]
      const bool two = st.nt > 1;                    // group 1 had a tile
      if (!wide) {
        if (mine > 0) sml[threadIdx.x] = make_float2(m2, l);
        sm100::tc_fence_before();
        group_sync();
        describe();
        if (!quad && two) {
          const float2 other = sml[128 + row];
          mj = fmaxf(m2, other.x), f0 = factor(m2, mj), f1 = factor(other.x, mj);
          lj = l * f0 + other.y * f1;
          joins = true;
        }
        sm100::tc_fence_after();
      }
      if (!quad) {
        if (!idle && (wide || t == 0)) finish_rows(mj, lj, f0, f1, joins);
      } else {
        // Lane = row. The two groups' states of a quarter lie in the same lanes: warp (t, w) adds them for the
        // half t of the columns and writes the quarter's sum; then a thread adds the quarters of four columns
        // of a row. A pass takes as many columns as fit; float4 c sits at place c ^ (r & 3).
        float* part = buf + 512;
        constexpr int kPart = C::kTileBytes / 4 - 512;
        mj = -INFINITY, lj = 0.f;
#pragma unroll 1
        for (int i = 0; i < (two ? 8 : 4); ++i) mj = fmaxf(mj, sml[i * 32 + lane].x);
#pragma unroll 1
        for (int i = 0; i < (two ? 8 : 4); ++i) lj += sml[i * 32 + lane].y * factor(sml[i * 32 + lane].x, mj);
        f0 = factor(sml[w4 * 32 + lane].x, mj);
        f1 = two ? factor(sml[(4 + w4) * 32 + lane].x, mj) : 0.f;
        if (warp == 0) {
          misc.inv[lane] = inverse(lj, valid && hi > max(lo, 0));
          if (!whole && valid) *reinterpret_cast<float2*>(ml + r * 2) = make_float2(mj, lj);
        }
        sm100::tc_fence_after();
        const uint32_t tO0 = tmem + lanes + kColO;
        int pass = D;
        while (4 * it.rows * pass > kPart) pass /= 2;  // 32 rows: 32 columns of 128, 16 of 64
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += pass) {
          if (c0) group_sync();
#pragma unroll 1
          for (int c = t * (pass / 2); c < (t + 1) * (pass / 2); c += 8) {
            uint32_t o0[8], o1[8];
            sm100::tmem_ld_32x32b_x8(tO0 + c0 + c, o0);
            if (two) sm100::tmem_ld_32x32b_x8(tO0 + 128 + c0 + c, o1);
            sm100::tmem_ld_wait();
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              // A factor of 0 drops no infinity: where a state holds one, seen or not, the column is settled below.
              y[e] = __uint_as_float(o0[e]) * f0;
              if (two) y[e] += __uint_as_float(o1[e]) * f1;
            }
            if (valid) {
              float4* dst = reinterpret_cast<float4*>(part + (w4 * it.rows + r) * pass);
              dst[(c / 4) ^ (r & 3)] = make_float4(y[0], y[1], y[2], y[3]);
              dst[(c / 4 + 1) ^ (r & 3)] = make_float4(y[4], y[5], y[6], y[7]);
            }
          }
          group_sync();
#pragma unroll 1
          for (int i = threadIdx.x; i < it.rows * (pass / 4); i += 256) {
            const int r2 = i / (pass / 4), c = i % (pass / 4);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float4 v = reinterpret_cast<const float4*>(part + (q * it.rows + r2) * pass)[c ^ (r2 & 3)];
              y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
            }
            if (whole) {
              const float inv = misc.inv[r2];
              if (inv == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
              y = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
              if (inv == inv && (y.x + y.y + y.z + y.w) * 0.f != 0.f) atomicOr(&misc.bad, 1u << r2);
              *reinterpret_cast<uint2*>(out_of(r2) + c0 + 4 * c) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
            } else {
              reinterpret_cast<float4*>(acc)[static_cast<int64_t>(c0 / 4 + c) * ws.row_cap + r2] = y;
            }
          }
        }
        if (whole) {
          group_sync();  // all rows are written
          const unsigned bad = *reinterpret_cast<volatile unsigned*>(&misc.bad);
          const bool some = cleared();
          if (bad != 0 || some) {
            const float inv = misc.inv[lane];
            const bool counts = valid && inv == inv && inv != 0.f;
            const unsigned rows = __ballot_sync(0xffffffffu, counts && (some || bad >> lane & 1u));
            const unsigned mine8 = rows & (0x01010101u << warp);  // every eighth row
            if (mine8) settle<T, D>(a, it, group, 0, mine8, (bad & mine8) != 0, some);
            group_sync();
            if (threadIdx.x == 0) misc.bad = 0;
          }
        }
      }
      if (!wide) arrive(&bar.gfree);
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&bar.iempty[item % kItems]);
    }
  }

  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, kTmemCols);
  }
  if (threadIdx.x == 0 && *s_err) {
    // Every load was waited for by its product, unless a role gave up: then it is here, so that none is in flight
    // when the CTA's memory goes.
#pragma unroll 1
    for (int sl = 0; sl < kSlots; ++sl) {
      const int n = max(misc.last[0][sl], misc.last[1][sl]);
      if (n >= 0) sm100::mbar_wait(&bar.full[sl], (n / kSlots) & 1);
    }
    atomicExch(a.err, kErrTimeout);
  }
}

// ------------------------------------------------------------------ merge
// Joins the parts of the blocks that a cut fell into. Grid (CTAs of the
// attention kernel, row groups); the CTA whose part starts such a block owns it.
// Parts are added in the order of the tiles, so results do not depend on timing.
// A lane has a row, a warp 16 columns of 32 rows; with fewer rows several lanes share a row's parts.
constexpr int kMaxParts = 1024;

// What settle() does, to 16 columns (from column c0 on) of a row for each lane; x: its row among the sequence's.
template <typename T>
__device__ __forceinline__ void settle_columns(const AttnArgs& a, const PartDesc& p, int group, int x, int c0,
                                               bool counts, float* o) {
  const int lane = threadIdx.x & 31;
  Item it;
  it.set_block(a, group, p.s, p.h, p.b, q_begin(a.batch, p.s + 1) - p.q0, __ldg(a.batch.kv_len + p.s), p.q0);
  unsigned plus = 0, minus = 0, nan = 0;  // columns
  auto look = [&](int pos) {
    const int page = page_of(a.batch, it.s, pos / a.page_size, a.num_pages);
    if (page < 0) return;
    const uint4* v = reinterpret_cast<const uint4*>(static_cast<const T*>(a.v.base) + page * a.v.page +
                                                    pos % a.page_size * a.v.tok + it.h * a.v.head + c0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 w4 = v[i];
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (finite2<T>(w[e]) == w[e]) continue;
        const float2 f = to_float2<T>(w[e]);
        const float two[2] = {f.x, f.y};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const unsigned bit = 1u << (8 * i + 2 * e + k);
          nan |= two[k] != two[k] ? bit : 0u;
          plus |= two[k] == INFINITY ? bit : 0u;
          minus |= two[k] == -INFINITY ? bit : 0u;
        }
      }
    }
  };
  const bool common = it.see0 < it.hide0;
  if (common) {
#pragma unroll 1
    for (int pos = it.see0 + lane; pos < it.hide0; pos += 32) look(pos);
    plus = __reduce_or_sync(0xffffffffu, plus);
    minus = __reduce_or_sync(0xffffffffu, minus);
    nan = __reduce_or_sync(0xffffffffu, nan);
  }
  const int at = it.len - it.n + x / group;
  const int lo = a.window > 0 ? max(it.begin, at - a.window + 1) : it.begin, hi = a.causal ? at + 1 : it.end;
#pragma unroll 1
  for (int pos = it.begin; pos < it.end; ++pos) {
    if (common && pos == it.see0) pos = it.hide0;
    if (pos >= lo && pos < min(hi, it.end)) look(pos);
  }
  if (counts)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const unsigned bits = (plus >> e & 1u) | (minus >> e & 1u) << 1 | (nan >> e & 1u) << 2;
      if (bits) o[e] = bits == 1u ? INFINITY : bits == 2u ? -INFINITY : __int_as_float(0x7fffffff);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(D * 2)
    merge_kernel(const __grid_constant__ AttnArgs a, const Workspace ws, int group, int ctas) {
  __shared__ int part[kMaxParts];
  __shared__ int parts;
  __shared__ int cleared;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const PartDesc first = ws.desc[2 * blockIdx.x + 1];
  if (first.q0 < 0 || first.t1 == first.tiles || static_cast<int>(blockIdx.y) * 32 >= first.rows) return;
  if (warp == 0) {
    // Continuations follow in the order of the CTAs; one that reaches the last tile is the last.
    int n = 1, some = first.cleared;
    if (lane == 0) part[0] = 2 * blockIdx.x + 1;
    for (int c0 = blockIdx.x + 1; c0 < ctas; c0 += 32) {
      const int c = c0 + lane;
      PartDesc d{};
      d.q0 = -1;
      if (c < ctas) d = ws.desc[2 * c];
      const bool on = d.q0 >= 0 && d.s == first.s && d.h == first.h && d.b == first.b;
      const unsigned who = __ballot_sync(0xffffffffu, on);
      if (on) part[n + __popc(who & ((1u << lane) - 1u))] = 2 * c;
      some |= __any_sync(0xffffffffu, on && d.cleared != 0);
      n += __popc(who);
      if (__any_sync(0xffffffffu, on && d.t1 == d.tiles)) break;
    }
    if (lane == 0) {
      parts = n;
      cleared = some;
    }
  }
  __syncthreads();
  const int n = parts;
  // Lanes to a row: 1, 2 or 4, `width` lanes apart.
  const int width = first.rows <= 8 ? 8 : (first.rows <= 16 ? 16 : 32);
  const int r = blockIdx.y * 32 + lane % width, rc = min(r, first.rows - 1);
  float m = -INFINITY, l = 0.f, o[16] = {};
  auto state = [&](int i) {
    return __ldcg(reinterpret_cast<const float2*>(ws.ml + (static_cast<int64_t>(part[i]) * ws.row_cap + rc) * 2));
  };
#pragma unroll 8
  for (int i = lane / width; i < n; i += 32 / width) m = fmaxf(m, state(i).x);
#pragma unroll 4
  for (int i = lane / width; i < n; i += 32 / width) {
    const float2 v = state(i);
    const float f = v.x == -INFINITY ? 0.f : fast_exp2(v.x - m);
    l += v.y * f;
    const float4* src = reinterpret_cast<const float4*>(ws.acc + static_cast<int64_t>(part[i]) * ws.row_cap * D) +
                        static_cast<int64_t>(warp * 4) * ws.row_cap + rc;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 x = __ldcg(src + static_cast<int64_t>(e) * ws.row_cap);
      o[4 * e] += x.x * f;  // a factor of 0 drops no infinity
      o[4 * e + 1] += x.y * f;
      o[4 * e + 2] += x.z * f;
      o[4 * e + 3] += x.w * f;
    }
  }
  for (int w = width; w < 32; w *= 2) {
    const float other = __shfl_xor_sync(0xffffffffu, m, w), top = fmaxf(m, other);
    const float f0 = m == -INFINITY ? 0.f : fast_exp2(m - top), f1 = other == -INFINITY ? 0.f : fast_exp2(other - top);
    m = top;
    l = l * f0 + __shfl_xor_sync(0xffffffffu, l, w) * f1;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = o[e] * f0 + __shfl_xor_sync(0xffffffffu, o[e], w) * f1;
  }
  const int x = first.b * kBlock + rc, tok = x / group, h = first.h * group + x % group;
  float inv = 1.f / l;
  if (l == 0.f) {  // (lengths are looked up only here and below: they would be waited for)
    const int len = __ldg(a.batch.kv_len + first.s), n_new = q_begin(a.batch, first.s + 1) - first.q0;
    inv = inverse(l, a.causal ? len - n_new + tok >= 0 : len > 0);  // a row's window holds its own position at least
  }
  const bool valid = r < first.rows && lane < width;
  float odd = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    o[e] = inv == 0.f ? 0.f : o[e] * inv;
    odd += o[e] * 0.f;
  }
  auto store = [&] {
    if (!valid) return;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (first.q0 + tok) * a.o_tok + h * a.o_head + warp * 16);
    dst[0] = make_uint4(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]), pack2<T>(o[4], o[5]), pack2<T>(o[6], o[7]));
    dst[1] = make_uint4(pack2<T>(o[8], o[9]), pack2<T>(o[10], o[11]), pack2<T>(o[12], o[13]), pack2<T>(o[14], o[15]));
  };
  store();
  const bool counts = valid && inv == inv && inv != 0.f;
  if (__any_sync(0xffffffffu, counts && (odd != 0.f || cleared != 0))) {
    settle_columns<T>(a, first, group, x, warp * 16, counts, o);
    store();
  }
}

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

// Map over a pool [pages, page_size, kv_heads, d] with its strides, in 64-value
// units: (64 values, 8 tokens, unit, tokens / 8, page). Units of 64 values from
// a token's first on hold all its heads, so a head is `unit` of them further
// and its halves are neighbours. A box is 64 values x 8 tokens x the halves x
// `box` / 8 x 1: runs of 8 tokens in the layout [half][token][128 bytes].
CUtensorMap pool_map(const Pool& p, int d, int hkv, int unit, int page_size, int num_pages, int box, Half type) {
  CUtensorMap m;
  const cuuint64_t dims[5] = {64, 8, static_cast<cuuint64_t>((hkv - 1) * static_cast<int64_t>(unit) + d / 64),
                              static_cast<cuuint64_t>(page_size / 8), static_cast<cuuint64_t>(num_pages)};
  // The stride of a dimension of one is never used; any valid one serves.
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(p.tok) * 2, 128, static_cast<cuuint64_t>(p.tok) * 16,
                                 num_pages == 1 ? 16 : static_cast<cuuint64_t>(p.page) * 2};
  const cuuint32_t boxes[5] = {64, 8, static_cast<cuuint32_t>(d / 64), static_cast<cuuint32_t>(box / 8), 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode()(
      &m, type == Half::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, p.base, dims,
      strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled (paged cache) failed: " + std::to_string(r));
  return m;
}

int sm_count() {
  int dev = 0, n = 0;
  B200AR_CUDA(cudaGetDevice(&dev));
  B200AR_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
  return std::min(n, kMaxParts);
}

int row_cap(int64_t rows, int group) { return static_cast<int>(std::min<int64_t>(kBlock, rows * group)); }

template <typename T, int D>
void launch(const AttnArgs& args, Half type, float* workspace, cudaStream_t s) {
  AttnArgs a = args;
  const auto unit = [&](const Pool& p) {
    if (a.hkv == 1) return D / 64;
    B200AR_CHECK(p.head % 64 == 0 && p.head / 64 * a.hkv < (1ll << 31),
                 "the pools' heads must be a multiple of 64 values apart");
    return static_cast<int>(p.head / 64);
  };
  a.unit_k = unit(a.k);
  a.unit_v = unit(a.v);
  const int group = a.hq / a.hkv, ctas = sm_count();
  int box = kTile;
  while (a.page_size % box) box /= 2;
  const CUtensorMap tk = pool_map(a.k, D, a.hkv, a.unit_k, a.page_size, a.num_pages, box, type);
  const CUtensorMap tv = pool_map(a.v, D, a.hkv, a.unit_v, a.page_size, a.num_pages, box, type);
  Workspace ws{};
  ws.row_cap = row_cap(a.rows, group);
  ws.desc = reinterpret_cast<PartDesc*>(workspace);
  ws.ml = workspace + 2ll * ctas * (sizeof(PartDesc) / 4);
  ws.acc = ws.ml + 2ll * ctas * ws.row_cap * 2;
  const bool tokens = a.batch.q_start == nullptr && group <= 32;
  auto kern = tokens ? attention_kernel<T, D, true> : attention_kernel<T, D, false>;
  static PerDeviceOnce attr;
  attr([&] {
    for (auto k : {attention_kernel<T, D, true>, attention_kernel<T, D, false>})
      B200AR_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Cfg<D>::kSmem)));
  });
  const float sign = a.scale > 0.f ? 1.f : (a.scale < 0.f ? -1.f : 0.f);
  const float scale_log2 = (sign == 0.f ? 1.f : a.scale * sign) * kLog2e;
  launch_pdl(kern, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), Cfg<D>::kSmem, s, 1, tk, tv, a, ws, group, box,
             sign, scale_log2);
  launch_pdl(merge_kernel<T, D>, dim3(static_cast<unsigned>(ctas), static_cast<unsigned>((ws.row_cap + 31) / 32)),
             dim3(D * 2), 0, s, 1, a, ws, group, ctas);
}

}  // namespace

int64_t paged_attention_workspace(int64_t rows, int hq, int hkv, int d) {
  const int64_t ctas = sm_count(), cap = row_cap(rows, hq / hkv);
  return 2 * ctas * (static_cast<int64_t>(sizeof(PartDesc)) / 4 + cap * (2 + d));
}

void paged_attention(const AttnArgs& a, int d, Half type, float* workspace, cudaStream_t s) {
  const TraceRange trace("b200ar::paged_attention");
  B200AR_CHECK(d == 64 || d == 128, "paged_attention is built for heads of 64 and 128");
  B200AR_CHECK(a.page_size % 8 == 0, "the page size must be a multiple of 8");
  B200AR_CHECK(static_cast<int64_t>(a.rows) * (a.hq / a.hkv) < (1ll << 31), "too many rows");
  if (a.rows == 0 || a.batch.seqs == 0) return;
  if (type == Half::kBf16)
    d == 64 ? launch<__nv_bfloat16, 64>(a, type, workspace, s) : launch<__nv_bfloat16, 128>(a, type, workspace, s);
  else
    d == 64 ? launch<__half, 64>(a, type, workspace, s) : launch<__half, 128>(a, type, workspace, s);
}

}  // namespace paged
}  // namespace b200ar
