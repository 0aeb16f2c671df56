// How the tiles of a paged attention call are given to CTAs, on the device.
//
// The new tokens of a sequence and the G query heads of a KV head are G n rows
// that share keys and values (row r: token r / G, head r % G). A block is 256
// such rows of one sequence and KV head; its work is the run of 128-token
// tiles that some row sees. All blocks' tiles, in the order sequence, head,
// block, tile, form one line, cut into equal parts, one for each CTA; a block
// that a cut falls into is computed in parts and merged (merge_kernel).
//
// The line is measured in a weight that has a closed form and is near the
// work: a block's tokens times G plus a constant for its start and end (kFixed),
// times the work of a tile. With causal rows it grows by the same step from block
// to block up to the window's limit, so the position of any block is a short sum, and a CTA
// finds its part from one scan over the sequences. Any weight gives a correct
// cut: only the balance depends on it.
#pragma once

#include "batch.cuh"

namespace b200ar {
namespace paged {

constexpr int kTile = 128;   // tokens of a K or V tile
constexpr int kBlock = 256;  // rows of a block
// The start and end of a block, in tiles: its queries, the first tile's way through the pipeline with nothing beside
// it, the join and the output. Measured with 1, 2, 3, 4, 5 and 6: 64 tokens over contexts of 1 to 4095 take 137, 116,
// 111, 107, 102 and 105 us, a first prompt of 2048 takes 155, 128, 120, 118, 121 and 123 us.
constexpr int kFixed = 5;
// Work of a tile for a sequence of over 128 rows against one of fewer. Measured 3 to 2 and 1 to 1: 24 prompts' chunks
// and single tokens over caches of up to 5000 with 32 heads of 128 take 181 and 197 us. (A call with single tokens only,
// kTokens, has none over 128: the second factor alone costs it 0.8 us of 17.)
constexpr int kWideTile = 3, kNarrowTile = 2;

// Quotients of numbers that are nearly always below 2^32.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

template <bool kTokens>
struct SeqWork {
  int n, len, q0, blocks;
  int64_t a, cap, head;  // weight of block 0, limit of a weight, weight of all blocks of one head
  static constexpr int64_t kNoLimit = 1ll << 60;
  int step;              // by which the weight grows from block to block, up to the limit

  __device__ __forceinline__ void load(const AttnArgs& p, int group, int s) {
    q0 = q_begin(p.batch, s);
    n = max(q_begin(p.batch, s + 1) - q0, 0);
    len = __ldg(p.batch.kv_len + s);
    blocks = static_cast<int>((static_cast<int64_t>(n) * group + kBlock - 1) / kBlock);
    const int unit = kTokens ? 1 : static_cast<int64_t>(n) * group > kBlock / 2 ? kWideTile : kNarrowTile;
    const int fixed = kFixed * kTile * group * unit;
    cap = kNoLimit;
    if (p.causal) {
      a = static_cast<int64_t>(unit * group) * max(len - n, 0) + unit * kBlock + fixed;
      step = unit * kBlock;
      if (p.window > 0)
        cap = static_cast<int64_t>(unit * group) * (static_cast<int64_t>(p.window) + kTile) + step + fixed;
    } else {
      a = static_cast<int64_t>(unit * group) * max(len, 0) + fixed;
      step = 0;
    }
    head = before(blocks);
  }
  __device__ __forceinline__ int64_t weight(int b) const { return min(a + static_cast<int64_t>(step) * b, cap); }
  // Weight of the blocks before b.
  __device__ __forceinline__ int64_t before(int b) const {
    if (step == 0) return a * b;
    if (cap == kNoLimit) return a * b + step * (static_cast<int64_t>(b) * (b - 1) / 2);
    const int64_t ramp = a >= cap ? 0 : min(static_cast<int64_t>(b), (cap - a + step - 1) / step);
    return a * ramp + step * (ramp * (ramp - 1) / 2) + (b - ramp) * cap;
  }
};

// A CTA's part of the line: from offset off0 of sequence s0 to offset off1 of s1.
struct Part {
  int64_t off0, off1;
  int s0, s1;
  int active;
};

// A part of a block: tiles [t0, t1) of its `tiles`, the first of which starts
// at token 128 tile0.
struct Item {
  int s, h, b;
  int n, len, q0;
  int row0, rows;  // rows of the block among the sequence's G n
  int pos0;        // position of the block's first row
  int begin, end;  // positions that some row sees
  int see0, hide0;  // positions [see0, hide0) are seen by every row, if there are any: see0 may lie behind hide0
  int tile0, tiles, t0, t1;
  bool over;       // some row sees positions behind the page table
  int cleared;     // values were taken out of V (attention_kernel)

  __device__ __forceinline__ bool whole() const { return t1 - t0 == tiles; }
  // Whether the row x of the sequence's G n sees anything: with a window its own position at least.
  __device__ __forceinline__ bool sees(int x, int group, bool causal) const {
    return causal ? len - n + x / group >= 0 : len > 0;
  }
  // Whether the tile from position c0 on has some that not every row sees.
  __device__ __forceinline__ bool cut(int c0) const { return c0 < see0 || c0 + kTile > hide0; }

  // All but the part: block b of KV head h of sequence s, whose n new rows of len tokens start at row q0.
  __device__ __forceinline__ void set_block(const AttnArgs& p, int group, int s_, int h_, int b_, int n_, int len_,
                                            int q0_) {
    s = s_, h = h_, b = b_, n = n_, len = len_, q0 = q0_;
    row0 = b * kBlock;
    rows = min(kBlock, n * group - row0);
    pos0 = len - n + row0 / group;
    const int last = len - n + (row0 + rows - 1) / group;
    begin = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
    end = max(0, p.causal ? last + 1 : len);
    over = end > p.capacity;
    end = min(end, p.capacity);
    see0 = p.window > 0 ? max(0, last - p.window + 1) : 0;
    hide0 = p.causal ? min(end, max(0, pos0 + 1)) : end;
    tile0 = begin / kTile;
    tiles = end > begin ? (end + kTile - 1) / kTile - tile0 : 1;
    cleared = 0;
  }
};

// Walks a CTA's items. Every role of the kernel walks them by itself.
template <bool kTokens>
struct Walk {
  Part part;
  SeqWork<kTokens> w;
  int s, h, b;
  int64_t at;  // offset of block b of head h in its sequence

  __device__ __forceinline__ void start(const AttnArgs& p, int group, const Part& pt) {
    part = pt;
    s = pt.s0;
    if (!pt.active) return;
    w.load(p, group, s);
    h = static_cast<int>(quotient(pt.off0, w.head));
    const int64_t rest = pt.off0 - h * w.head;
    int lo = 0, hi = w.blocks - 1;  // the last block with before(b) <= rest
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (w.before(mid) <= rest)
        lo = mid;
      else
        hi = mid - 1;
    }
    b = lo;
    at = h * w.head + w.before(b);
  }

  __device__ __forceinline__ bool next(const AttnArgs& p, int group, Item& it) {
    if (!part.active) return false;
    for (;;) {
      if (b >= w.blocks) {
        b = 0;
        if (w.blocks == 0 || ++h >= p.hkv) {
          if (++s > part.s1) return false;
          h = 0;
          at = 0;
          w.load(p, group, s);
          if (w.blocks == 0) continue;
        }
      }
      if (s > part.s1 || (s == part.s1 && at >= part.off1)) return false;
      const int64_t weight = w.weight(b);
      it.set_block(p, group, s, h, b, w.n, w.len, w.q0);
      const int64_t x0 = s == part.s0 ? max(part.off0 - at, static_cast<int64_t>(0)) : 0;
      const int64_t x1 = s == part.s1 ? min(part.off1 - at, weight) : weight;
      it.t0 = x0 == 0 ? 0 : static_cast<int>(quotient(x0 * it.tiles, weight));
      it.t1 = x1 == weight ? it.tiles : static_cast<int>(quotient(x1 * it.tiles, weight));
      at += weight;
      ++b;
      if (it.t0 < it.t1) return true;
    }
  }
};

// Finds the calling CTA's part. Called by all `kThreads` threads; `red` is
// shared scratch of 33 int64. One CTA gets at least about one tile.
template <int kThreads, bool kTokens>
__device__ __forceinline__ void find_part(const AttnArgs& p, int group, int64_t* red, Part* part) {
  constexpr int kWarps = kThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (p.batch.seqs + kThreads - 1) / kThreads;
  const int lo = min(static_cast<int>(threadIdx.x) * per, p.batch.seqs), hi = min(lo + per, p.batch.seqs);
  int64_t mine = 0;
  SeqWork<kTokens> w;
  for (int s = lo; s < hi; ++s) {
    w.load(p, group, s);
    mine += w.head * p.hkv;
  }
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (threadIdx.x == 0) part->active = 0;
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) base += red[i];
    total += red[i];
  }
  // Equal parts, none below the weight of one tile (its tokens and its block's constant).
  const int64_t least = static_cast<int64_t>((kTokens ? 1 : kNarrowTile) * kTile) * group;
  const int64_t part_weight = max(quotient(total + gridDim.x - 1, gridDim.x), least);
  const int64_t x0 = part_weight * blockIdx.x, x1 = min(x0 + part_weight, total);
  if (x0 < total) {
    int64_t off = base + inc - mine;  // the line's position of sequence lo
    if (mine > 0 && x1 > off && x0 < off + mine)
      for (int s = lo; s < hi; ++s) {
        w.load(p, group, s);
        const int64_t size = w.head * p.hkv;
        if (size > 0 && x0 >= off && x0 < off + size) {
          part->s0 = s;
          part->off0 = x0 - off;
          part->active = 1;
        }
        if (size > 0 && x1 > off && x1 <= off + size) {
          part->s1 = s;
          part->off1 = x1 - off;
        }
        off += size;
      }
  }
  __syncthreads();
}

}  // namespace paged
}  // namespace b200ar
