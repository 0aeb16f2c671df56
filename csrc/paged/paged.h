// Host API of the operators on a paged KV cache (rope_paged.cu, attention_paged.cu).
//
// A batch is S sequences. Sequence s has kv_len[s] tokens in the cache, its
// last n_s = q_start[s + 1] - q_start[s] of them new in this call; row
// q_start[s] + i of the call's inputs is the token at position
// kv_len[s] - n_s + i. Without q_start every sequence has one new token
// (row s). Position p of sequence s lives in slot p % page_size of page
// page_table[s][p / page_size]. Rows behind q_start[S] are not touched.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace b200ar {
namespace paged {

// Element type of queries, keys and values.
enum class Half { kBf16 = 0, kFp16 = 1 };

// Codes left in the error word; the access that they speak of is skipped.
constexpr int kErrTimeout = 2;   // a bounded wait expired
constexpr int kErrPosition = 3;  // a token's position is outside the rotary table
constexpr int kErrPage = 4;      // a position without a page, or a page outside the pool

struct Batch {
  const int* page_table;  // [S, max_pages], row stride `table_stride`
  const int* kv_len;      // [S]
  const int* q_start;     // [S + 1] or null
  int64_t table_stride;
  int seqs, max_pages;
  int rows;  // of the call's inputs: offsets are cut to them
};

// K and V pools [num_pages, page_size, kv_heads, d], strides in elements.
struct Pool {
  void* base;
  int64_t page, tok, head;
};

struct RopeArgs {
  const void* qkv;      // [rows, (hq + 2 hkv) * d], row stride `qkv_stride`
  const void* q_gamma;  // [d] or null
  const void* k_gamma;
  const float* cos_t;   // [positions, d / 2]
  const float* sin_t;
  void* q_out;          // [rows, hq, d], strides q_tok and q_head
  int64_t qkv_stride, q_tok, q_head;
  Pool k, v;
  Batch batch;
  int* err;
  int rows, hq, hkv, positions, num_pages, page_size;
  float eps;
};
void qk_norm_rope_paged(const RopeArgs& a, int d, Half type, cudaStream_t s);

struct AttnArgs {
  const void* q;  // [rows, hq, d]
  void* out;      // [rows, hq, d]
  int64_t q_tok, q_head, o_tok, o_head;
  Pool k, v;
  Batch batch;
  int* err;
  int rows, hq, hkv, num_pages, page_size;
  int capacity;  // positions of a row of the page table
  int window;    // positions that a row sees, its own included; 0: all
  int unit_k, unit_v;  // set by paged_attention(): 64-value units from KV head to KV head
  bool causal;
  float scale;
};
// Floats of workspace for a call: partial results of the blocks that the
// schedule cuts, and their descriptions. Not kept from call to call.
int64_t paged_attention_workspace(int64_t rows, int hq, int hkv, int d);
void paged_attention(const AttnArgs& a, int d, Half type, float* workspace, cudaStream_t s);

}  // namespace paged
}  // namespace b200ar
