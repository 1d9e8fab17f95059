// Paged key / value cache: launch entry points of its kernels (host-callable).
//
// The cache holds n_blocks blocks of block_size tokens; K and V block b, head
// h, token o of the block start at b * block_stride + (h * block_size + o) * 128.
// A request's tokens lie in the blocks its row of the block table names, in order.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace dcpp {

constexpr int kKvHeadDim = 128;
constexpr int kKvMaxPlanBatch = 8192;  // requests of one plan: its prefix sums live in shared memory
constexpr int kKvMaxGroup = 128;        // query heads per key / value head

// One step's block tables and maps (kv_plan_kernel).
struct KvPlanArgs {
  const int32_t* cached;   // [batch] tokens each request has in the cache
  const int32_t* n_new;    // [batch] tokens it adds; < 0: finished, its blocks go back
  int32_t* free_blocks;    // [n_blocks] ring of free block ids
  const int64_t* free_in;  // {head, tail} counters of the ring: free = tail - head
  int64_t* free_out;       // the same after the step (may be free_in)
  int32_t* table;          // [batch, max_blocks]
  int32_t* seq_lens;       // [batch] (may be cached)
  int32_t* cu_new;         // [batch + 1]
  int32_t* slots;          // [max_tokens]
  int32_t* positions;      // [max_tokens]
  int64_t max_blocks;
  int32_t batch;
  int32_t max_tokens;
  int32_t n_blocks;
  int32_t block_shift;     // log2(block_size)
  int* err;
};
cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t s);

// RMSNorm + rotary embedding of q and k, k and v into their cache slots.
struct KvStoreArgs {
  const uint16_t* qkv;     // [tokens, >= (heads + 2 heads_kv) * 128], row stride ld_qkv
  uint16_t* q;             // [tokens, heads * 128], row stride ld_q (may be qkv's own q columns)
  uint16_t* k;
  uint16_t* v;
  const float* norm_q;     // [128] or null
  const float* norm_k;
  const int32_t* positions;
  const int32_t* slots;    // < 0: the row is skipped
  int64_t ld_qkv, ld_q, block_stride;
  int64_t n_slots;         // n_blocks * block_size
  int32_t tokens, heads, heads_kv;
  int32_t block_shift;
  int32_t rope;            // 0 none, 1 pairs (2i, 2i + 1), 2 pairs (i, i + 64)
  float eps;
  int* err;
  uint64_t turns[64];      // 2^64 x the turns per position of pair i, theta^(-i / 64) / (2 pi)
};
cudaError_t launch_kv_store(const KvStoreArgs& a, bool f16, int num_sms, cudaStream_t s);

// The unit that the cut before a part goes through (rows = 0: none): its parts and
// where its rows go.
struct KvCut {
  int32_t first, last;  // the parts it lies in
  int32_t rows;
  int32_t tok0;         // row of q and out of its first token
  int32_t head0;        // its first query head
  int32_t pad[3];
};

// Attention of a batch's new tokens over the cache.
struct KvAttnArgs {
  const uint16_t* q;        // [tokens, heads, 128], row stride ld_q
  uint16_t* out;            // [tokens, heads, 128], row stride ld_out
  int64_t ld_q, ld_out;
  const int32_t* cu_new;    // [batch + 1]
  const int32_t* seq_lens;  // [batch] cached tokens, the new ones included
  const int32_t* table;     // [batch, max_blocks]
  int64_t max_blocks;
  int64_t max_kv;           // max_blocks * block_size
  int32_t batch, tokens, heads, heads_kv, group;
  int32_t n_blocks, block_shift, box_rows;
  int32_t max_new;
  int32_t causal;
  float scale_log2;         // scale * log2(e)
  int32_t unit_tokens;      // query tokens of one work unit
  int32_t unit_shift;       // log2 of it, -1: not a power of two
  int32_t grid;             // parts that the work is cut into, at most
  int32_t direct;           // > 0: the direct form, units of the longest possible sequence
  struct KvCut* cuts;       // [grid] what the cut before each part goes through
  float* part_o;            // [2 * grid][unit rows][128] partial sums
  float2* part_ml;          // [2 * grid][unit rows] their running maximum and sum
  int* err;
  uint32_t group_inv;       // ceil(2^16 / group)
  // row / group of a unit's row: its rounding up adds less than 1 / group below 2^16 / group.
  __host__ __device__ int row_token(int row) const { return static_cast<int>(static_cast<uint32_t>(row) * group_inv >> 16); }
};

// Geometry of a launch: which kernel runs and the workspace it needs.
struct KvAttnPlan {
  int unit_rows;    // query rows (token, head of the group) of one work unit
  int unit_tokens;
  int grid;
  size_t cut_bytes, ml_bytes, bytes;
};
KvAttnPlan kv_attention_plan(int heads, int heads_kv, int64_t max_new, int num_sms);

struct KvCacheView {
  const void* k;
  const void* v;
  int64_t n_blocks, heads_kv, block_stride;
  int block_size;
  bool f16;
};
// `a` carries everything but the fields that follow from the plan.
cudaError_t launch_kv_attention(const KvCacheView& c, KvAttnArgs a, const KvAttnPlan& plan, void* workspace,
                                cudaStream_t s);

}  // namespace dcpp
