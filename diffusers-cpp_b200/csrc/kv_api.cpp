// C ABI of the paged key / value cache: argument checks and launches.
#include <algorithm>
#include <cmath>

#include "kv_cache.cuh"
#include "runtime.hpp"

using dcpp::Ctx;
using dcpp::fail;

namespace {

// Runs f on the context's device; the caller's current device is restored.
template <class F>
dcpp_status kv_guarded(dcpp_ctx* ctx, const char* entry, F&& f) {
  if (!ctx) return DCPP_ERR_INVALID_ARG;
  int prev = -1;
  dcpp_status st = DCPP_OK;
  try {
    ctx->maybe_inject(entry);
    dcpp::cuda_check(cudaGetDevice(&prev), "cudaGetDevice");
    if (prev != ctx->device) dcpp::cuda_check(cudaSetDevice(ctx->device), "cudaSetDevice");
    f();
  } catch (const dcpp::Error& e) {
    ctx->last_error = e.what();
    st = e.status;
  } catch (const std::exception& e) {
    ctx->last_error = e.what();
    st = DCPP_ERR_INVALID_ARG;
  }
  if (prev >= 0 && prev != ctx->device) cudaSetDevice(prev);
  return st;
}

[[noreturn]] void bad(const char* entry, const char* what) {
  fail(DCPP_ERR_INVALID_ARG, std::string(entry) + ": " + what);
}
[[noreturn]] void unsupported(const char* entry, const char* what) {
  fail(DCPP_ERR_UNSUPPORTED, std::string(entry) + ": " + what);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int block_shift(const dcpp_kv_cache& c, const char* entry) {
  switch (c.block_size) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    case 256: return 8;
    default: unsupported(entry, "block_size must be 16, 32, 64, 128 or 256");
  }
}

// The cache's geometry (the planes too, if they are used); returns log2(block_size).
int check_cache(const dcpp_kv_cache* c, const char* entry, bool planes) {
  if (!c) bad(entry, "null cache");
  const int shift = block_shift(*c, entry);
  if (c->n_blocks < 1) bad(entry, "n_blocks must be positive");
  if (c->n_blocks > (INT32_MAX >> shift)) unsupported(entry, "n_blocks * block_size must fit 31 bits");
  if (!planes) return shift;
  if (c->type != DCPP_TYPE_BF16 && c->type != DCPP_TYPE_F16) unsupported(entry, "the cache must be BF16 or F16");
  if (c->head_dim != dcpp::kKvHeadDim) unsupported(entry, "head_dim must be 128");
  if (c->heads_kv < 1 || c->heads_kv > 4096) bad(entry, "heads_kv must be 1 .. 4096");
  const int64_t packed = c->heads_kv * c->block_size * dcpp::kKvHeadDim;
  if (c->block_stride != 0 && (c->block_stride < packed || c->block_stride % 8 || c->block_stride > (int64_t(1) << 38)))
    bad(entry, "block_stride must be 0 (packed) or a multiple of 8 not below heads_kv * block_size * head_dim");
  if (!c->d_k || !c->d_v) bad(entry, "null cache plane");
  if (!aligned(c->d_k, 16) || !aligned(c->d_v, 16)) bad(entry, "the cache planes must be 16-byte aligned");
  return shift;
}

int64_t stride_of(const dcpp_kv_cache& c) {
  return c.block_stride ? c.block_stride : c.heads_kv * c.block_size * dcpp::kKvHeadDim;
}

// Query heads over this cache.
void check_heads(const dcpp_kv_cache& c, int64_t heads, const char* entry) {
  if (heads < 1 || heads > 65535) bad(entry, "heads must be 1 .. 65535");
  if (heads % c.heads_kv) bad(entry, "heads must be a multiple of the cache's heads_kv");
}

// Rows [rows, cols] of 16-bit values with row stride ld.
void check_rows(const void* p, int64_t cols, int64_t ld, const char* entry, const char* name) {
  if (!p) fail(DCPP_ERR_INVALID_ARG, std::string(entry) + ": null " + name);
  if (!aligned(p, 16) || ld % 8 || ld < cols || ld > (int64_t(1) << 38))
    fail(DCPP_ERR_INVALID_ARG, std::string(entry) + ": " + name +
                                   " must be 16-byte aligned, its row stride a multiple of 8 not below its columns");
}

bool overlap(const void* a, int64_t a_elems, const void* b, int64_t b_elems) {
  const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + 2 * static_cast<uintptr_t>(b_elems) && y < x + 2 * static_cast<uintptr_t>(a_elems);
}

void check_attention_shape(const dcpp_kv_cache& c, int64_t heads, int64_t max_new, const char* entry) {
  check_heads(c, heads, entry);
  if (heads / c.heads_kv > dcpp::kKvMaxGroup) unsupported(entry, "too many query heads per key / value head");
  if (max_new < 1) bad(entry, "max_new must be positive");
}

}  // namespace

extern "C" {

dcpp_status dcpp_kv_plan(dcpp_ctx* ctx, const dcpp_kv_cache* cache, int64_t batch, const int32_t* d_cached,
                         const int32_t* d_new, int32_t* d_free_blocks, const int64_t* d_free_in, int64_t* d_free_out,
                         int32_t* d_block_table, int64_t max_blocks, int32_t* d_seq_lens, int32_t* d_cu_new,
                         int64_t max_tokens, int32_t* d_slots, int32_t* d_positions) {
  constexpr const char* kName = "dcpp_kv_plan";
  return kv_guarded(ctx, kName, [&] {
    dcpp::KvPlanArgs a{};
    a.block_shift = check_cache(cache, kName, false);
    if (batch < 1 || max_blocks < 1 || max_tokens < 0) bad(kName, "batch and max_blocks must be positive, max_tokens not negative");
    if (batch > dcpp::kKvMaxPlanBatch) unsupported(kName, "at most 8192 requests");
    if (max_blocks > (INT32_MAX >> a.block_shift)) unsupported(kName, "max_blocks * block_size must fit 31 bits");
    if (max_tokens > INT32_MAX - 1) unsupported(kName, "max_tokens must fit 31 bits");
    if (!d_cached || !d_new || !d_free_blocks || !d_free_in || !d_free_out || !d_block_table || !d_seq_lens || !d_cu_new ||
        (max_tokens > 0 && (!d_slots || !d_positions)))
      bad(kName, "null pointer");
    a.cached = d_cached;
    a.n_new = d_new;
    a.free_blocks = d_free_blocks;
    a.free_in = d_free_in;
    a.free_out = d_free_out;
    a.table = d_block_table;
    a.seq_lens = d_seq_lens;
    a.cu_new = d_cu_new;
    a.slots = d_slots;
    a.positions = d_positions;
    a.max_blocks = max_blocks;
    a.batch = static_cast<int32_t>(batch);
    a.max_tokens = static_cast<int32_t>(max_tokens);
    a.n_blocks = static_cast<int32_t>(cache->n_blocks);
    a.err = ctx->d_err;
    dcpp::cuda_check(dcpp::launch_kv_plan(a, ctx->stream), kName);
  });
}

dcpp_status dcpp_kv_store(dcpp_ctx* ctx, const dcpp_kv_cache* cache, int64_t tokens, int64_t heads,
                          const uint16_t* d_qkv, int64_t ld_qkv, const float* d_norm_q, const float* d_norm_k,
                          float eps, int rope, float theta, const int32_t* d_positions, const int32_t* d_slots,
                          uint16_t* d_q, int64_t ld_q) {
  constexpr const char* kName = "dcpp_kv_store";
  return kv_guarded(ctx, kName, [&] {
    dcpp::KvStoreArgs a{};
    a.block_shift = check_cache(cache, kName, true);
    check_heads(*cache, heads, kName);
    if (tokens < 0) bad(kName, "tokens must not be negative");
    if (tokens > INT32_MAX) unsupported(kName, "tokens must fit 31 bits");
    if (rope < DCPP_ROPE_NONE || rope > DCPP_ROPE_NEOX) bad(kName, "rope must be one of DCPP_ROPE_*");
    if (rope != DCPP_ROPE_NONE && !(theta > 0.0f && std::isfinite(theta))) bad(kName, "theta must be positive");
    if (!(eps >= 0.0f && std::isfinite(eps))) bad(kName, "eps must not be negative");
    if (tokens == 0) return;
    const int64_t cols = (heads + 2 * cache->heads_kv) * dcpp::kKvHeadDim;
    check_rows(d_qkv, cols, ld_qkv, kName, "qkv");
    check_rows(d_q, heads * dcpp::kKvHeadDim, ld_q, kName, "q");
    if (!(d_q == d_qkv && ld_q == ld_qkv) && overlap(d_qkv, (tokens - 1) * ld_qkv + cols, d_q, (tokens - 1) * ld_q + heads * dcpp::kKvHeadDim))
      bad(kName, "q must be apart from qkv, or be its own q columns");
    if (!d_slots || (rope != DCPP_ROPE_NONE && !d_positions)) bad(kName, "null pointer");
    if (!aligned(d_norm_q, 16) || !aligned(d_norm_k, 16)) bad(kName, "norm_q and norm_k must be 16-byte aligned");
    a.qkv = d_qkv;
    a.q = d_q;
    a.k = static_cast<uint16_t*>(cache->d_k);
    a.v = static_cast<uint16_t*>(cache->d_v);
    a.norm_q = d_norm_q;
    a.norm_k = d_norm_k;
    a.positions = d_positions;
    a.slots = d_slots;
    a.ld_qkv = ld_qkv;
    a.ld_q = ld_q;
    a.block_stride = stride_of(*cache);
    a.n_slots = cache->n_blocks << a.block_shift;
    a.tokens = static_cast<int32_t>(tokens);
    a.heads = static_cast<int32_t>(heads);
    a.heads_kv = static_cast<int32_t>(cache->heads_kv);
    a.rope = rope;
    a.eps = eps;
    a.err = ctx->d_err;
    if (rope != DCPP_ROPE_NONE) {
      // theta^(-i / 64) as a product of the powers for i's bits: six exponentials, not 64
      // (a call takes 9 us in all).
      const double base = std::log(static_cast<double>(theta));
      double f[64];
      f[0] = 1.0 / (2.0 * M_PI);
      for (int n = 1; n < 64; n *= 2) {
        const double by = std::exp(-base * n / 64.0);
        for (int i = 0; i < n; ++i) f[n + i] = f[i] * by;
      }
      // Modulo whole turns: theta below 1 may turn more than once a position.
      for (int i = 0; i < 64; ++i) a.turns[i] = static_cast<uint64_t>((f[i] < 1.0 ? f[i] : f[i] - std::floor(f[i])) * 0x1p64);
    }
    dcpp::cuda_check(dcpp::launch_kv_store(a, cache->type == DCPP_TYPE_F16, ctx->num_sms, ctx->stream), kName);
  });
}

dcpp_status dcpp_kv_attention_workspace(dcpp_ctx* ctx, const dcpp_kv_cache* cache, int64_t heads, int64_t max_new,
                                        size_t* out_bytes) {
  constexpr const char* kName = "dcpp_kv_attention_workspace";
  return kv_guarded(ctx, kName, [&] {
    if (!out_bytes) bad(kName, "null output");
    check_cache(cache, kName, true);
    check_attention_shape(*cache, heads, max_new, kName);
    *out_bytes = dcpp::kv_attention_plan(static_cast<int>(heads), static_cast<int>(cache->heads_kv), std::min<int64_t>(max_new, 1 << 24), ctx->num_sms).bytes;
  });
}

dcpp_status dcpp_kv_attention(dcpp_ctx* ctx, const dcpp_kv_cache* cache, int64_t batch, int64_t tokens, int64_t heads,
                              const uint16_t* d_q, int64_t ld_q, const int32_t* d_cu_new, const int32_t* d_seq_lens,
                              const int32_t* d_block_table, int64_t max_blocks, int64_t max_new, int causal,
                              float scale, void* d_workspace, size_t workspace_bytes, uint16_t* d_out,
                              int64_t ld_out) {
  constexpr const char* kName = "dcpp_kv_attention";
  return kv_guarded(ctx, kName, [&] {
    dcpp::KvAttnArgs a{};
    a.block_shift = check_cache(cache, kName, true);
    check_attention_shape(*cache, heads, max_new, kName);
    if (batch < 1 || tokens < 0 || max_blocks < 1) bad(kName, "batch and max_blocks must be positive, tokens not negative");
    if (batch > (1 << 20) || tokens > (1 << 24)) unsupported(kName, "at most 2^20 requests and 2^24 tokens");
    // A margin, so that sums of a length and a tile's keys fit 32 bits too.
    if (max_blocks > ((INT32_MAX - 4096) >> a.block_shift)) unsupported(kName, "max_blocks * block_size must stay below 2^31 - 4096");
    if (causal != 0 && causal != 1) bad(kName, "causal must be 0 or 1");
    if (!(scale > 0.0f && std::isfinite(scale))) bad(kName, "scale must be positive");
    if (tokens == 0) return;
    const int64_t cols = heads * dcpp::kKvHeadDim;
    check_rows(d_q, cols, ld_q, kName, "q");
    check_rows(d_out, cols, ld_out, kName, "out");
    if (overlap(d_q, (tokens - 1) * ld_q + cols, d_out, (tokens - 1) * ld_out + cols)) bad(kName, "out must be apart from q");
    if (!d_cu_new || !d_seq_lens || !d_block_table) bad(kName, "null pointer");
    const dcpp::KvAttnPlan plan =
        dcpp::kv_attention_plan(static_cast<int>(heads), static_cast<int>(cache->heads_kv), std::min<int64_t>(max_new, 1 << 24), ctx->num_sms);
    if (!d_workspace || !aligned(d_workspace, 16) || workspace_bytes < plan.bytes)
      bad(kName, ("needs a 16-byte aligned workspace of " + std::to_string(plan.bytes) + " bytes").c_str());
    a.q = d_q;
    a.out = d_out;
    a.ld_q = ld_q;
    a.ld_out = ld_out;
    a.cu_new = d_cu_new;
    a.seq_lens = d_seq_lens;
    a.table = d_block_table;
    a.max_blocks = max_blocks;
    a.max_kv = max_blocks << a.block_shift;
    a.batch = static_cast<int32_t>(batch);
    a.tokens = static_cast<int32_t>(tokens);
    a.heads = static_cast<int32_t>(heads);
    a.heads_kv = static_cast<int32_t>(cache->heads_kv);
    a.group = a.heads / a.heads_kv;
    a.n_blocks = static_cast<int32_t>(cache->n_blocks);
    a.max_new = static_cast<int32_t>(max_new < tokens ? max_new : tokens);
    a.causal = causal;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.err = ctx->d_err;
    dcpp::KvCacheView v{cache->d_k, cache->d_v, cache->n_blocks, cache->heads_kv, stride_of(*cache),
                        static_cast<int>(cache->block_size), cache->type == DCPP_TYPE_F16};
    dcpp::cuda_check(dcpp::launch_kv_attention(v, a, plan, d_workspace, ctx->stream), kName);
  });
}

}  // extern "C"
