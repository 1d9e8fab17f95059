// Helpers shared by the paged attention kernels.
#pragma once

#include <atomic>

#include "common.cuh"
#include "kv_cache.cuh"
#include "softmax.cuh"

namespace dcpp {

template <bool F16>
__device__ __forceinline__ uint32_t kv_pack2(float lo, float hi) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

// Bounded wait that looks at nothing but its barrier and the clock: another
// kernel's recorded error does not end this one's work.
__device__ __forceinline__ bool kv_wait(uint64_t* bar, uint32_t parity, int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer();
  for (;;) {
    if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    if (globaltimer() - t0 > kWaitTimeoutNs) {
      record_error(err, kDevTimeoutKv);
      return false;
    }
  }
}

// Dynamic shared memory limit of a kernel, set once per device.
template <class K>
cudaError_t allow_smem(K* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Tensor map of one cache plane: {channel, token of the block, head, block}, boxes of 64 channels x box_rows tokens.
cudaError_t kv_cache_map(CUtensorMap* m, const KvCacheView& c, const void* base, int box_rows);
// Tensor map of the query rows: {channel, head, token}, boxes of 64 channels x group heads x box_tokens tokens.
cudaError_t kv_query_map(CUtensorMap* m, const KvAttnArgs& a, bool f16, int box_tokens);

// The tensor-core kernel for many query rows (kv_attention_tc.cu).
constexpr int kTcKT = 128;         // keys of a tile
constexpr int kTcRows = 256;       // query rows of a unit: two tiles of 128
constexpr int kTcMinTiles = 4;     // fewest key tiles of a part
cudaError_t launch_kv_tc(const KvCacheView& c, KvAttnArgs a, cudaStream_t s);

}  // namespace dcpp
