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

// One try on the barrier at a shared-memory address (the thread may sleep for a while in it).
__device__ __forceinline__ bool kv_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Bounded wait that looks at nothing but its barrier and the clock: another
// kernel's recorded error does not end this one's work.  The part behind the first
// try stays out of line: these kernels' loops are long, and instruction fetch counts.
static __device__ __noinline__ bool kv_wait_on(uint32_t bar, uint32_t parity, int* err) {
  unsigned long long t0 = 0;
  for (uint32_t k = 1;; ++k) {
    if (kv_try_wait(bar, parity)) return true;
    if ((k & 255u) == 0) {  // the clock is slow to read: not on the way of a wait that ends soon
      const unsigned long long t = globaltimer();
      if (t0 == 0) t0 = t;
      if (t - t0 > kWaitTimeoutNs) {
        record_error(err, kDevTimeoutKv);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool kv_wait(uint64_t* bar, uint32_t parity, int* err) {
  const uint32_t b = smem_u32(bar);
  return kv_try_wait(b, parity) || kv_wait_on(b, parity, err);
}
// The same for a converged warp: met by all its lanes.
__device__ __forceinline__ bool kv_wait_warp(uint32_t bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, kv_try_wait(bar, parity)) || __all_sync(0xffffffffu, kv_wait_on(bar, parity, err));
}
__device__ __forceinline__ bool kv_wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  return kv_wait_warp(smem_u32(bar), parity, err);
}

// Barrier `id` among `threads` threads (whole warps) of the block.
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The maximum; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ int cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return static_cast<int>(n);
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
cudaError_t launch_kv_tc(const KvCacheView& c, KvAttnArgs a, int ctas, int cluster, cudaStream_t s);

}  // namespace dcpp
