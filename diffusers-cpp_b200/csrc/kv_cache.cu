// Paged key / value cache: the step plan (block tables, slot maps) and the
// store of a step's keys and values.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kv_cache.cuh"

namespace dcpp {

namespace {

// ------------------------------------------------------------------ plan
// With old_b = ceil(cached_b / bs), a live request grows to seq_b = cached_b +
// new_b tokens and needs need_b = ceil(seq_b / bs) - old_b blocks; they are
// ring[(head + P(need)_b + i) mod n], P the exclusive prefix sum in request
// order.  A finished request (new_b < 0) returns its old_b blocks to ring[(tail
// + P(back)_b + i) mod n].  Nothing read is written: allocations come from
// [head, tail), returned blocks go behind tail (free from the next step on), and
// of the table only entries >= old_b change, so the result does not depend on
// the order of the threads.
//
// The work is a few hundred KB at most: what it costs is the launch and a chain
// of dependent reads (lengths -> prefix sums -> block ids -> slots).  So one
// launch does all of it.  Every CTA of one cluster computes the prefix sums of
// the whole batch for itself (the lengths come from L2; cheaper than another
// launch or a grid barrier), the cluster barrier orders all reads of the lengths
// and ring counters before their in-place update, and the tokens are spread over
// the cluster's threads, each finding its request by binary search in shared
// memory.
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int64_t warp_incl_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

__global__ void __launch_bounds__(kPlanThreads, 1) kv_plan_kernel(const __grid_constant__ KvPlanArgs p) {
  namespace cg = cooperative_groups;
  extern __shared__ int32_t plan_smem[];
  const int B = p.batch;
  int32_t* s_cached = plan_smem;       // [B]
  int32_t* s_cu = s_cached + B;        // [B + 1]
  int32_t* s_need = s_cu + B + 1;      // [B + 1]
  int32_t* s_back = s_need + B + 1;    // [B + 1]
  __shared__ int64_t s_warp[3][32];
  __shared__ int64_t s_head, s_tail;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = p.block_shift;
  const int32_t mask = (1 << shift) - 1;
  const int64_t max_kv = p.max_blocks << shift;  // <= INT32_MAX
  if (tid == 0) {
    s_head = p.free_in[0];
    s_tail = p.free_in[1];
  }

  // Each thread sums its run of requests; 64-bit sums, so that no input overflows them.
  const int seg = (B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * seg, B), b1 = min(b0 + seg, B);
  int64_t sum[3] = {0, 0, 0};
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const int32_t c = p.cached[b], n = p.n_new[b];
    s_cached[b] = c;
    bad |= c < 0 || c > max_kv || (n > 0 && n > max_kv - c);
    const int64_t old = (static_cast<int64_t>(c) + mask) >> shift;
    if (n < 0) {
      sum[2] += old;
    } else {
      sum[0] += n;
      sum[1] += ((static_cast<int64_t>(c) + n + mask) >> shift) - old;
    }
  }
  int64_t at[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    at[k] = warp_incl_scan(sum[k], lane);
    if (lane == 31) s_warp[k][warp] = at[k];
    at[k] -= sum[k];
  }
  const bool any_bad = __syncthreads_or(bad);
  int64_t total[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int64_t w = warp_incl_scan(s_warp[k][lane], lane);
    total[k] = __shfl_sync(0xffffffffu, w, 31);
    const int64_t before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    at[k] += warp > 0 ? before : 0;
  }
  const int64_t head = s_head, tail = s_tail;
  const bool ring_ok = head >= 0 && tail >= head && tail - head <= p.n_blocks && total[2] + (tail - head) <= p.n_blocks;
  const bool fits = total[0] <= p.max_tokens && total[1] <= tail - head;
  const bool ok = !any_bad && ring_ok && fits;  // the same in every CTA

  // Prefix sums of an accepted step (each fits 32 bits); a refused one has no tokens.
  for (int b = b0; b < b1; ++b) {
    s_cu[b] = ok ? static_cast<int32_t>(at[0]) : 0;
    s_need[b] = ok ? static_cast<int32_t>(at[1]) : 0;
    s_back[b] = ok ? static_cast<int32_t>(at[2]) : 0;
    const int32_t c = s_cached[b], n = p.n_new[b];
    const int64_t old = (static_cast<int64_t>(c) + mask) >> shift;
    if (n < 0) {
      at[2] += old;
    } else {
      at[0] += n;
      at[1] += ((static_cast<int64_t>(c) + n + mask) >> shift) - old;
    }
  }
  if (tid == 0) {
    s_cu[B] = ok ? static_cast<int32_t>(total[0]) : 0;
    s_need[B] = ok ? static_cast<int32_t>(total[1]) : 0;
    s_back[B] = ok ? static_cast<int32_t>(total[2]) : 0;
  }
  auto cluster = cg::this_cluster();
  const int n_cta = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  // All reads of lengths and ring counters (any of which may be updated in place) come before this.
  if (n_cta > 1)
    cluster.sync();
  else
    __syncthreads();

  if (rank == 0) {
    for (int b = tid; b <= B; b += kPlanThreads) {
      p.cu_new[b] = s_cu[b];
      if (b == B) break;
      const bool gone = s_back[b + 1] > s_back[b];
      p.seq_lens[b] = gone ? 0 : s_cached[b] + (s_cu[b + 1] - s_cu[b]);
    }
    if (tid == 0) {
      p.free_out[0] = head + s_need[B];
      p.free_out[1] = tail + s_back[B];
      if (!ok) record_error(p.err, (any_bad || !ring_ok) ? kDevBadCache : kDevNoBlocks);
    }
  }

  const int n = p.n_blocks;
  const int head_at = ok ? static_cast<int>(head % n) : 0;
  const int tail_at = ok ? static_cast<int>(tail % n) : 0;
  const int total_new = s_cu[B];
  bool wrong_block = false;
  for (int64_t t64 = static_cast<int64_t>(rank) * kPlanThreads + tid; t64 < p.max_tokens;
       t64 += static_cast<int64_t>(n_cta) * kPlanThreads) {
    const int t = static_cast<int>(t64);
    if (t >= total_new) {
      p.slots[t] = -1;
      p.positions[t] = 0;
      continue;
    }
    int lo = 0, hi = B;  // s_cu[lo] <= t < s_cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cu[mid] <= t) lo = mid; else hi = mid;
    }
    const int c = s_cached[lo];
    const int pos = c + (t - s_cu[lo]);
    const int idx = pos >> shift, old = (c + mask) >> shift;
    int32_t* row = p.table + lo * p.max_blocks;
    int32_t blk;
    if (idx < old) {
      blk = row[idx];
    } else {
      int64_t r = static_cast<int64_t>(head_at) + s_need[lo] + (idx - old);
      if (r >= n) r -= n;
      blk = p.free_blocks[r];
      // The first token of a new block is a new token: it writes the table entry.
      if ((pos & mask) == 0) row[idx] = blk;
    }
    const bool in = blk >= 0 && blk < n;
    wrong_block |= !in;
    p.slots[t] = in ? (blk << shift) + (pos & mask) : -1;
    p.positions[t] = pos;
  }
  // Blocks of finished requests: a warp for each request.
  if (s_back[B] > 0) {
    for (int b = rank * 32 + warp; b < B; b += n_cta * 32) {
      const int from = s_back[b], count = s_back[b + 1] - from;
      for (int i = lane; i < count; i += 32) {
        int64_t r = static_cast<int64_t>(tail_at) + from + i;
        if (r >= n) r -= n;
        const int32_t blk = p.table[b * p.max_blocks + i];
        wrong_block |= blk < 0 || blk >= n;
        p.free_blocks[r] = blk;
      }
    }
  }
  if (wrong_block) record_error(p.err, kDevBadCache);
}

// ----------------------------------------------------------------- store
// y = x * rsqrt(mean(x^2) + eps) * w over a head's 128 channels, then each pair
// (a, b) -> (a cos - b sin, a sin + b cos), angle = position * theta^(-i / 64).
// Everything is read and written once: bound by HBM.  One CTA per token, eight
// lanes per head vector, each with 16-byte loads of channels 8l.. and 64 + 8l..
// (both members of the half-split pairs in one lane), all loads of up to
// kStoreVecs vectors per lane issued before anything waits.  The 64 angles are
// shared by all heads of the token: computed once into shared memory by the
// first 64 threads, in turns and in 64 bits (position * turns keeps 2^-53
// relative, so a far position's fraction of a turn is good to far below an f32
// rounding of the sine), then reduced to [-1/2, 1/2] turn.  Sums and the
// rotation are f32, rounded once to the cache's type.
constexpr int kStoreThreads = 128;
constexpr int kStoreVecs = 3;

template <bool F16>
__device__ __forceinline__ void unpack2(uint32_t u, float& lo, float& hi) {
  if constexpr (F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    lo = f.x;
    hi = f.y;
  } else {
    lo = __uint_as_float(u << 16);
    hi = __uint_as_float(u & 0xFFFF0000u);
  }
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

template <bool F16>
__global__ void __launch_bounds__(kStoreThreads) kv_store_kernel(const __grid_constant__ KvStoreArgs p) {
  __shared__ float2 s_cs[64];
  const int t = blockIdx.x;
  const int slot = p.slots[t];
  if (slot < 0) return;
  if (slot >= p.n_slots) {
    if (threadIdx.x == 0) record_error(p.err, kDevBadCache);
    return;
  }
  const int l = threadIdx.x & 7, vec0 = threadIdx.x >> 3;
  constexpr int kPerPass = kStoreThreads / 8;
  const int n_vec = p.heads + 2 * p.heads_kv;
  const uint16_t* src = p.qkv + t * p.ld_qkv + l * 8;
  const int64_t blk = slot >> p.block_shift, off = slot & ((1 << p.block_shift) - 1);
  bool angles = false;
  for (int base = 0; base < n_vec; base += kPerPass * kStoreVecs) {
    uint4 lo[kStoreVecs], hi[kStoreVecs];
#pragma unroll
    for (int j = 0; j < kStoreVecs; ++j) {
      const int vec = base + j * kPerPass + vec0;
      if (vec < n_vec) {
        lo[j] = *reinterpret_cast<const uint4*>(src + vec * 128);
        hi[j] = *reinterpret_cast<const uint4*>(src + vec * 128 + 64);
      }
    }
    if (p.rope && !angles) {
      if (threadIdx.x < 64) {
        const double u = static_cast<double>(p.positions[t]) * p.turns[threadIdx.x];
        const float f = static_cast<float>(u - rint(u));
        float sn, cs;
        sincospif(2.0f * f, &sn, &cs);
        s_cs[threadIdx.x] = make_float2(cs, sn);
      }
      __syncthreads();
      angles = true;
    }
#pragma unroll
    for (int j = 0; j < kStoreVecs; ++j) {
      const int vec = base + j * kPerPass + vec0;
      // The eight lanes of a vector agree on vec, so their shuffles stay together.
      if (vec >= n_vec) continue;
      if (vec < p.heads + p.heads_kv) {
        const bool is_q = vec < p.heads;
        float x[16];
        const uint32_t* a = reinterpret_cast<const uint32_t*>(&lo[j]);
        const uint32_t* b = reinterpret_cast<const uint32_t*>(&hi[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          unpack2<F16>(a[i], x[2 * i], x[2 * i + 1]);
          unpack2<F16>(b[i], x[8 + 2 * i], x[9 + 2 * i]);
        }
        const float* w = is_q ? p.norm_q : p.norm_k;
        if (w) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
          const unsigned lanes = 0xFFu << (threadIdx.x & 24);
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
          const float rs = 1.0f / sqrtf(ss * (1.0f / 128.0f) + p.eps);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= rs * __ldg(w + (i < 8 ? l * 8 + i : 56 + l * 8 + i));
        }
        if (p.rope == 2) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 cs = s_cs[l * 8 + i];
            const float u = x[i], v = x[8 + i];
            x[i] = u * cs.x - v * cs.y;
            x[8 + i] = u * cs.y + v * cs.x;
          }
        } else if (p.rope == 1) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // pairs 4l.. of the low half, 32 + 4l.. of the high half
            const float2 cs = s_cs[(i < 4 ? l * 4 + i : 28 + l * 4 + i)];
            const float u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = u * cs.x - v * cs.y;
            x[2 * i + 1] = u * cs.y + v * cs.x;
          }
        }
        lo[j] = make_uint4(pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(x[4], x[5]), pack2<F16>(x[6], x[7]));
        hi[j] = make_uint4(pack2<F16>(x[8], x[9]), pack2<F16>(x[10], x[11]), pack2<F16>(x[12], x[13]),
                           pack2<F16>(x[14], x[15]));
      }
      uint16_t* dst;
      if (vec < p.heads) {
        dst = p.q + t * p.ld_q + vec * 128;
      } else {
        const int h = (vec - p.heads) % p.heads_kv;
        dst = (vec < p.heads + p.heads_kv ? p.k : p.v) + blk * p.block_stride +
              ((static_cast<int64_t>(h) << p.block_shift) + off) * 128;
      }
      *reinterpret_cast<uint4*>(dst + l * 8) = lo[j];
      *reinterpret_cast<uint4*>(dst + 64 + l * 8) = hi[j];
    }
  }
}

}  // namespace

cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t s) {
  if (a.batch < 1 || a.batch > kKvMaxPlanBatch) return cudaErrorInvalidValue;
  const size_t smem = (static_cast<size_t>(a.batch) * 4 + 3) * sizeof(int32_t);
  cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  // A CTA for every 4096 rows of the maps, at most a portable cluster of 8.
  const int64_t want = (static_cast<int64_t>(a.max_tokens) + 4095) / 4096;
  const unsigned n = want <= 1 ? 1 : want <= 2 ? 2 : want <= 4 ? 4 : 8;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_plan_kernel, a);
}

cudaError_t launch_kv_store(const KvStoreArgs& a, bool f16, cudaStream_t s) {
  if (a.tokens <= 0) return cudaSuccess;
  if (f16)
    kv_store_kernel<true><<<a.tokens, kStoreThreads, 0, s>>>(a);
  else
    kv_store_kernel<false><<<a.tokens, kStoreThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace dcpp
