// Paged key / value cache: the step plan (block tables, slot maps) and the
// store of a step's keys and values.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "kv_cache.cuh"
#include "kv_device.cuh"

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
// memory.  Measured: 64 requests of one token 4.6 us, 1000 requests with 30k tokens
// 9.2 us (10.8 us with one row of the maps to a thread instead of four).
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int64_t warp_incl_scan(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// The maps of PER consecutive rows to a thread: one search, and their block ids on the
// way together.  Returns whether a block id was wrong.
template <int PER>
__device__ __forceinline__ bool plan_rows(const KvPlanArgs& p, const int32_t* s_cached, const int32_t* s_cu,
                                          const int32_t* s_need, int head_at, int rank, int n_cta) {
  const int tid = threadIdx.x, B = p.batch, shift = p.block_shift, n = p.n_blocks;
  const int32_t mask = (1 << shift) - 1;
  const int total_new = s_cu[B];
  bool wrong_block = false;
  const bool wide = ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) & 15) == 0;
  for (int64_t t64 = PER * (static_cast<int64_t>(rank) * kPlanThreads + tid); t64 < p.max_tokens;
       t64 += PER * static_cast<int64_t>(n_cta) * kPlanThreads) {
    const int t0 = static_cast<int>(t64);
    int slot[PER], where[PER];
    if (t0 < total_new) {
      int lo = 0, hi = B;  // s_cu[lo] <= t0 < s_cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t0) lo = mid; else hi = mid;
      }
      int32_t blk[PER];
      int32_t* entry[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int t = t0 + k;
        where[k] = 0;
        blk[k] = -1;
        entry[k] = nullptr;
        if (t >= total_new) continue;
        while (s_cu[lo + 1] <= t) ++lo;  // ends: t < total_new = s_cu[B]
        const int c = s_cached[lo];
        const int pos = where[k] = c + (t - s_cu[lo]);
        const int idx = pos >> shift, old = (c + mask) >> shift;
        int32_t* row = p.table + lo * p.max_blocks;
        if (idx < old) {
          blk[k] = row[idx];
        } else {
          int64_t r = static_cast<int64_t>(head_at) + s_need[lo] + (idx - old);
          if (r >= n) r -= n;
          blk[k] = p.free_blocks[r];
          // The first token of a new block is a new token: it writes the table entry.
          if ((pos & mask) == 0) entry[k] = row + idx;
        }
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        if (entry[k]) *entry[k] = blk[k];
        const bool in = blk[k] >= 0 && blk[k] < n;
        wrong_block |= !in && t0 + k < total_new;
        slot[k] = in ? (blk[k] << shift) + (where[k] & mask) : -1;
      }
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        slot[k] = -1;
        where[k] = 0;
      }
    }
    if (PER == 4 && wide && t64 + 4 <= p.max_tokens) {
      *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1 % PER], slot[2 % PER], slot[3 % PER]);
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(where[0], where[1 % PER], where[2 % PER], where[3 % PER]);
    } else {
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (t64 + k < p.max_tokens) {
          p.slots[t0 + k] = slot[k];
          p.positions[t0 + k] = where[k];
        }
    }
  }
  return wrong_block;
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
  bool wrong_block = p.max_tokens > n_cta * kPlanThreads ? plan_rows<4>(p, s_cached, s_cu, s_need, head_at, rank, n_cta)
                                                         : plan_rows<1>(p, s_cached, s_cu, s_need, head_at, rank, n_cta);
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

__device__ __forceinline__ void load8(const float* w, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(w)), b = __ldg(reinterpret_cast<const float4*>(w) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// One head vector: this lane's sixteen channels (lo: 8l .., hi: 64 + 8l ..) normalised
// with weights w (null: not) and turned by cs, rounded in place.  The eight lanes of a
// vector run it together.
template <bool F16, int ROPE>
__device__ __forceinline__ void store_vec(uint4& lo, uint4& hi, const float* w, float eps, const float2 (&cs)[8]) {
  const int l = threadIdx.x & 7;
  float x[16];
  const uint32_t* a = reinterpret_cast<const uint32_t*>(&lo);
  const uint32_t* b = reinterpret_cast<const uint32_t*>(&hi);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unpack2<F16>(a[i], x[2 * i], x[2 * i + 1]);
    unpack2<F16>(b[i], x[8 + 2 * i], x[9 + 2 * i]);
  }
  if (w) {
    float w0[8], w1[8];
    load8(w + l * 8, w0);
    load8(w + 64 + l * 8, w1);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
    const unsigned lanes = 0xFFu << (threadIdx.x & 24);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
    const float rs = rsqrtf(ss * (1.0f / 128.0f) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] *= rs * w0[i];
      x[8 + i] *= rs * w1[i];
    }
  }
  if (ROPE == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = x[i], v = x[8 + i];
      x[i] = u * cs[i].x - v * cs[i].y;
      x[8 + i] = u * cs[i].y + v * cs[i].x;
    }
  } else if (ROPE == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = x[2 * i], v = x[2 * i + 1];
      x[2 * i] = u * cs[i].x - v * cs[i].y;
      x[2 * i + 1] = u * cs[i].y + v * cs[i].x;
    }
  }
  lo = make_uint4(pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(x[4], x[5]), pack2<F16>(x[6], x[7]));
  hi = make_uint4(pack2<F16>(x[8], x[9]), pack2<F16>(x[10], x[11]), pack2<F16>(x[12], x[13]), pack2<F16>(x[14], x[15]));
}

// cos and sin of pair i at `pos`: the angle in turns and in 64 bits, its fraction kept.
__device__ __forceinline__ float2 store_angle(const KvStoreArgs& p, int pos, int i) {
  const double u = static_cast<double>(pos) * p.turns[i];
  const float f = static_cast<float>(u - rint(u));
  float sn, cs;
  sincospif(2.0f * f, &sn, &cs);
  return make_float2(cs, sn);
}

// This lane's eight pairs: 8l .. (half-split), or 4l .. of the low and 32 + 4l .. of the
// high half (neighbours).
template <int ROPE>
__device__ __forceinline__ void store_pairs(const float2* s_cs, float2 (&cs)[8]) {
  const int l = threadIdx.x & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = s_cs[ROPE == 2 ? l * 8 + i : (i < 4 ? l * 4 + i : 28 + l * 4 + i)];
}

// Where vector `vec` of token t goes (this lane's part of its low half).
__device__ __forceinline__ uint16_t* store_dst(const KvStoreArgs& p, int64_t t, int slot, int vec) {
  const int l = threadIdx.x & 7, n_qk = p.heads + p.heads_kv;
  if (vec < p.heads) return p.q + t * p.ld_q + vec * 128 + l * 8;
  const int64_t blk = slot >> p.block_shift, off = slot & ((1 << p.block_shift) - 1);
  const int h = vec < n_qk ? vec - p.heads : vec - n_qk;
  return (vec < n_qk ? p.k : p.v) + blk * p.block_stride + ((static_cast<int64_t>(h) << p.block_shift) + off) * 128 + l * 8;
}

// Few tokens: one CTA per token, what counts is the chain of loads.  The first vectors
// are on their way before the slot that says where they go is known.  Measured, 48 head
// vectors a token: 64 tokens 3.2 us, 2048 tokens 15.0 us (3.4 TB/s, read and written).
template <bool F16, int ROPE>
__global__ void __launch_bounds__(kStoreThreads) kv_store_kernel(const __grid_constant__ KvStoreArgs p) {
  __shared__ float2 s_cs[64];
  const int t = blockIdx.x;
  const int l = threadIdx.x & 7, vec0 = threadIdx.x >> 3;
  constexpr int kPerPass = kStoreThreads / 8;
  const int n_qk = p.heads + p.heads_kv, n_vec = n_qk + p.heads_kv;
  const uint16_t* src = p.qkv + t * p.ld_qkv + l * 8;
  uint4 lo[kStoreVecs], hi[kStoreVecs];
  auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < kStoreVecs; ++j) {
      const int vec = base + j * kPerPass + vec0;
      if (vec < n_vec) {
        lo[j] = *reinterpret_cast<const uint4*>(src + vec * 128);
        hi[j] = *reinterpret_cast<const uint4*>(src + vec * 128 + 64);
      }
    }
  };
  load(0);
  const int slot = p.slots[t];
  if (ROPE != 0 && threadIdx.x < 64) s_cs[threadIdx.x] = store_angle(p, p.positions[t], threadIdx.x);
  if (slot < 0 || slot >= p.n_slots) {  // the whole block
    if (slot >= 0 && threadIdx.x == 0) record_error(p.err, kDevBadCache);
    return;
  }
  float2 cs[8];
  if (ROPE != 0) {
    __syncthreads();
    store_pairs<ROPE>(s_cs, cs);
  }
  for (int base = 0; base < n_vec; base += kPerPass * kStoreVecs) {
    if (base > 0) load(base);
#pragma unroll
    for (int j = 0; j < kStoreVecs; ++j) {
      const int vec = base + j * kPerPass + vec0;
      if (vec >= n_vec) continue;  // the eight lanes of a vector agree
      if (vec < n_qk) store_vec<F16, ROPE>(lo[j], hi[j], vec < p.heads ? p.norm_q : p.norm_k, p.eps, cs);
      uint16_t* dst = store_dst(p, t, slot, vec);
      *reinterpret_cast<uint4*>(dst) = lo[j];
      *reinterpret_cast<uint4*>(dst + 64) = hi[j];
    }
  }
}

// Many tokens: one CTA of 24 warps per SM, each warp walks tokens by itself, a row in
// slices of up to 16 vectors, with two slice buffers in shared memory: the next slice
// arrives as one bulk copy while this one is computed.  (CTAs that load, compute and
// store in turn leave the memory idle between: 66 us for 16.3k tokens of 36 heads; 11
// warps with whole rows too few instructions in flight: 63 us; this takes 57 us, 4.8 TB/s.)
constexpr int kStreamWarps = 24;
constexpr int kSliceVecs = 16;
constexpr int kStreamSmem = kStreamWarps * 2 * kSliceVecs * 256;  // 192 KB

template <bool F16, int ROPE>
__global__ void __launch_bounds__(kStreamWarps * 32, 1)
    kv_store_stream_kernel(const __grid_constant__ KvStoreArgs p, int slices, int slice_vecs) {
  extern __shared__ __align__(128) uint8_t stream_smem[];
  __shared__ uint64_t s_full[kStreamWarps][2];
  __shared__ float2 s_angles[kStreamWarps][64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 7;
  const int n_qk = p.heads + p.heads_kv, n_vec = n_qk + p.heads_kv;
  uint8_t* buf = stream_smem + warp * (2 * kSliceVecs * 256);
  uint64_t* full = s_full[warp];
  float2* s_cs = s_angles[warp];
  if (lane == 0) {
    mbar_init(&full[0], 1);
    mbar_init(&full[1], 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int stride = gridDim.x * kStreamWarps;
  int t = blockIdx.x * kStreamWarps + warp;
  if (t >= p.tokens) return;
  // Slice s of row t into buffer b.
  auto fetch = [&](int64_t row, int s, int b) {
    const uint32_t bytes = static_cast<uint32_t>(min(slice_vecs, n_vec - s * slice_vecs)) * 256;
    mbar_arrive_expect_tx(&full[b], bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(buf + b * (kSliceVecs * 256))),
                 "l"(p.qkv + row * p.ld_qkv + s * slice_vecs * 128), "r"(bytes), "r"(smem_u32(&full[b]))
                 : "memory");
  };
  if (lane == 0) fetch(t, 0, 0);
  int slot = p.slots[t], pos = ROPE != 0 ? p.positions[t] : 0;
  int slot_next = -1, pos_next = 0;
  float2 cs[8];
  for (int k = 0, s = 0;; ++k) {
    const int b = k & 1;
    const bool row_ends = s + 1 == slices;
    const int64_t next = row_ends ? static_cast<int64_t>(t) + stride : t;
    const bool more = next < p.tokens;
    if (more && lane == 0) fetch(next, row_ends ? 0 : s + 1, b ^ 1);  // read by all lanes before the last __syncwarp
    if (s == 0) {
      const int64_t after = static_cast<int64_t>(t) + stride;
      if (after < p.tokens) {
        slot_next = p.slots[after];
        if (ROPE != 0) pos_next = p.positions[after];
      }
      if (ROPE != 0) {
        s_cs[lane] = store_angle(p, pos, lane);
        s_cs[lane + 32] = store_angle(p, pos, lane + 32);
        __syncwarp();
        store_pairs<ROPE>(s_cs, cs);
      }
    }
    const bool ok = kv_wait_warp(&full[b], (k >> 1) & 1, p.err);
    if (ok && slot >= 0 && slot < p.n_slots) {
      const uint8_t* row = buf + b * (kSliceVecs * 256) + l * 16;
      const int end = min(slice_vecs, n_vec - s * slice_vecs);
#pragma unroll 2
      for (int v = lane >> 3; v < end; v += 4) {  // the eight lanes of a vector agree
        const int vec = s * slice_vecs + v;
        uint4 lo = *reinterpret_cast<const uint4*>(row + v * 256);
        uint4 hi = *reinterpret_cast<const uint4*>(row + v * 256 + 128);
        if (vec < n_qk) store_vec<F16, ROPE>(lo, hi, vec < p.heads ? p.norm_q : p.norm_k, p.eps, cs);
        uint16_t* dst = store_dst(p, t, slot, vec);
        *reinterpret_cast<uint4*>(dst) = lo;
        *reinterpret_cast<uint4*>(dst + 64) = hi;
      }
    } else if (slot >= p.n_slots && s == 0 && lane == 0) {
      record_error(p.err, kDevBadCache);
    }
    fence_proxy_async_smem();  // this slice has been read before the buffer is filled again
    __syncwarp();
    if (!more) return;
    if (row_ends) {
      t = static_cast<int>(next);
      slot = slot_next;
      pos = pos_next;
      s = 0;
    } else {
      ++s;
    }
  }
}

template <bool F16, int ROPE>
cudaError_t launch_store(const KvStoreArgs& a, int num_sms, cudaStream_t s) {
  const int vecs = a.heads + 2 * a.heads_kv;
  if (a.tokens >= 2 * kStreamWarps * num_sms) {  // measured: 2048 tokens 14.3 us one by one, 16.6 us so; 16.3k tokens 66 and 57 us
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(kv_store_stream_kernel<F16, ROPE>, kStreamSmem, done);
    if (e != cudaSuccess) return e;
    const int slices = (vecs + kSliceVecs - 1) / kSliceVecs;
    const int slice_vecs = ((vecs + slices - 1) / slices + 3) / 4 * 4;  // four vectors to a pass of a warp
    kv_store_stream_kernel<F16, ROPE><<<num_sms, kStreamWarps * 32, kStreamSmem, s>>>(
        a, (vecs + slice_vecs - 1) / slice_vecs, slice_vecs);
  } else {
    kv_store_kernel<F16, ROPE><<<a.tokens, kStoreThreads, 0, s>>>(a);
  }
  return cudaGetLastError();
}

template <bool F16>
cudaError_t launch_store_t(const KvStoreArgs& a, int num_sms, cudaStream_t s) {
  switch (a.rope) {
    case 0: return launch_store<F16, 0>(a, num_sms, s);
    case 1: return launch_store<F16, 1>(a, num_sms, s);
    default: return launch_store<F16, 2>(a, num_sms, s);
  }
}

}  // namespace

cudaError_t launch_kv_plan(const KvPlanArgs& a, cudaStream_t s) {
  if (a.batch < 1 || a.batch > kKvMaxPlanBatch) return cudaErrorInvalidValue;
  const size_t smem = (static_cast<size_t>(a.batch) * 4 + 3) * sizeof(int32_t);
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(kv_plan_kernel, (kKvMaxPlanBatch * 4 + 3) * sizeof(int32_t), done);
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

cudaError_t launch_kv_store(const KvStoreArgs& a, bool f16, int num_sms, cudaStream_t s) {
  if (a.tokens <= 0) return cudaSuccess;
  return f16 ? launch_store_t<true>(a, num_sms, s) : launch_store_t<false>(a, num_sms, s);
}

}  // namespace dcpp
