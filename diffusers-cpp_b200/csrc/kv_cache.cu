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
// first 64 threads, as fractions of a turn in 64-bit fixed point (the product with
// the position wraps, which drops whole turns; what is left is off by position *
// 2^-55 turns, so a far position is as good as a near one), then cos and sin of
// [-1/2, 1/2] turn.  Sums and the rotation are f32 (two values an instruction),
// rounded once to the cache's type.
constexpr int kStoreThreads = 128;
constexpr int kStoreVecs = 3;

// Two packed values as a pair of f32 (lanes of a 64-bit register, for f32x2 arithmetic).
template <bool F16>
__device__ __forceinline__ uint64_t unpack2(uint32_t u) {
  if constexpr (F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    return f2(f.x, f.y);
  } else {
    return (static_cast<uint64_t>(u & 0xFFFF0000u) << 32) | (u << 16);
  }
}

// This lane's rotations: 8l .. and their partners 64 + 8l .. (half-split), or the pairs
// 4l .. of the low and 32 + 4l .. of the high half (neighbours).
template <int ROPE>
struct StoreTurn {
  // Half-split: cosines, and sines, of two neighbouring channels.  Neighbours: (cos, cos) and
  // (-sin, sin) of a pair.
  uint64_t c[ROPE == 2 ? 4 : 8], s[ROPE == 2 ? 4 : 8];
  __device__ __forceinline__ void load(const float2* s_cs) {
    const int l = threadIdx.x & 7;
    if constexpr (ROPE == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = s_cs[l * 8 + 2 * i], b = s_cs[l * 8 + 2 * i + 1];
        c[i] = f2(a.x, b.x);
        s[i] = f2(a.y, b.y);
      }
    } else if constexpr (ROPE == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 a = s_cs[i < 4 ? l * 4 + i : 28 + l * 4 + i];
        c[i] = f2(a.x, a.x);
        s[i] = f2(-a.y, a.y);
      }
    }
  }
};

// One head vector: this lane's sixteen channels (lo: 8l .., hi: 64 + 8l ..) normalised
// with weights w (null: not) and turned, rounded in place.  The eight lanes of a vector
// run it together.
template <bool F16, int ROPE>
__device__ __forceinline__ void store_vec(uint4& lo, uint4& hi, const float* w, float eps, const StoreTurn<ROPE>& turn) {
  const int l = threadIdx.x & 7;
  uint64_t x[8];  // pairs of channels: four of the low, four of the high half
  const uint32_t* a = reinterpret_cast<const uint32_t*>(&lo);
  const uint32_t* b = reinterpret_cast<const uint32_t*>(&hi);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = unpack2<F16>(a[i]);
    x[4 + i] = unpack2<F16>(b[i]);
  }
  if (w) {
    const ulonglong2* wl = reinterpret_cast<const ulonglong2*>(w + l * 8);
    const ulonglong2* wh = reinterpret_cast<const ulonglong2*>(w + 64 + l * 8);
    const ulonglong2 w0 = __ldg(wl), w1 = __ldg(wl + 1), w2 = __ldg(wh), w3 = __ldg(wh + 1);
    const uint64_t wv[8] = {w0.x, w0.y, w1.x, w1.y, w2.x, w2.y, w3.x, w3.y};
    uint64_t q0 = 0, q1 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q0 = fma2(x[i], x[i], q0);
      q1 = fma2(x[4 + i], x[4 + i], q1);
    }
    q0 = add2(q0, q1);
    float ss = f2lo(q0) + f2hi(q0);
    const unsigned lanes = 0xFFu << (threadIdx.x & 24);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
    const float rs = rsqrtf(ss * (1.0f / 128.0f) + eps);
    const uint64_t rs2 = f2(rs, rs);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = mul2(x[i], mul2(rs2, wv[i]));
  }
  if constexpr (ROPE == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t u = x[i], v = x[4 + i];
      x[i] = fma2(mul2(v, turn.s[i]), f2(-1.0f, -1.0f), mul2(u, turn.c[i]));
      x[4 + i] = fma2(u, turn.s[i], mul2(v, turn.c[i]));
    }
  } else if constexpr (ROPE == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fma2(x[i], turn.c[i], mul2(f2(f2hi(x[i]), f2lo(x[i])), turn.s[i]));
  }
  uint32_t y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = kv_pack2<F16>(f2lo(x[i]), f2hi(x[i]));
  lo = make_uint4(y[0], y[1], y[2], y[3]);
  hi = make_uint4(y[4], y[5], y[6], y[7]);
}

// cos and sin of pair i at `pos`: the angle as a 64-bit fraction of a turn, its whole
// turns dropped by wrapping around.
__device__ __forceinline__ float2 store_angle(const KvStoreArgs& p, int pos, int i) {
  const uint64_t u = static_cast<uint64_t>(static_cast<int64_t>(pos)) * p.turns[i];
  float sn, cs;
  sincospif(static_cast<float>(static_cast<int32_t>(u >> 32)) * 0x1p-31f, &sn, &cs);
  return make_float2(cs, sn);
}

// Where a token's vectors go (this lane's part of their low halves).
struct StoreDst {
  uint16_t *q, *k, *v;
  int64_t head;  // elements between the heads of a block
  __device__ __forceinline__ StoreDst(const KvStoreArgs& p, int64_t t, int slot) {
    const int l = threadIdx.x & 7;
    const int64_t at = static_cast<int64_t>(slot >> p.block_shift) * p.block_stride + (slot & ((1 << p.block_shift) - 1)) * 128 + l * 8;
    head = 128 << p.block_shift;
    q = p.q + t * p.ld_q + l * 8;
    // By the vector's number in the row.
    k = p.k + at - p.heads * head;
    v = p.v + at - (p.heads + p.heads_kv) * head;
  }
  __device__ __forceinline__ uint16_t* of(const KvStoreArgs& p, int vec) const {
    return vec < p.heads ? q + vec * 128 : (vec < p.heads + p.heads_kv ? k : v) + vec * head;
  }
};

// Few tokens: one CTA per token, what counts is the chain of loads.  The first vectors
// are on their way before the slot that says where they go is known.  Measured, 48 head
// vectors a token: 64 tokens 3.1 us, 1024 tokens 7.2 us (3.5 TB/s, read and written).
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
  StoreTurn<ROPE> turn;
  if (ROPE != 0) {
    __syncthreads();
    turn.load(s_cs);
  }
  const StoreDst to(p, t, slot);
  for (int base = 0; base < n_vec; base += kPerPass * kStoreVecs) {
    if (base > 0) load(base);
#pragma unroll
    for (int j = 0; j < kStoreVecs; ++j) {
      const int vec = base + j * kPerPass + vec0;
      if (vec >= n_vec) continue;  // the eight lanes of a vector agree
      if (vec < n_qk) store_vec<F16, ROPE>(lo[j], hi[j], vec < p.heads ? p.norm_q : p.norm_k, p.eps, turn);
      uint16_t* dst = to.of(p, vec);
      *reinterpret_cast<uint4*>(dst) = lo[j];
      *reinterpret_cast<uint4*>(dst + 64) = hi[j];
    }
  }
}

// Many tokens: one CTA of 16 warps per SM, each warp walks tokens by itself, a row in
// slices of up to 16 vectors, with two slice buffers in shared memory: the next slice
// arrives as one bulk copy while this one is computed.  Bound by HBM for wide rows, by
// the instructions for narrow ones (hence two f32 values to an
// instruction, and addresses once a token).  Measured: 2048 tokens of 48 vectors 12.4 us
// (4.1 TB/s), 16.3k 68.7 us (5.8 TB/s), 16.3k of 36 in f16 56 us, 40k of 12 58 us; 24
// warps leave too few registers (15.2, 76, 63 and 64 us); three or more buffers are no
// faster.
constexpr int kStreamWarps = 16;
constexpr int kSliceVecs = 16;
constexpr int kStreamSmem = kStreamWarps * 2 * kSliceVecs * 256;  // 128 KB

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
  int t = warp * gridDim.x + blockIdx.x;  // neighbouring tokens on different SMs: few tokens fill all of them
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
  StoreTurn<ROPE> turn;
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
        turn.load(s_cs);
      }
    }
    if (!kv_wait_warp(&full[b], (k >> 1) & 1, p.err)) {
      // A barrier whose copy has not landed must not be armed again: no more work, but the
      // other copy has its own time to land.
      if (more) kv_wait_warp(&full[b ^ 1], ((k + 1) >> 1) & 1, p.err);
      return;
    }
    if (slot >= 0 && slot < p.n_slots) {
      const StoreDst to(p, t, slot);
      const uint8_t* row = buf + b * (kSliceVecs * 256) + l * 16;
      const int end = min(slice_vecs, n_vec - s * slice_vecs);
#pragma unroll 2
      for (int v = lane >> 3; v < end; v += 4) {  // the eight lanes of a vector agree
        const int vec = s * slice_vecs + v;
        uint4 lo = *reinterpret_cast<const uint4*>(row + v * 256);
        uint4 hi = *reinterpret_cast<const uint4*>(row + v * 256 + 128);
        if (vec < n_qk) store_vec<F16, ROPE>(lo, hi, vec < p.heads ? p.norm_q : p.norm_k, p.eps, turn);
        uint16_t* dst = to.of(p, vec);
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
  // Measured, one by one / so: 1024 tokens of 48 vectors 7.2 / 7.8 us, 1500 10.9 / 9.9 us, 16.3k
  // 80 / 69 us; 4096 of 10 12.1 / 8.1 us.
  if (a.tokens >= kStreamWarps / 2 * num_sms) {
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
