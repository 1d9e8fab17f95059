// Attention over the paged cache for many query rows, on the 5th-generation
// tensor cores (tcgen05 + TMEM + TMA).
//
// A unit is two tiles of up to 128 query rows (tokens x the heads of a key /
// value group) of one request and key / value head; CTAs (one per SM) walk their
// run of (unit, key tile) steps.  352 threads:
//   warp 0      TMA: Q of a unit, then K_j, V_j (128 keys, gathered block by block)
//               into two 64 KB slots
//   warps 1, 10 the MMAs of tile A and of tile B, one thread each (a wait that is
//               already met costs some 80 cycles; one thread for both tiles spent
//               more time in its eight waits per step than the tensor core in its
//               products)
//   warps 2-5   softmax of tile A, warps 6-9 of tile B: one thread per row
// A step is 64 keys.  Scores and numerators have TMEM of their own, so that neither
// product waits for the other: the scores' buffer is free again as soon as the
// softmax warps have them in registers, and S(i + 1) is computed while they work on
// step i; the numerators have two buffers, and P V of step i runs while they work on
// step i + 1.  (Scores in two buffers with P written back over them, the layout that
// holds one more step of scores, made S(i + 2) wait for P V(i): a chain of some 2100
// cycles a step where the softmax needs 1500 and the tensor core 1280.)
// V stays as the cache holds it, keys x channels: the P V product takes it as an
// operand whose rows run along the channels (MN-major), so no transposed copy of the
// cache is kept.
// Measured in a graph, 32 heads over 8: two prompts of 8k tokens 940 to 1030 us (1020 to 1120
// TFLOP/s; the products alone take some 775 us, the softmax alone 870 us), 512 tokens
// over 32k keys 255 us (1070 TFLOP/s), 4 prompts of 301 to 512 tokens 20 to 26 us
// (launch, first loads and last stores of two units for most CTAs); 16 heads over 2, 16
// requests of 5 tokens over 700 to 4000 keys 19 to 21 us.  Called back to back for a tenth of
// a second the power cap lowers the clock: 1050 us (1000 TFLOP/s) and 301 us (904 TFLOP/s).
// TMEM (512 columns): tile X at 128 X: S 0 .. 63, P 64 and 96; O_A 256, O_B 384.
#include "kv_device.cuh"
#include "kv_form.cuh"
#include "kv_sched.cuh"

#include <algorithm>

namespace dcpp {

namespace {

constexpr int kTThreads = 352;
constexpr int kTSlots = 2;                // tiles of K and V in flight
constexpr int kTHalf = 128 * 128;         // 128 rows x 64 channels: 16 KB
constexpr int kTTile = 2 * kTHalf;        // 128 x 128: 32 KB
constexpr int kTStage = 32 * 128;         // 128 bytes of a warp's rows
constexpr int kTSmem = (2 + 2 * kTSlots) * kTTile + 1024;
constexpr int kTSmemOut = kTSmem + 8 * kTStage;  // with the rows on their way out (in clusters they meet in the operands' place)
constexpr int kTLd = 132;                 // f32 row of sums in shared memory, padded: stores without bank conflicts
static_assert(kTcRows * kTLd * 4 <= (2 + 2 * kTSlots) * kTTile, "sums of a unit in place of its operands");
constexpr float kTRescale = 8.0f;         // log2 units a row maximum may grow before O is rescaled
// Lift of the numerators (see kv_attention.cu): with the growth at most 14 in f16, two bits
// below its largest value.  (A growth of 4 and a lift of 10 rescale more often: 16 requests
// of 5 tokens 23.5 instead of 20.4 us.)
template <bool F16>
constexpr float kTLift = F16 ? 6.0f : 0.0f;

struct TcBars {
  uint64_t q_full, q_empty;                // empty barriers: one arrival from each MMA thread
  uint64_t full[2][kTSlots], empty[2][kTSlots];  // [K, V][slot]
  uint64_t s_full[2], s_free[2];           // [tile] scores computed; read (4 warps)
  uint64_t p_full[2][2], pv_done[2][2];    // [tile][buffer] P written (4 warps); P read, O current
};

// Instruction descriptor: M 128, N columns, f32 accumulator, both operands of the
// cache's type; B_MN: the B operand's rows run along N.
template <bool F16, int N, bool B_MN>
__host__ __device__ constexpr uint32_t tc_idesc() {
  return (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (B_MN ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | ((128u >> 4) << 24);
}

// Descriptor of a 128-byte-swizzled operand whose rows (64 channels each) run
// along N and whose K steps go down the rows: 8-row groups 1024 bytes apart, the
// second 64 channels kTHalf further on.
__device__ __forceinline__ uint64_t tc_desc_mn(uint32_t addr) {
  uint64_t d = static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(kTHalf >> 4) << 16;  // between 64-channel atoms
  d |= static_cast<uint64_t>(1024u >> 4) << 32;   // between groups of 8 keys
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;           // SWIZZLE_128B
  return d;
}

// The MMA warps' instructions, issued by the one lane whose `leader` is set; barriers
// by their shared-memory address.
__device__ __forceinline__ void tc_mma_ss(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t phase, int* err) {
  return kv_wait_warp(bar, phase & 1, err);
}

// What tile x of a CTA does with the unit at `at`, whose key tiles [first, last) are the
// CTA's: n_tok tokens, and the steps of 64 keys from 2 first up to end.
struct TcWork {
  int first, last;
  int end;
  int tok0, n_tok;  // first token of the unit, tokens of the tile
  bool two;         // the unit has a tile B
};

__device__ __forceinline__ TcWork tc_work(const KvAttnArgs& p, const KvPos& at, int64_t left, int x) {
  TcWork w;
  const int half = p.unit_tokens / 2;
  w.first = at.tile;
  w.last = at.tile + static_cast<int>(min(left, static_cast<int64_t>(at.n_tiles - at.tile)));
  w.tok0 = at.u * p.unit_tokens;
  const int n = min(p.unit_tokens, at.s.q_len - w.tok0);
  w.two = n > half;
  w.n_tok = min(max(n - x * half, 0), half);
  int keys = at.s.kv;
  if (p.causal) keys = min(keys, at.s.off + w.tok0 + x * half + w.n_tok);
  const int steps = w.n_tok > 0 ? max(1, (keys + 63) >> 6) : 0;
  w.end = max(2 * w.first, min(2 * w.last, steps));
  return w;
}

// Eight f32 values times `by`, rounded to the output's type.
template <bool F16>
__device__ __forceinline__ uint4 tc_pack8(const uint32_t* r, float by) {
  return make_uint4(kv_pack2<F16>(__uint_as_float(r[0]) * by, __uint_as_float(r[1]) * by),
                    kv_pack2<F16>(__uint_as_float(r[2]) * by, __uint_as_float(r[3]) * by),
                    kv_pack2<F16>(__uint_as_float(r[4]) * by, __uint_as_float(r[5]) * by),
                    kv_pack2<F16>(__uint_as_float(r[6]) * by, __uint_as_float(r[7]) * by));
}

struct TcState {
  KvPos at;
  int64_t left;
  int tiles;  // key tiles of the runs before this one
};

// Joins a unit whose key tiles the CTAs of a cluster shared: every CTA's numerators
// (rows of kTLd f32) and (maximum, sum) lie in its shared memory, and each CTA adds up
// every cluster-th row, a warp 8 / cluster rows at a time, so that eight loads are on
// their way together.  Rows of a unit in order of (token, head): tile B follows tile
// A's half_rows.
template <bool F16>
__device__ __forceinline__ void tc_join_cluster(const KvAttnArgs& p, const KvPos& at, uint32_t sums, uint32_t ml, int cluster,
                                                int rank) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half_rows = p.unit_tokens / 2 * p.group, tok0 = at.u * p.unit_tokens;
  const int rows = min(p.unit_tokens, at.s.q_len - tok0) * p.group;
  const int per = 8 / cluster, shift = 31 - __clz(cluster);
  for (int r0 = rank * per + warp * per * cluster; r0 < rows; r0 += kTThreads / 32 * per * cluster) {
    // Slot q: row r0 + q / cluster in CTA q % cluster.
    const int q = lane & 7, r = min(r0 + (q >> shift), rows - 1);
    const int at_row = r < half_rows ? r : 128 + r - half_rows;
    const float2 v = ld_cluster2(mapa_shared(ml + at_row * 8, q & (cluster - 1)));
    float4 a[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      a[k] = ld_cluster4(mapa_shared(sums + __shfl_sync(0xffffffffu, at_row, k) * (kTLd * 4) + lane * 16, k & (cluster - 1)));
    float M = v.x;
    for (int o = cluster >> 1; o > 0; o >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, o));
    float w = v.x == -INFINITY ? 0.f : ex2(v.x - M);
    float L = w * v.y;
    for (int o = cluster >> 1; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    w = L != 0.f ? w / L : 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      if (wk != 0.f) {  // a part of weight 0 has not written its sums
        s.x = fmaf(wk, a[k].x, s.x); s.y = fmaf(wk, a[k].y, s.y);
        s.z = fmaf(wk, a[k].z, s.z); s.w = fmaf(wk, a[k].w, s.w);
      }
      if (((k + 1) & (cluster - 1)) == 0) {
        const int row = r0 + (k >> shift);
        if (row < rows) {
          const int tok = p.row_token(row), head = row - tok * p.group;
          uint16_t* dst = p.out + static_cast<int64_t>(at.s.q0 + tok0 + tok) * p.ld_out +
                          (static_cast<int64_t>(at.h) * p.group + head) * 128 + lane * 4;
          *reinterpret_cast<uint2*>(dst) = make_uint2(kv_pack2<F16>(s.x, s.y), kv_pack2<F16>(s.z, s.w));
        }
        s = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
}

template <bool F16, bool CLUSTER>
__global__ void __launch_bounds__(kTThreads, 1)
    kv_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ KvAttnArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                // tile A | tile B
  uint8_t* sKV = smem + 2 * kTTile;  // kTSlots slots
  __shared__ TcBars bar;
  __shared__ uint32_t tmem_slot;
  __shared__ TcState state[8];
  __shared__ KvSchedSmem<kTThreads> sched;
  __shared__ float2 s_ml[CLUSTER ? kTcRows : 1];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_empty, 2);
    for (int i = 0; i < kTSlots; ++i)
      for (int kv = 0; kv < 2; ++kv) {
        mbar_init(&bar.full[kv][i], 1);
        mbar_init(&bar.empty[kv][i], 2);
      }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bar.s_full[x], 1);
      mbar_init(&bar.s_free[x], 4);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bar.p_full[x][b], 4);
        mbar_init(&bar.pv_done[x][b], 1);
      }
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  KvRange range;
  KvPos at;
  // The direct form: one unit for each CTA, or for each cluster, whose CTAs share its key
  // tiles and join their sums through shared memory.
  const int cluster = CLUSTER ? cluster_size() : 1, rank = CLUSTER ? static_cast<int>(cluster_ctarank()) : 0;
  int64_t left = CLUSTER || p.direct ? kv_direct<kTcKT>(p, cluster, rank, at) : kv_share<kTcKT, kTThreads, kTcMinTiles>(p, sched, range, at);
  const bool no_unit = left < 0;
  left = max(left, static_cast<int64_t>(0));
  // The producer's block ids come from the table 32 at a time, the next 32 fetched ahead;
  // those of the first tile are on their way while the CTA sets up.
  int cur = -1, nxt = -1;
  auto fetch = [&](int i) { return i < p.max_blocks ? __ldg(p.table + at.b * p.max_blocks + i) : -1; };
  auto fetch_first = [&] {
    const int win = (at.tile * kTcKT) >> p.block_shift;
    cur = fetch(win + lane);
    nxt = fetch(win + 32 + lane);
  };
  if (warp == 0 && left > 0) fetch_first();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!CLUSTER && threadIdx.x == 0 && !p.direct) kv_write_cut(p, range, at, left > 0, blockIdx.x);
  const uint32_t tmem = tmem_slot;
  const int half_tok = p.unit_tokens / 2;

  if (warp == 0) {
    const int boxes = kTcKT / p.box_rows;
    const int box = lane & (boxes - 1), half = lane / boxes;
    const int bs_mask = (1 << p.block_shift) - 1;
    const uint32_t q_bytes = 2u * 128u * static_cast<uint32_t>(half_tok * p.group);
    int it = 0, unit = 0;          // key tiles and units so far
    int issued[2] = {0, 0};        // copies of K and of V
    bool ok = true;
    while (left > 0 && ok) {
      const TcWork w = tc_work(p, at, left, 0);
      ok = kv_wait_warp(&bar.q_empty, (unit & 1) ^ 1, p.err);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar.q_full, w.two ? 2 * q_bytes : q_bytes);
        for (int x = 0; x < 2; ++x)
          if (x == 0 || w.two)
            for (int k = 0; k < 2; ++k)
              tma_load_3d(sQ + x * kTTile + k * kTHalf, &tmQ, &bar.q_full, k * 64, at.h * p.group,
                          at.s.q0 + w.tok0 + x * half_tok);
      }
      __syncwarp();
      ++unit;
      int win = (w.first * kTcKT) >> p.block_shift;
      for (int j = w.first; j < w.last && ok; ++j) {
        const int key0 = j * kTcKT + box * p.box_rows;
        const int idx = key0 >> p.block_shift;
        if (__shfl_sync(0xffffffffu, idx, 0) - win >= 32) {  // a tile's boxes never straddle a window
          win += 32;
          cur = nxt;
          nxt = fetch(win + 32 + lane);
        }
        const int blk = __shfl_sync(0xffffffffu, cur, idx - win);
        const bool load = half < 2 && key0 < at.s.kv;
        const bool wrong = blk < 0 || blk >= p.n_blocks;
        if (load && wrong) record_error(p.err, kDevBadCache);
        const int c3 = wrong ? p.n_blocks : blk;  // one past the end: TMA fills zeros
        const int loads = __popc(__ballot_sync(0xffffffffu, load));
        const int st = it & 1;
        for (int kv = 0; kv < 2 && ok; ++kv) {  // K_j, then V_j
          ok = kv_wait_warp(&bar.empty[kv][st], ((it >> 1) & 1) ^ 1, p.err);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&bar.full[kv][st], loads * p.box_rows * 128);
          __syncwarp();
          if (load)
            tma_load_4d(sKV + (2 * st + kv) * kTTile + half * kTHalf + box * p.box_rows * 128, kv ? &tmV : &tmK,
                        &bar.full[kv][st], half * 64, key0 & bs_mask, at.h, c3);
          issued[kv] = it + 1;
        }
        ++it;
      }
      left -= w.last - w.first;
      if (left > 0) {
        if (!kv_next_unit<kTcKT>(p, at)) break;
        fetch_first();
      }
    }
    // Nothing may be in flight when the CTA ends: all copies landed, and (unless a
    // wait ran out) every slot handed back, i.e. the last commits have arrived.
    bool landed = unit == 0 || kv_wait(&bar.q_full, (unit - 1) & 1, p.err);
    for (int kv = 0; kv < 2; ++kv)
      for (int k = max(0, issued[kv] - kTSlots); k < issued[kv]; ++k)
        landed &= kv_wait(&bar.full[kv][k & 1], (k >> 1) & 1, p.err);
    if (ok && landed && unit > 0) {
      for (int kv = 0; kv < 2; ++kv)
        for (int k = max(0, it - kTSlots); k < it; ++k) ok = ok && kv_wait(&bar.empty[kv][k & 1], (k >> 1) & 1, p.err);
      if (ok) kv_wait(&bar.q_empty, (unit - 1) & 1, p.err);
    }
  } else if (warp == 1 || warp == kTThreads / 32 - 1) {
    // The whole warp runs the loop, without a branch around the products: one elected
    // lane issues them by predicate.
    const int x = warp == 1 ? 0 : 1;
    constexpr uint32_t idS = tc_idesc<F16, 64, false>(), idPV = tc_idesc<F16, 128, true>();
    const uint64_t dQ = make_sdesc_sw128(smem_u32(sQ + x * kTTile));
    const uint64_t dK = make_sdesc_sw128(smem_u32(sKV));
    const uint64_t dV = tc_desc_mn(smem_u32(sKV + kTTile));
    // The descriptors' low words; a slot, a step or a K step only moves the address in them.
    const uint32_t hiK = static_cast<uint32_t>(dK >> 32), hiV = static_cast<uint32_t>(dV >> 32);
    const uint32_t loQ = static_cast<uint32_t>(dQ), loK = static_cast<uint32_t>(dK), loV = static_cast<uint32_t>(dV);
    constexpr uint32_t kSlotD = 2 * kTTile >> 4, kStepD = 64 * 128 >> 4;
    const uint32_t tS = tmem + x * 128, tO = tmem + 256 + x * 128;
    const uint32_t fullK = smem_u32(bar.full[0]), fullV = smem_u32(bar.full[1]);
    const uint32_t emptyK = smem_u32(bar.empty[0]), emptyV = smem_u32(bar.empty[1]);
    const uint32_t s_full = smem_u32(&bar.s_full[x]), s_free = smem_u32(&bar.s_free[x]);
    const uint32_t p_full = smem_u32(bar.p_full[x]), pv_done = smem_u32(bar.pv_done[x]), q_empty = smem_u32(&bar.q_empty);
    const uint32_t leader = elect_one_sync();
    int unit = 0, n = 0, n_s = 0;  // units; P V products and scores issued for this tile
    int tk = 0, tv = 0;            // tiles whose K, and whose V, this warp is done with
    bool ok = true;
    while (left > 0 && ok) {
      const TcWork w = tc_work(p, at, left, x);
      const int s0 = 2 * w.first, end = w.end, tiles = w.last - w.first;
      // Both sides meet every phase of every barrier in order and hand back every slot, and
      // Q, themselves, used or not: a parity wait tells a phase only from its neighbours, so
      // nothing may be filled again before both have seen it.
      if (!(ok = kv_wait_warp(&bar.q_full, unit & 1, p.err))) break;
      if (x == 1 && !w.two) {
        if (leader) mbar_arrive_at(q_empty);
        for (int k = 0; k < tiles; ++k, ++tk, ++tv) {
          if (!(ok = tc_wait(fullK + 8 * (tk & 1), tk >> 1, p.err))) break;
          if (leader) mbar_arrive_at(emptyK + 8 * (tk & 1));
          if (!(ok = tc_wait(fullV + 8 * (tv & 1), tv >> 1, p.err))) break;
          if (leader) mbar_arrive_at(emptyV + 8 * (tv & 1));
        }
        __syncwarp();
      } else {
        if (end == s0) tc_commit(leader, q_empty);
        // S(i + 1) = Q K_{i+1}^T, then O += P(i) V_i.
#pragma unroll 1
        for (int i = s0 - 1; i < end; ++i) {
          const int is = i + 1;
          if (is < end) {
            if (!(is & 1) && !(ok = tc_wait(fullK + 8 * (tk & 1), tk >> 1, p.err))) break;
            if (n_s > 0 && !(ok = tc_wait(s_free, n_s - 1, p.err))) break;
            tc_fence_after();
            const uint32_t kd = loK + (tk & 1) * kSlotD + (is & 1) * kStepD;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t off = ((k >> 2) * kTHalf + (k & 3) * 32) >> 4;
              tc_mma_ss(leader, tS, loQ + off, kd + off, hiK, idS, k > 0);
            }
            tc_commit(leader, s_full);
            if ((is & 1) || is + 1 == end) {
              tc_commit(leader, emptyK + 8 * (tk & 1));
              ++tk;
              if (is + 1 == end) tc_commit(leader, q_empty);
            }
            ++n_s;
          }
          if (i >= s0) {
            const uint32_t b = n & 1;
            if ((!(i & 1) || i == s0) && !(ok = tc_wait(fullV + 8 * (tv & 1), tv >> 1, p.err))) break;
            if (!(ok = tc_wait(p_full + 8 * b, n >> 1, p.err))) break;
            tc_fence_after();
            const uint32_t tP = tS + 64 + b * 32, vd = loV + (tv & 1) * kSlotD + (i & 1) * kStepD;
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 16 keys: 8 packed TMEM columns of P, 16 rows (2 KB) of V
              tc_mma_ts(leader, tO, tP + k * 8, vd + k * (2048 >> 4), hiV, idPV, i > s0 || k > 0);
            tc_commit(leader, pv_done + 8 * b);
            if ((i & 1) || i + 1 == end) {
              tc_commit(leader, emptyV + 8 * (tv & 1));
              ++tv;
            }
            ++n;
          }
        }
        // Tiles of the run that only the other row tile needs.
        for (int j = (end + 1) >> 1; j < w.last && ok; ++j, ++tk, ++tv) {
          if (!(ok = tc_wait(fullK + 8 * (tk & 1), tk >> 1, p.err) && tc_wait(fullV + 8 * (tv & 1), tv >> 1, p.err))) break;
          tc_commit(leader, emptyK + 8 * (tk & 1));
          tc_commit(leader, emptyV + 8 * (tv & 1));
        }
      }
      ++unit;
      left -= tiles;
      if (left > 0 && !kv_next_unit<kTcKT>(p, at)) break;
    }
  } else {
    const int x = (warp - 2) >> 2;
    const int row = (warp & 3) * 32 + lane;  // TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + x * 128, tO = tmem + lane_off + 256 + x * 128;
    const uint32_t s_full = smem_u32(&bar.s_full[x]), s_free = smem_u32(&bar.s_free[x]);
    const uint32_t p_full = smem_u32(bar.p_full[x]), pv_done = smem_u32(bar.pv_done[x]);
    const float c = p.scale_log2;
    int n = 0;  // steps done by this tile
    bool ok = true;
    // The walk's state rests in shared memory while a unit is computed: its registers
    // are needed for the scores.
    TcState& st = state[warp - 2];
    uint8_t* stage = smem + (2 + 2 * kTSlots) * kTTile + (warp - 2) * kTStage;  // 128 bytes of each row on their way out
    if (lane == 0) {
      st.at = at;
      st.left = left;
      st.tiles = 0;
    }
    __syncwarp();
    if (CLUSTER && st.left == 0) s_ml[x * 128 + row] = make_float2(-INFINITY, 0.f);  // nothing of the unit is this CTA's
    while (ok && st.left > 0) {
      int first, end, keys, limit, all_below;
      {
        const KvPos u = st.at;
        const TcWork w = tc_work(p, u, st.left, x);
        first = 2 * w.first;
        end = w.end;
        const int tile0 = u.s.off + w.tok0 + x * half_tok;  // position of the tile's first token
        keys = u.s.kv;
        limit = u.s.kv;  // keys this row attends to: [0, limit)
        if (p.causal) limit = min(limit, tile0 + p.row_token(row) + 1);
        all_below = u.s.kv;  // keys that every row of the tile attends to
        if (p.causal) all_below = min(all_below, tile0 + 1);
      }
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int i = first; i < end; ++i, ++n) {
        const int b = n & 1;
        if (!(ok = kv_wait_warp(s_full, n & 1, p.err))) break;
        tc_fence_after();
        float s[64];
        {
          uint32_t r0[32], r1[32];
          tmem_ld32(tS, r0);
          tmem_ld32(tS + 32, r1);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_at(s_free);
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            s[k] = __uint_as_float(r0[k]);
            s[32 + k] = __uint_as_float(r1[k]);
          }
        }
        const int kbase = i * 64;
        if (kbase + 64 > all_below) {
          if (kbase + 64 > keys) {
            // Behind the last key a block holds anything, and 0 x NaN is NaN: clear those
            // rows of V (both row tiles do; zeros over zeros).
            const int tile = st.tiles + (i >> 1) - (first >> 1);
            if (!(ok = kv_wait_warp(&bar.full[1][tile & 1], (tile >> 1) & 1, p.err))) break;
            uint8_t* v = sKV + (2 * (tile & 1) + 1) * kTTile + (i & 1) * 64 * 128;
#pragma unroll 1
            for (int k = max(keys - kbase, 0) * 8 + row; k < 64 * 8; k += 128) {
              *reinterpret_cast<uint4*>(v + k * 16) = make_uint4(0, 0, 0, 0);
              *reinterpret_cast<uint4*>(v + kTHalf + k * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
#pragma unroll
          for (int k = 0; k < 64; ++k)
            if (kbase + k >= limit) s[k] = -INFINITY;
        }
        float mp[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mp[k] = s[k];
#pragma unroll
        for (int k = 4; k < 64; k += 2) mp[(k >> 1) & 3] = max3_nan(mp[(k >> 1) & 3], s[k], s[k + 1]);
        const float mx = c * max_nan(max3_nan(mp[0], mp[1], mp[2]), mp[3]);
        const bool grow = mx > m + kTRescale;
        const float m_use = grow ? mx : m;
        // A stale maximum is exact (l uses the same one); without a key so far every numerator is 0.
        const float ref = m_use == -INFINITY ? 0.f : m_use;
        const float alpha = grow ? ex2(m - ref) : 1.0f;
        if (i > first && __any_sync(0xffffffffu, grow)) {
          // O has to hold every earlier step before it is rescaled.
          if (!(ok = kv_wait_warp(pv_done + 8 * (b ^ 1), ((n - 1) >> 1) & 1, p.err))) break;
          tc_fence_after();
#pragma unroll 1
          for (int ch = 0; ch < 8; ++ch) {
            uint32_t r[16];
            tmem_ld16(tO + ch * 16, r);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
            tmem_st16(tO + ch * 16, r);
          }
        }
        const uint64_t c2 = f2(c, c), nm2 = f2(kTLift<F16> - ref, kTLift<F16> - ref);
        uint64_t sp[4] = {0, 0, 0, 0};
        uint32_t pk[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const uint64_t y = fma2(f2(s[2 * k], s[2 * k + 1]), c2, nm2);
          const uint64_t e = (k & 3) == 3 ? ex2_poly2_zero(y) : f2(ex2(f2lo(y)), ex2(f2hi(y)));
          sp[k & 3] = add2(sp[k & 3], e);
          pk[k] = kv_pack2<F16>(f2lo(e), f2hi(e));
          // P V of step n - 2, which read this buffer, was issued before the scores of step n.
          if (k == 15) tmem_st16(tS + 64 + b * 32, pk);
        }
        tmem_st16(tS + 80 + b * 32, pk + 16);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(p_full + 8 * b);
        const uint64_t t = add2(add2(sp[0], sp[1]), add2(sp[2], sp[3]));
        // A score that is NaN or +inf makes the row NaN, whichever exponential it met.
        l = mx < INFINITY ? l * alpha + f2lo(t) + f2hi(t) : NAN;
        m = m_use;
      }
      if (ok && first < end) ok = kv_wait_warp(pv_done + 8 * ((n - 1) & 1), ((n - 1) >> 1) & 1, p.err);
      if (!CLUSTER && !ok) break;
      if (l != l) m = l;  // the row is NaN, not empty
      const KvPos u = st.at;
      const TcWork w = tc_work(p, u, st.left, x);
      const int tok_in = p.row_token(row), head_in = row - tok_in * p.group;
      const int tok = w.tok0 + x * half_tok + tok_in;
      const bool mine = tok_in < w.n_tok;
      if constexpr (CLUSTER) {
        if (!ok) m = -INFINITY;  // a wait ran out
        named_sync(1, 256);      // all products of the CTA are done: their operands' place is free
        s_ml[x * 128 + row] = make_float2(m, m != -INFINITY ? l : 0.f);
        tc_fence_after();
        float4* to = reinterpret_cast<float4*>(smem + (x * 128 + row) * (kTLd * 4));
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {
          uint32_t r[32];
          tmem_ld32(tO + g * 32, r);
          tmem_ld_wait();
          if (mine && m != -INFINITY)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              to[g * 8 + k] = make_float4(__uint_as_float(r[4 * k]), __uint_as_float(r[4 * k + 1]),
                                          __uint_as_float(r[4 * k + 2]), __uint_as_float(r[4 * k + 3]));
        }
        break;
      }
      const bool whole = w.first == 0 && w.last == u.n_tiles;
      // A lane holds a row; a store of one row per lane would touch 32 lines with 16
      // bytes each.  So the rows go through shared memory, 128 bytes of each at a time
      // (16-byte pieces at places ^ (row & 7): no bank conflicts), and eight lanes write
      // a row's 128 bytes together.  (Eight lanes trading their pieces by shuffles cost
      // three times the instructions: 2 us of 12 for a unit of four key tiles.)
      uint8_t* dst = nullptr;
      if (mine && whole) {
        dst = reinterpret_cast<uint8_t*>(p.out + static_cast<int64_t>(u.s.q0 + tok) * p.ld_out +
                                         (static_cast<int64_t>(u.h) * p.group + head_in) * 128);
      } else if (mine) {
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (w.first == 0 ? 1 : 0);
        // Rows of a unit in order of (token, head): tile B follows tile A's half_tok * group rows.
        const int64_t at_row = slot * kTcRows + x * half_tok * p.group + row;
        p.part_ml[at_row] = make_float2(m, m != -INFINITY ? l : 0.f);
        if (m != -INFINITY) dst = reinterpret_cast<uint8_t*>(p.part_o + at_row * 128);  // a part of weight 0 is never read
      }
      uint8_t* to[8];  // rows 4 k + lane / 8, this lane's 16 bytes
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        to[k] = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), 4 * k + (lane >> 3)));
        if (to[k]) to[k] += (lane & 7) * 16;
      }
      tc_fence_after();
      const float inv = m != -INFINITY ? 1.0f / l : 0.f;
      uint8_t* mine_at = stage + lane * 128;
#pragma unroll 1
      for (int g = 0; g < 4; ++g) {  // 32 columns at a time; two of them make 128 bytes of output
        const int at_byte = whole ? g * 64 : g * 128;
        __syncwarp();  // the pieces before have been read
        uint32_t r[32];
        tmem_ld32(tO + g * 32, r);
        tmem_ld_wait();
        if (whole) {
#pragma unroll
          for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4*>(mine_at + ((k ^ (lane & 7)) << 4)) = tc_pack8<F16>(r + k * 8, inv);
          ++g;
          tmem_ld32(tO + g * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4*>(mine_at + (((k + 4) ^ (lane & 7)) << 4)) = tc_pack8<F16>(r + k * 8, inv);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            *reinterpret_cast<uint4*>(mine_at + ((k ^ (lane & 7)) << 4)) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r8 = 4 * k + (lane >> 3);
          const uint4 v = *reinterpret_cast<const uint4*>(stage + r8 * 128 + (((lane & 7) ^ (r8 & 7)) << 4));
          if (to[k]) *reinterpret_cast<uint4*>(to[k] + at_byte) = v;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        KvPos next = st.at;
        const int64_t rest = st.left - (w.last - w.first);
        st.left = rest > 0 && kv_next_unit<kTcKT>(p, next) ? rest : 0;
        st.at = next;
        st.tiles += w.last - w.first;
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (CLUSTER) {
    cluster_sync();
    if (!no_unit) tc_join_cluster<F16>(p, state[0].at, smem_u32(smem), smem_u32(s_ml), cluster, rank);
    cluster_sync();  // nobody's shared memory goes away while it is read
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool F16, bool CLUSTER>
cudaError_t launch_tc_t(const KvCacheView& c, KvAttnArgs a, int ctas, int cluster, cudaStream_t s) {
  constexpr int smem = CLUSTER ? kTSmem : kTSmemOut;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(kv_tc_kernel<F16, CLUSTER>, smem, done);
  if (e != cudaSuccess) return e;
  a.box_rows = std::min(c.block_size, kTcKT);
  CUtensorMap mq, mk, mv;
  e = kv_query_map(&mq, a, F16, a.unit_tokens / 2);
  if (e == cudaSuccess) e = kv_cache_map(&mk, c, c.k, a.box_rows);
  if (e == cudaSuccess) e = kv_cache_map(&mv, c, c.v, a.box_rows);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kTThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CLUSTER ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kv_tc_kernel<F16, CLUSTER>, mq, mk, mv, a);
}

template <bool F16>
cudaError_t launch_tc(const KvCacheView& c, const KvAttnArgs& a, int ctas, int cluster, cudaStream_t s) {
  return cluster > 1 ? launch_tc_t<F16, true>(c, a, ctas, cluster, s) : launch_tc_t<F16, false>(c, a, ctas, 1, s);
}

}  // namespace

cudaError_t launch_kv_tc(const KvCacheView& c, KvAttnArgs a, int ctas, int cluster, cudaStream_t s) {
  return c.f16 ? launch_tc<true>(c, a, ctas, cluster, s) : launch_tc<false>(c, a, ctas, cluster, s);
}

}  // namespace dcpp
