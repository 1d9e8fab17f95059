// Attention over the paged cache for many query rows, on the 5th-generation
// tensor cores (tcgen05 + TMEM + TMA).
//
// A unit is two tiles of up to 128 query rows (tokens x the heads of a key /
// value group) of one request and key / value head; CTAs (one per SM) walk their
// run of (unit, key tile) steps.  384 threads:
//   warp 0      TMA: Q of a unit, then K_j, V_j (128 keys, gathered block by block)
//               into a ring of five 32 KB slots
//   warp 1      TMEM allocation and the MMAs: S_X = Q_X K_j^T, O_X += P_X V_j for
//               the tiles X = A, B, in the order
//                 S_A S_B | PV_A S_A' PV_B S_B' | ...
//   warps 4-7   softmax of tile A, warps 8-11 of tile B: one thread per row
// The first four warps hand registers to the softmax warps (a row's 128 scores
// stay in registers): 128 x (96 + 2 x 200) of the 384 x 168 the CTA starts with.
// V stays as the cache holds it, keys x channels: the P V product reads it as an
// operand whose rows run along the channels (MN-major), so no transposed copy of
// the cache is kept.  P goes back over its own scores in TMEM, in two halves of
// 64 keys, each signalled by itself: the first half's product runs while the
// second half's exponentials are computed.
// TMEM (512 columns): S_A / P_A 0, S_B / P_B 128, O_A 256, O_B 384.
#include "kv_device.cuh"
#include "kv_sched.cuh"

#include <algorithm>

namespace dcpp {

namespace {

constexpr int kTThreads = 384;
constexpr int kTSlots = 5;
constexpr int kTHalf = 128 * 128;         // 128 rows x 64 channels: 16 KB
constexpr int kTTile = 2 * kTHalf;        // 128 x 128: 32 KB
constexpr int kTSmem = (2 + kTSlots) * kTTile + 1024;
constexpr float kTRescale = 8.0f;         // log2 units a row maximum may grow before O is rescaled

struct TcBars {
  uint64_t q_full, q_empty;
  uint64_t full[kTSlots], empty[kTSlots];
  uint64_t s_full[2];
  uint64_t p_full[2][2];  // [tile][half], 128 arrivals
  uint64_t pv_done[2];
};

// Instruction descriptor: M 128, N 128, f32 accumulator, both operands of the
// cache's type; B_MN: the B operand's rows run along N.
template <bool F16, bool B_MN>
__host__ __device__ constexpr uint32_t tc_idesc() {
  return (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (B_MN ? 1u << 16 : 0u) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
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

// What a CTA does with the unit at `at`: its key tiles [first, last), and of those
// the ones that each row tile needs (a causal tile A ends before tile B).
struct TcWork {
  int first, last;
  int end[2];
  int tok0, n_tok[2];  // first token of the unit, tokens of each tile
};

__device__ __forceinline__ TcWork tc_work(const KvAttnArgs& p, const KvPos& at, int64_t left) {
  TcWork w;
  const int half = p.unit_tokens / 2;
  w.first = at.tile;
  w.last = at.tile + static_cast<int>(min(left, static_cast<int64_t>(at.n_tiles - at.tile)));
  w.tok0 = at.u * p.unit_tokens;
  const int n = min(p.unit_tokens, at.s.q_len - w.tok0);
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    w.n_tok[x] = min(max(n - x * half, 0), half);
    int keys = at.s.kv;
    if (p.causal) keys = min(keys, at.s.off + w.tok0 + x * half + w.n_tok[x]);
    const int tiles = w.n_tok[x] > 0 ? max(1, (keys + kTcKT - 1) / kTcKT) : 0;
    w.end[x] = max(w.first, min(w.last, tiles));
  }
  return w;
}

struct TcState {
  KvPos at;
  int64_t left;
};

template <bool F16>
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

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_empty, 1);
    for (int i = 0; i < kTSlots; ++i) {
      mbar_init(&bar.full[i], 1);
      mbar_init(&bar.empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bar.s_full[x], 1);
      mbar_init(&bar.p_full[x][0], 128);
      mbar_init(&bar.p_full[x][1], 128);
      mbar_init(&bar.pv_done[x], 1);
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
  const bool have = kv_locate<kTcKT, kTThreads, kTcMinTiles>(p, sched, range, at, [&](const KvRange& r) {
    return static_cast<int>(blockIdx.x) < r.parts ? kv_cut(r, blockIdx.x) : static_cast<int64_t>(-1);
  });
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  int64_t left = have ? kv_cut(range, blockIdx.x + 1) - kv_cut(range, blockIdx.x) : 0;
  const int half_tok = p.unit_tokens / 2;

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
  if (warp == 0) {
    const int boxes = kTcKT / p.box_rows;
    const int box = lane & (boxes - 1), half = lane / boxes;
    const int bs_mask = (1 << p.block_shift) - 1;
    const uint32_t q_bytes = 2u * 128u * static_cast<uint32_t>(half_tok * p.group);
    int it = 0, unit = 0;
    bool ok = true;
    while (left > 0 && ok) {
      const TcWork w = tc_work(p, at, left);
      ok = __all_sync(0xffffffffu, kv_wait(&bar.q_empty, (unit & 1) ^ 1, p.err));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar.q_full, w.n_tok[1] > 0 ? 2 * q_bytes : q_bytes);
        for (int x = 0; x < 2; ++x)
          if (w.n_tok[x] > 0)
            for (int k = 0; k < 2; ++k)
              tma_load_3d(sQ + x * kTTile + k * kTHalf, &tmQ, &bar.q_full, k * 64, at.h * p.group,
                          at.s.q0 + w.tok0 + x * half_tok);
      }
      __syncwarp();
      ++unit;
      const int32_t* row = p.table + at.b * p.max_blocks;
      const int n_ids = (at.s.kv + bs_mask) >> p.block_shift;
      int win = (w.first * kTcKT) >> p.block_shift;
      auto fetch = [&](int i) { return i < n_ids ? __ldg(row + i) : -1; };
      int cur = fetch(win + lane), nxt = fetch(win + 32 + lane);
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
        for (int kv = 0; kv < 2; ++kv, ++it) {  // K_j, then V_j
          const int st = it % kTSlots;
          ok = __all_sync(0xffffffffu, kv_wait(&bar.empty[st], ((it / kTSlots) & 1) ^ 1, p.err));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&bar.full[st], loads * p.box_rows * 128);
          __syncwarp();
          if (load)
            tma_load_4d(sKV + st * kTTile + half * kTHalf + box * p.box_rows * 128, kv ? &tmV : &tmK, &bar.full[st],
                        half * 64, key0 & bs_mask, at.h, c3);
        }
      }
      left -= w.last - w.first;
      if (left > 0 && !kv_next_unit<kTcKT>(p, at)) break;
    }
    // Nothing may be in flight when the CTA ends: all copies landed, and (unless a
    // wait ran out) every slot handed back, i.e. the last commits have arrived.
    for (int k = max(0, it - kTSlots); k < it; ++k)
      if (!kv_wait(&bar.full[k % kTSlots], (k / kTSlots) & 1, p.err)) ok = false;
    if (unit > 0 && !kv_wait(&bar.q_full, (unit - 1) & 1, p.err)) ok = false;
    if (ok) {
      for (int k = max(0, it - kTSlots); k < it; ++k)
        if (!kv_wait(&bar.empty[k % kTSlots], (k / kTSlots) & 1, p.err)) break;
      if (unit > 0) kv_wait(&bar.q_empty, (unit - 1) & 1, p.err);
    }
  } else if (warp == 1) {
    // The whole warp runs the loop; one elected lane issues the MMAs and commits.
    constexpr uint32_t idS = tc_idesc<F16, false>(), idPV = tc_idesc<F16, true>();
    const uint64_t dQ = make_sdesc_sw128(smem_u32(sQ));
    const uint64_t dK = make_sdesc_sw128(smem_u32(sKV));
    const uint64_t dV = tc_desc_mn(smem_u32(sKV));
    auto koff = [](int k) -> uint64_t { return static_cast<uint64_t>(((k >> 2) * kTHalf + (k & 3) * 32) >> 4); };
    constexpr uint64_t kTileD = kTTile >> 4;
    const bool leader = elect_one_sync();
    int it = 0, unit = 0;
    int n_pv[2] = {0, 0}, n_p[2] = {0, 0};
    bool ok = true;
    auto wait = [&](uint64_t* b, int phase) {
      ok = __all_sync(0xffffffffu, ok && kv_wait(b, phase & 1, p.err));
      if (ok) tc_fence_after();
      return ok;
    };
    // S_X = Q_X K^T from slot `slot`; last: the last use of this K slot; done: of this unit's Q.
    auto issue_s = [&](int x, int slot, bool last, bool done) {
      if (n_pv[x] > 0 && !wait(&bar.pv_done[x], n_pv[x] - 1)) return;  // P over S has been read
      if (leader) {
        const uint64_t q = dQ + x * kTileD, kd = dK + slot * kTileD;
#pragma unroll
        for (int k = 0; k < 8; ++k) umma_bf16(tmem + x * 128, q + koff(k), kd + koff(k), idS, k > 0 ? 1u : 0u);
        umma_commit(&bar.s_full[x]);
        if (last) umma_commit(&bar.empty[slot]);
        if (done) umma_commit(&bar.q_empty);
      }
      __syncwarp();
    };
    while (left > 0 && ok) {
      const TcWork w = tc_work(p, at, left);
      const int top = w.n_tok[1] > 0 ? 1 : 0;  // the tile that needs every key tile of the run
      if (!wait(&bar.q_full, unit)) break;
      ++unit;
      const int n = w.last - w.first;
      auto k_slot = [&](int i) { return (it + 2 * i) % kTSlots; };
      auto k_phase = [&](int i) { return (it + 2 * i) / kTSlots; };
      if (!wait(&bar.full[k_slot(0)], k_phase(0))) break;
      for (int x = 0; x <= top && ok; ++x)
        if (w.first < w.end[x]) issue_s(x, k_slot(0), x == top, x == top && n == 1);
      for (int i = 0; i < n && ok; ++i) {
        const int j = w.first + i;
        const int vs = (it + 2 * i + 1) % kTSlots;
        if (!wait(&bar.full[vs], (it + 2 * i + 1) / kTSlots)) break;
        const int valid = at.s.kv - j * kTcKT;
        if (valid < kTcKT) {
          // Behind the last key a block holds anything, and 0 x NaN is NaN: clear those rows.
          uint8_t* v = sKV + vs * kTTile;
          for (int c = max(valid, 0) * 8 + lane; c < kTcKT * 8; c += 32) {
            *reinterpret_cast<uint4*>(v + c * 16) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(v + kTHalf + c * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        for (int x = 0; x <= top && ok; ++x) {
          if (j >= w.end[x]) continue;
          const uint32_t tO = tmem + 256 + x * 128, tP = tmem + x * 128;
          const uint64_t vd = dV + vs * kTileD;
          for (int h = 0; h < 2; ++h) {
            if (!wait(&bar.p_full[x][h], n_p[x])) break;
            if (leader) {
#pragma unroll
              for (int k = 0; k < 4; ++k)  // 16 keys: 8 packed TMEM columns of P, 16 rows (2 KB) of V
                umma_bf16_ts(tO, tP + h * 32 + k * 8, vd + ((h * 4 + k) * 2048 >> 4), idPV, i > 0 || h > 0 || k > 0 ? 1u : 0u);
              if (h == 1) {
                umma_commit(&bar.pv_done[x]);
                if (x == top) umma_commit(&bar.empty[vs]);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          ++n_p[x];
          ++n_pv[x];
          if (j + 1 < w.end[x]) {
            if (!wait(&bar.full[k_slot(i + 1)], k_phase(i + 1))) break;
            issue_s(x, k_slot(i + 1), x == top, x == top && i + 2 == n);
          }
        }
      }
      it += 2 * n;
      left -= n;
      if (left > 0 && !kv_next_unit<kTcKT>(p, at)) break;
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int x = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;  // TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + x * 128, tO = tmem + lane_off + 256 + x * 128;
    const float c = p.scale_log2;
    int n_s = 0;
    bool ok = true;
    // The walk's state rests in shared memory while a unit is computed: its registers
    // are needed for the scores.
    TcState& st = state[warp - 4];
    if (lane == 0) {
      st.at = at;
      st.left = left;
    }
    __syncwarp();
    while (ok && st.left > 0) {
      int first, end, limit, all_below;
      {
        const KvPos u = st.at;
        const TcWork w = tc_work(p, u, st.left);
        first = w.first;
        end = w.end[x];
        const int tile0 = u.s.off + w.tok0 + x * half_tok;  // position of the tile's first token
        limit = u.s.kv;  // keys this row attends to: [0, limit)
        if (p.causal) limit = min(limit, tile0 + row / p.group + 1);
        all_below = u.s.kv;  // keys that every row of the tile attends to
        if (p.causal) all_below = min(all_below, tile0 + 1);
      }
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = first; j < end; ++j) {
        ok = __all_sync(0xffffffffu, kv_wait(&bar.s_full[x], n_s & 1, p.err));
        if (!ok) break;
        ++n_s;
        tc_fence_after();
        float s[128];
        {
          uint32_t r0[32], r1[32], r2[32], r3[32];
          tmem_ld32(tS, r0);
          tmem_ld32(tS + 32, r1);
          tmem_ld32(tS + 64, r2);
          tmem_ld32(tS + 96, r3);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            s[i] = __uint_as_float(r0[i]);
            s[32 + i] = __uint_as_float(r1[i]);
            s[64 + i] = __uint_as_float(r2[i]);
            s[96 + i] = __uint_as_float(r3[i]);
          }
        }
        const int kbase = j * kTcKT;
        if (kbase + kTcKT > all_below) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (kbase + i >= limit) s[i] = -INFINITY;
        }
        float mp[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mp[k] = s[k];
#pragma unroll
        for (int i = 8; i < 128; i += 2) mp[(i >> 1) & 7] = max3(mp[(i >> 1) & 7], s[i], s[i + 1]);
        const float mx = c * max3(max3(mp[0], mp[1], mp[2]), max3(mp[3], mp[4], mp[5]), fmaxf(mp[6], mp[7]));
        const bool grow = mx > m + kTRescale;
        const float m_use = grow ? mx : m;
        // A stale maximum is exact (l uses the same one); without a key so far every numerator is 0.
        const float ref = m_use == -INFINITY ? 0.f : m_use;
        const float alpha = grow ? ex2(m - ref) : 1.0f;
        const uint64_t c2 = f2(c, c), nm2 = f2(-ref, -ref);
        uint64_t sp[4] = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint64_t y = fma2(f2(s[h * 64 + 2 * i], s[h * 64 + 2 * i + 1]), c2, nm2);
            const uint64_t e = (i & 3) == 3 ? ex2_poly2(y) : f2(ex2(f2lo(y)), ex2(f2hi(y)));
            sp[i & 3] = add2(sp[i & 3], e);
            pk[i] = kv_pack2<F16>(f2lo(e), f2hi(e));
          }
          if (h == 0 && j > first && __any_sync(0xffffffffu, grow)) {  // S_j complete: so is P V of every earlier tile
#pragma unroll 1
            for (int ch = 0; ch < 4; ++ch) {
              uint32_t r[32];
              tmem_ld32(tO + ch * 32, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
              tmem_st32(tO + ch * 32, r);
            }
          }
          tmem_st32(tS + h * 32, pk);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&bar.p_full[x][h]);
        }
        const uint64_t t = add2(add2(sp[0], sp[1]), add2(sp[2], sp[3]));
        l = l * alpha + f2lo(t) + f2hi(t);
        m = m_use;
      }
      if (ok && first < end) ok = __all_sync(0xffffffffu, kv_wait(&bar.pv_done[x], (n_s - 1) & 1, p.err));
      if (!ok) break;
      const KvPos u = st.at;
      const TcWork w = tc_work(p, u, st.left);
      const int tok_in = row / p.group, head_in = row - tok_in * p.group;
      const int tok = w.tok0 + x * half_tok + tok_in;
      const bool mine = tok_in < w.n_tok[x];
      const bool whole = w.first == 0 && w.last == u.n_tiles;
      uint32_t r0[32], r1[32], r2[32], r3[32];
      tc_fence_after();
      tmem_ld32(tO, r0);
      tmem_ld32(tO + 32, r1);
      tmem_ld32(tO + 64, r2);
      tmem_ld32(tO + 96, r3);
      tmem_ld_wait();
      tc_fence_before();
      const uint32_t* rs[4] = {r0, r1, r2, r3};
      if (mine && whole) {
        const float inv = m != -INFINITY ? 1.0f / l : 0.f;
        uint16_t* dst = p.out + static_cast<int64_t>(u.s.q0 + tok) * p.ld_out +
                        (static_cast<int64_t>(u.h) * p.group + head_in) * 128;
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint4* d4 = reinterpret_cast<uint4*>(dst + ch * 32);
          const uint32_t* r = rs[ch];
#pragma unroll
          for (int v = 0; v < 4; ++v)
            d4[v] = make_uint4(
                kv_pack2<F16>(__uint_as_float(r[8 * v]) * inv, __uint_as_float(r[8 * v + 1]) * inv),
                kv_pack2<F16>(__uint_as_float(r[8 * v + 2]) * inv, __uint_as_float(r[8 * v + 3]) * inv),
                kv_pack2<F16>(__uint_as_float(r[8 * v + 4]) * inv, __uint_as_float(r[8 * v + 5]) * inv),
                kv_pack2<F16>(__uint_as_float(r[8 * v + 6]) * inv, __uint_as_float(r[8 * v + 7]) * inv));
        }
      } else if (mine) {
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (w.first == 0 ? 1 : 0);
        // Rows of a unit in order of (token, head): tile B follows tile A's half_tok * group rows.
        const int64_t at_row = slot * kTcRows + x * half_tok * p.group + row;
        p.part_ml[at_row] = make_float2(m, m != -INFINITY ? l : 0.f);
        if (m != -INFINITY) {  // a part of weight 0 is never read
          float4* d4 = reinterpret_cast<float4*>(p.part_o + at_row * 128);
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
#pragma unroll
            for (int v = 0; v < 8; ++v)
              d4[ch * 8 + v] = make_float4(__uint_as_float(rs[ch][4 * v]), __uint_as_float(rs[ch][4 * v + 1]),
                                           __uint_as_float(rs[ch][4 * v + 2]), __uint_as_float(rs[ch][4 * v + 3]));
        }
      }
      __syncwarp();
      if (lane == 0) {
        KvPos next = st.at;
        const int64_t rest = st.left - (w.last - w.first);
        st.left = rest > 0 && kv_next_unit<kTcKT>(p, next) ? rest : 0;
        st.at = next;
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool F16>
cudaError_t launch_tc_t(const KvCacheView& c, KvAttnArgs a, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(kv_tc_kernel<F16>, kTSmem, done);
  if (e != cudaSuccess) return e;
  a.box_rows = std::min(c.block_size, kTcKT);
  CUtensorMap mq, mk, mv;
  e = kv_query_map(&mq, a, F16, a.unit_tokens / 2);
  if (e == cudaSuccess) e = kv_cache_map(&mk, c, c.k, a.box_rows);
  if (e == cudaSuccess) e = kv_cache_map(&mv, c, c.v, a.box_rows);
  if (e != cudaSuccess) return e;
  kv_tc_kernel<F16><<<a.grid, kTThreads, kTSmem, s>>>(mq, mk, mv, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_tc(const KvCacheView& c, KvAttnArgs a, cudaStream_t s) {
  return c.f16 ? launch_tc_t<true>(c, a, s) : launch_tc_t<false>(c, a, s);
}

}  // namespace dcpp
