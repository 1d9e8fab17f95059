// How the paged attention kernels share out their work.
//
// A sequence's query rows are cut into units of `unit_tokens` tokens; a unit of
// one key / value head has n(u) key tiles of KT keys (causal: up to its last
// token's position).  All (sequence, head, unit, tile) quadruples in this order
// form one line of `total` tiles, cut into equal runs, one for each CTA, so that
// any mix of lengths fills the GPU evenly.  A unit that a cut goes through is
// computed in parts by neighbouring CTAs and joined afterwards.  Lengths live on
// the device: every CTA sums them for itself (no plan launch, nothing to keep
// between calls), and every quantity here is a function of them alone.
#pragma once

#include "common.cuh"
#include "kv_cache.cuh"

namespace dcpp {

// sum_{i < n} floor((a i + b) / m), all values below 2^31.
//
// Whole multiples of m in a and b come out as sums of i and of 1.  With a, b < m the terms
// rise from 0 to T = floor((a (n - 1) + b) / m); counted level by level, term i reaches
// level j from i = ceil((j m - b) / a) on, so the sum is
//   sum_{j = 1..T} (n - ceil((j m - b) / a)) = n T - sum_{j < T} floor((m j + m - b + a - 1) / a),
// the same kind of sum with a and m in each other's place: a few turns, as in Euclid's
// algorithm.
static __host__ __device__ __noinline__ int64_t kv_floor_sum(int64_t n, uint32_t m, uint32_t a, uint32_t b) {
  int64_t sum = 0, sign = 1;
  while (n > 0) {
    const uint32_t qa = a / m, qb = b / m;
    sum += sign * (n * (n - 1) / 2 * qa + n * qb);
    a -= qa * m;
    b -= qb * m;
    const int64_t levels = (a * static_cast<uint32_t>(n - 1) + b) / m;  // a < 128, n <= 2^24
    sum += sign * n * levels;
    b = m - b + a - 1;
    const uint32_t was = m;
    m = a;
    a = was;
    n = levels;  // 0 if a was
    sign = -sign;
  }
  return sum;
}

// One sequence's share of the work.
struct KvSeq {
  int32_t q0, q_len;  // its rows in q
  int32_t kv;         // cached keys
  int32_t off;        // position of its first new token: kv - q_len (negative: no key for it)
  int32_t units;
};

// Lengths out of range record an error and leave the sequence out.
__device__ __forceinline__ KvSeq kv_seq(const KvAttnArgs& p, int b) {
  KvSeq s;
  const int32_t c0 = p.cu_new[b], c1 = p.cu_new[b + 1];
  s.kv = p.seq_lens[b];
  s.q0 = c0;
  s.q_len = c1 - c0;
  if (c0 < 0 || c1 < c0 || c1 > p.tokens || s.q_len > p.max_new || s.kv < 0 || s.kv > p.max_kv) {
    record_error(p.err, kDevBadCache);
    s.q0 = s.q_len = s.kv = 0;
  }
  s.off = s.kv - s.q_len;
  s.units = p.unit_shift >= 0 ? (s.q_len + p.unit_tokens - 1) >> p.unit_shift : (s.q_len + p.unit_tokens - 1) / p.unit_tokens;
  return s;
}

// Key tiles of unit u: at least one, so that a unit without keys still writes its zeros.
template <int KT>
__host__ __device__ __forceinline__ int kv_unit_tiles(const KvAttnArgs& p, const KvSeq& s, int u) {
  int keys = s.kv;
  if (p.causal) keys = min(keys, s.off + (u + 1) * p.unit_tokens);
  return max(1, (keys + KT - 1) / KT);
}

// sum_{v < u} n(v).
template <int KT>
__host__ __device__ __forceinline__ int64_t kv_units_before(const KvAttnArgs& p, const KvSeq& s, int u) {
  if (u <= 0) return 0;
  const int full = max(1, (s.kv + KT - 1) / KT);
  if (!p.causal) return static_cast<int64_t>(u) * full;
  int64_t sum = 0;
  int n = u;
  if (u == s.units) {  // the last unit may end before unit_tokens tokens
    sum = full;
    --n;
  }
  // Units whose last key lies in the first tile (or before it) count 1.
  const int U = p.unit_tokens;
  int ones = 0;
  if (s.off + U <= KT) ones = min(n, p.unit_shift >= 0 ? (KT - s.off) >> p.unit_shift : (KT - s.off) / U);
  sum += ones;
  if (n > ones) {
    const int64_t k = n - ones;
    const uint32_t b = static_cast<uint32_t>(s.off + (ones + 1) * U + KT - 1);
    if (p.unit_shift < 0) {
      sum += kv_floor_sum(k, KT, static_cast<uint32_t>(U), b);
    } else if (U >= KT) {  // powers of two, whole tiles per unit: an arithmetic progression
      sum += k * (b / KT) + k * (k - 1) / 2 * (U / KT);
    } else {               // 2^r units per tile: floor((b + i U) / KT) = floor((b / U + i) / 2^r)
      constexpr int kLog = KT == 64 ? 6 : 7;
      static_assert(1 << kLog == KT, "tile size");
      const int r = kLog - p.unit_shift;
      auto below = [r](int64_t x) { const int64_t q = x >> r; return ((q * (q - 1) / 2) << r) + q * (x - (q << r)); };
      const int64_t c = b >> p.unit_shift;
      sum += below(c + k) - below(c);
    }
  }
  return sum;
}

struct KvPos {
  KvSeq s;
  int32_t b, h, u;
  int32_t tile, n_tiles;  // current tile of the unit, tiles of the unit
};

// The line of tiles and its parts: the first `more` have each + 1 tiles.
struct KvRange {
  int64_t total;  // tiles in all
  int64_t each;
  int32_t parts;  // CTAs that have work
  int32_t more;
};

// Shared memory of the schedule: per-thread tile sums and the position found.
template <int NT>
struct KvSchedSmem {
  int64_t warp[NT / 32];
  int64_t base;
  int32_t b;
};

// First tile of part i of r.parts, and the part that tile `pos` lies in.
__host__ __device__ __forceinline__ int64_t kv_cut(const KvRange& r, int i) { return r.each * i + min(i, r.more); }
__host__ __device__ __forceinline__ int kv_part_of(const KvRange& r, int64_t pos) {
  const int64_t big = (r.each + 1) * r.more;
  return static_cast<int>(pos < big ? pos / (r.each + 1) : r.more + (pos - big) / r.each);
}

// All NT threads of the block: the position of the tile at `pos` (on the line).
// base, mine: first tile and tiles of the thread's run of sequences [b0, b1).
template <int KT, int NT>
__device__ __forceinline__ void kv_find(const KvAttnArgs& p, KvSchedSmem<NT>& sm, int64_t base, int64_t mine, int b0, int b1,
                                        int64_t pos, KvPos& at) {
  if (pos >= base && pos < base + mine) {
    for (int b = b0; b < b1; ++b) {
      const KvSeq s = kv_seq(p, b);
      const int64_t n = kv_units_before<KT>(p, s, s.units) * p.heads_kv;
      if (pos < base + n) {
        sm.b = b;
        sm.base = base;
        break;
      }
      base += n;
    }
  }
  __syncthreads();
  at.b = sm.b;
  int64_t rem = pos - sm.base;
  at.s = kv_seq(p, at.b);
  const int64_t per_head = kv_units_before<KT>(p, at.s, at.s.units);
  at.h = static_cast<int>(rem >> 31 || per_head >> 31 ? rem / per_head
                                                      : static_cast<int64_t>(static_cast<uint32_t>(rem) / static_cast<uint32_t>(per_head)));
  rem -= at.h * per_head;
  int lo = 0, hi = at.s.units;  // units_before(lo) <= rem < units_before(hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + NT - 1) / NT;
    const int64_t cand = static_cast<int64_t>(lo) + static_cast<int64_t>(threadIdx.x) * step;
    const bool in = cand < hi && kv_units_before<KT>(p, at.s, static_cast<int>(min(cand, static_cast<int64_t>(hi)))) <= rem;
    const int k = __syncthreads_count(in);  // thread 0 always counts
    lo += (k - 1) * step;
    hi = min(hi, lo + step);
  }
  at.u = lo;
  at.tile = static_cast<int>(rem - kv_units_before<KT>(p, at.s, lo));
  at.n_tiles = kv_unit_tiles<KT>(p, at.s, lo);
  __syncthreads();  // sm.b and sm.base have been read
}

// The next unit on the line (false: there is none).
template <int KT>
__device__ __forceinline__ bool kv_next_unit(const KvAttnArgs& p, KvPos& at) {
  at.tile = 0;
  if (++at.u >= at.s.units) {
    at.u = 0;
    if (++at.h >= p.heads_kv) {
      at.h = 0;
      do {
        if (++at.b >= p.batch) return false;
        at.s = kv_seq(p, at.b);
      } while (at.s.units == 0);
    }
  }
  at.n_tiles = kv_unit_tiles<KT>(p, at.s, at.u);
  return true;
}

// All NT threads of the block: what this CTA (part blockIdx.x of at most p.grid) has
// to do, as the position of its first tile and the number of tiles on the line from
// there (0: nothing).  MIN_TILES: fewest tiles of a part.
template <int KT, int NT, int MIN_TILES>
__device__ __forceinline__ int64_t kv_share(const KvAttnArgs& p, KvSchedSmem<NT>& sm, KvRange& r, KvPos& at) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seg = (p.batch + NT - 1) / NT;
  const int b0 = min(tid * seg, p.batch), b1 = min(b0 + seg, p.batch);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const KvSeq s = kv_seq(p, b);
    mine += kv_units_before<KT>(p, s, s.units) * p.heads_kv;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) sm.warp[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += sm.warp[w];
    total += sm.warp[w];
  }
  r.total = total;
  r.parts = static_cast<int>(max(static_cast<int64_t>(1), min(static_cast<int64_t>(p.grid), total / MIN_TILES)));
  if (total >> 32) {
    r.each = total / r.parts;
    r.more = static_cast<int>(total - r.each * r.parts);
  } else {  // the usual case, without a 64-bit division
    const uint32_t n = static_cast<uint32_t>(total), d = static_cast<uint32_t>(r.parts), q = n / d;
    r.each = q;
    r.more = static_cast<int>(n - q * d);
  }
  const int c = blockIdx.x;
  if (c >= r.parts || total == 0) return 0;
  const int64_t base = before + incl - mine, from = kv_cut(r, c);
  kv_find<KT, NT>(p, sm, base, mine, b0, b1, from, at);
  return kv_cut(r, c + 1) - from;
}

// The direct form, for short units: each cluster of `cluster` CTAs (or each CTA) has
// one unit (long ones of all sequences first), each CTA an equal run of its tiles.
// Nothing has to be summed up or searched.  Returns this CTA's tiles; -1: there is no
// such unit.
template <int KT>
__device__ __forceinline__ int64_t kv_direct(const KvAttnArgs& p, int cluster, int rank, KvPos& at) {
  const int per_unit = p.batch * p.heads_kv, i = blockIdx.x / cluster;
  const int u = i / per_unit, rest = i - u * per_unit;
  at.b = rest / p.heads_kv;
  at.h = rest - at.b * p.heads_kv;
  at.u = p.direct - 1 - u;
  at.s = kv_seq(p, at.b);
  if (at.u >= at.s.units) return -1;
  at.n_tiles = kv_unit_tiles<KT>(p, at.s, at.u);
  at.tile = at.n_tiles * rank / cluster;
  return at.n_tiles * (rank + 1) / cluster - at.tile;
}

// Records what the cut before part `c` goes through, for the kernel that joins parts.
__device__ __forceinline__ void kv_write_cut(const KvAttnArgs& p, const KvRange& r, const KvPos& at, bool have, int c) {
  KvCut cut{};
  if (have && at.tile > 0) {
    const int64_t start = kv_cut(r, c) - at.tile;
    cut.first = kv_part_of(r, start);
    cut.last = kv_part_of(r, start + at.n_tiles - 1);
    cut.rows = min(p.unit_tokens, at.s.q_len - at.u * p.unit_tokens) * p.group;
    cut.tok0 = at.s.q0 + at.u * p.unit_tokens;
    cut.head0 = at.h * p.group;
  }
  p.cuts[c] = cut;
}

}  // namespace dcpp
