// Attention of a batch's new tokens over the paged key / value cache.
//
//   o[t, h] = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q[t, h] . k_j,
// j over the request's cached keys (causal: up to the token's own position); a row
// without a key is 0.  Sums, maxima and the scores are f32; the numerators are
// rounded once to the cache's type (half a step: 2^-8 of each in bf16, 2^-11 in f16, as the
// output's own rounding) because the matrix instructions take their operands in it.  f16 has
// a fixed step below its smallest normal, so its numerators (and the sum of them, which
// cancels the factor) are kept 2^lift times larger: what is lost of a key is at most
// 2^-(25 + lift) of the row's largest numerator.  Unlifted, 131k keys 17 lower than one
// were 0 in the products and 0.4 % of the sum.
//
// Rows of one key / value head: the `group` query heads that share it times the
// tokens of a unit, so that K and V are read once for all of them.
#include "kv_device.cuh"
#include "kv_form.cuh"
#include "kv_sched.cuh"

#include <algorithm>

namespace dcpp {

namespace {

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ------------------------------------------------------------ few query rows
// Up to 16 rows per unit (single tokens, a few drafted ones): bound by reading K
// and V once from HBM, so the tensor work only has to stay out of the way:
// mma.sync m16n8k16.  Two CTAs per SM, each with a ring of 3 stages of 64 keys (K
// 16 KB + V 16 KB, two 128-byte-swizzled halves of the head dimension each) that one
// warp fills with TMA, a box for each piece of a block.
// The four consumer warps each own 16 keys of every tile: scores, running maximum,
// numerators and all 128 output columns of their keys, so the loop has no barrier
// among them; their four partial results are joined once per unit.  Measured, 32 heads
// over 8: 64 requests of 100 to 8000 keys 186 us (6.3 TB/s), 1 of 131k keys 90 us
// (6.0 TB/s), 1 of 517 keys 6.8 us.
constexpr int kRStages = 3;
constexpr int kRHalf = kRKT * 128;          // 8 KB: 64 keys x 64 channels
constexpr int kRStageBytes = 4 * kRHalf;    // K lo, K hi, V lo, V hi
constexpr int kRThreads = 160;              // 4 consumer warps + the producer
constexpr int kRJoinBytes = 8192;           // Q rows, later the partial sums being joined
constexpr int kRSmem = kRStages * kRStageBytes + kRJoinBytes + 1024;
// Fewest tiles of a part.  Measured with 2 / 4 / 6, 8 heads over 1: 12k keys 12.1 / 13.5 /
// 15.6 us, 60k keys 19.0 / 16.9 / 17.8 us.
constexpr int kRMinTiles = 2;
// Numerators are at most 2^lift (the maximum is never stale): three bits below f16's largest
// value, for the rounding of maximum x scale (half a step: 2 at 2^25).
template <bool F16>
constexpr float kRLift = F16 ? 13.0f : 0.0f;

// Joins a unit that the CTAs of a cluster computed together: every warp's sums go to
// its CTA's shared memory (the stages, all read by now), and each CTA adds up the four
// warps of all CTAs for its share of the 128 output columns, eight lanes to four
// columns of a row, each with every eighth of the sums (in an order that does not
// change).  The four consumer warps; the producer warp meets the two cluster barriers
// by itself.
template <bool F16>
__device__ __forceinline__ void kv_rows_join_cluster(const KvAttnArgs& p, const KvPos& at, uint8_t* smem,
                                                     float2 (&s_ml)[4][kRRows], const float (&o)[16][4], int cluster,
                                                     int rank, int t0, int rows) {
  constexpr int R = kRRows, kLd = 136;  // padded rows: stores without bank conflicts
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cq = (lane & 3) * 2;
  float* sums = reinterpret_cast<float*>(smem);  // [warp][R][kLd]
#pragma unroll
  for (int d = 0; d < 16; ++d)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float2*>(sums + (warp * R + g + e * 8) * kLd + d * 8 + cq) =
          make_float2(o[d][2 * e], o[d][2 * e + 1]);
  cluster_sync();
  const uint32_t ml_at = smem_u32(s_ml), sums_at = smem_u32(sums);
  const int quads = 32 / cluster, units = rows * quads;  // four columns of a row: this CTA's share
  const int j = lane & 7;
  for (int i0 = 0; i0 < units; i0 += 16) {
    const int i = min(i0 + (tid >> 3), units - 1);
    const int r = i / quads, c4 = (rank * quads + (i - r * quads)) * 4;
    float2 ml[4];
    float4 a[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k = j + 8 * q;  // warp k % 4 of CTA k / 4
      if (k < 4 * cluster) {
        ml[q] = ld_cluster2(mapa_shared(ml_at + static_cast<uint32_t>((k & 3) * R + r) * 8, k >> 2));
        a[q] = ld_cluster4(mapa_shared(sums_at + static_cast<uint32_t>(((k & 3) * R + r) * kLd + c4) * 4, k >> 2));
      } else {
        ml[q] = make_float2(-INFINITY, 0.f);
        a[q] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    float M = max_nan(max_nan(ml[0].x, ml[1].x), max_nan(ml[2].x, ml[3].x));
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, x));
    float L = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float w = ml[q].x == -INFINITY ? 0.f : ex2(ml[q].x - M);
      L = fmaf(w, ml[q].y, L);
      s.x = fmaf(w, a[q].x, s.x); s.y = fmaf(w, a[q].y, s.y);
      s.z = fmaf(w, a[q].z, s.z); s.w = fmaf(w, a[q].w, s.w);
    }
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) {
      L += __shfl_xor_sync(0xffffffffu, L, x);
      s.x += __shfl_xor_sync(0xffffffffu, s.x, x);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, x);
      s.z += __shfl_xor_sync(0xffffffffu, s.z, x);
      s.w += __shfl_xor_sync(0xffffffffu, s.w, x);
    }
    if (j == 0 && i0 + (tid >> 3) < units) {
      const float inv = L != 0.f ? 1.0f / L : 0.f;
      const int tok = p.row_token(r), hh = r - tok * p.group;
      uint16_t* dst = p.out + static_cast<int64_t>(t0 + tok) * p.ld_out +
                      (static_cast<int64_t>(at.h) * p.group + hh) * 128 + c4;
      *reinterpret_cast<uint2*>(dst) = make_uint2(kv_pack2<F16>(s.x * inv, s.y * inv), kv_pack2<F16>(s.z * inv, s.w * inv));
    }
  }
  cluster_sync();  // nobody's shared memory goes away while it is read
}

template <bool F16, bool DIRECT>
__global__ void __launch_bounds__(kRThreads, 2)
    kv_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ KvAttnArgs p) {
  constexpr int R = kRRows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* join = smem + kRStages * kRStageBytes;
  __shared__ uint64_t full[kRStages], empty[kRStages];
  __shared__ float2 s_ml[4][R];
  __shared__ KvSchedSmem<kRThreads> sched;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kRStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  KvRange range;
  KvPos at;
  // In the direct form a cluster shares a unit and joins it through its shared memory.
  int cluster = 1, rank = 0;
  int64_t left;
  if constexpr (DIRECT) {
    cluster = cluster_size();
    rank = static_cast<int>(cluster_ctarank());
    left = kv_direct<kRKT>(p, cluster, rank, at);
  } else {
    left = kv_share<kRKT, kRThreads, kRMinTiles>(p, sched, range, at);
  }
  // The producer's block ids come from the table 32 at a time, the next 32 fetched ahead;
  // those of the first tile are on their way while the CTA sets up.
  int cur = -1, nxt = -1;
  auto fetch = [&](int i) { return i < p.max_blocks ? __ldg(p.table + at.b * p.max_blocks + i) : -1; };
  auto fetch_first = [&] {
    const int win = (at.tile * kRKT) >> p.block_shift;
    cur = fetch(win + lane);
    nxt = fetch(win + 32 + lane);
  };
  if (warp == 4 && left > 0) fetch_first();
  __syncthreads();  // barriers initialised
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!DIRECT && tid == 0) kv_write_cut(p, range, at, left > 0, blockIdx.x);
  if (DIRECT ? left < 0 : left == 0) return;

  if (warp == 4) {
    // Producer: lane -> (K or V, half, box).
    const int boxes = kRKT / p.box_rows;             // 1, 2 or 4 boxes per tile and half
    const int box = lane & (boxes - 1);
    const int part = lane / boxes;                   // 0, 1: K halves; 2, 3: V halves; more: idle
    const int bs_mask = (1 << p.block_shift) - 1;
    int it = 0;
    bool ok = true;
    while (left > 0 && ok) {
      const int n = static_cast<int>(min(left, static_cast<int64_t>(at.n_tiles - at.tile)));
      int win = (at.tile * kRKT) >> p.block_shift;  // first block id held
      for (int j = at.tile; j < at.tile + n && ok; ++j, ++it) {
        const int key0 = j * kRKT + box * p.box_rows;
        int idx = key0 >> p.block_shift;
        if (__shfl_sync(0xffffffffu, idx, 0) - win >= 32) {  // a tile's boxes never straddle a window
          win += 32;
          cur = nxt;
          nxt = fetch(win + 32 + lane);
        }
        const int blk = __shfl_sync(0xffffffffu, cur, idx - win);
        const bool load = part < 4 && key0 < at.s.kv;
        if (load && (blk < 0 || blk >= p.n_blocks)) record_error(p.err, kDevBadCache);
        const int c3 = blk < 0 || blk >= p.n_blocks ? p.n_blocks : blk;  // one past the end: TMA fills zeros
        const int st = it % kRStages;
        ok = kv_wait(&empty[st], ((it / kRStages) & 1) ^ 1, p.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int loads = __popc(__ballot_sync(0xffffffffu, load));
        if (lane == 0) mbar_arrive_expect_tx(&full[st], loads * p.box_rows * 128);
        __syncwarp();
        if (load) {
          uint8_t* dst = smem + st * kRStageBytes + part * kRHalf + box * p.box_rows * 128;
          tma_load_4d(dst, part < 2 ? &tmK : &tmV, &full[st], (part & 1) * 64, key0 & bs_mask, at.h, c3);
        }
      }
      left -= n;
      if (DIRECT || left <= 0 || !kv_next_unit<kRKT>(p, at)) break;
      fetch_first();
    }
    // Every copy has landed before the CTA may end (a consumer that gave up waits for none).
    for (int k = max(0, it - kRStages); k < it; ++k)
      if (!kv_wait(&full[k % kRStages], (k / kRStages) & 1, p.err)) break;
    if (DIRECT && cluster > 1) {  // the consumers' two barriers
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  // Consumers.
  const uint32_t sbase = smem_u32(smem), jbase = smem_u32(join);
  const int g = lane >> 2, cq = (lane & 3) * 2;  // accumulator row within 8, first of two columns
  int it = 0;
  bool ok = true;
  for (;;) {
    const int n = static_cast<int>(min(left, static_cast<int64_t>(at.n_tiles - at.tile)));
    const int first = at.tile;
    const int t0 = at.s.q0 + at.u * p.unit_tokens;
    const int n_tok = min(p.unit_tokens, at.s.q_len - at.u * p.unit_tokens);
    const int rows = n_tok * p.group;

    // Q rows into shared memory (two halves of R rows x 128 bytes, 128-byte swizzle).
    named_sync(1, 128);
    for (int i = tid; i < R * 16; i += 128) {
      const int r = i >> 4, ch = i & 15;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        const int tok = p.row_token(r), hh = r - tok * p.group;
        v = *reinterpret_cast<const uint4*>(p.q + static_cast<int64_t>(t0 + tok) * p.ld_q +
                                            (static_cast<int64_t>(at.h) * p.group + hh) * 128 + ch * 8);
      }
      *reinterpret_cast<uint4*>(join + (ch >> 3) * (R * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
    }
    named_sync(1, 128);
    // A fragment (channels ks * 16..).
    auto load_q = [&](int ks, uint32_t (&a)[4]) {
      const int r = lane & 15, ch = (ks & 3) * 2 + (lane >> 4);
      ldsm4(jbase + (ks >> 2) * (R * 128) + r * 128 + ((ch ^ (r & 7)) << 4), a);
    };
    uint32_t qf[8][4];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) load_q(ks, qf[ks]);
    // Keys each accumulator row attends to: [0, limit).
    int limit[2];
    int min_limit = at.s.kv;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = g + e * 8;
      int lim = at.s.kv;
      if (p.causal) lim = min(lim, at.s.off + at.u * p.unit_tokens + p.row_token(r) + 1);
      limit[e] = lim;
    }
    if (p.causal) min_limit = min(min_limit, at.s.off + at.u * p.unit_tokens + 1);

    float o[16][4];
    float m[2], l[2];
#pragma unroll
    for (int d = 0; d < 16; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
    for (int j = first; j < first + n; ++j, ++it) {
      const int st = it % kRStages;
      if (ok) ok = __all_sync(0xffffffffu, kv_wait(&full[st], (it / kRStages) & 1, p.err));
      if (!ok) continue;  // a wait ran out: no more work, but every barrier below is still met
      const int key0 = j * kRKT + warp * 16;
      if (key0 < at.s.kv) {
        const uint32_t kb = sbase + st * kRStageBytes, vb = kb + 2 * kRHalf;
        const int krow = warp * 16 + ((lane >> 4) << 3) + (lane & 7);  // ldmatrix row of K
        float s[2][4];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nb][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t b[4];
          const int ch = (ks & 3) * 2 + ((lane >> 3) & 1);
          ldsm4(kb + (ks >> 2) * kRHalf + krow * 128 + ((ch ^ (krow & 7)) << 4), b);
          mma16816<F16>(s[0], qf[ks], b[0], b[1]);
          mma16816<F16>(s[1], qf[ks], b[2], b[3]);
        }
        if (key0 + 16 > min_limit) {
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + nb * 8 + cq + (e & 1) >= limit[e >> 1]) s[nb][e] = -INFINITY;
        }
        uint32_t pf[4];
        bool grew = false;
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          mx *= p.scale_log2;
          const float m_new = fmaxf(m[e], mx);
          const float ref = m_new == -INFINITY ? 0.f : m_new;  // no key so far: every numerator 0
          const float up = kRLift<F16> - ref;
          grew |= m_new != m[e];
          alpha[e] = ex2(m[e] - ref);
          float sum = 0.f;
#pragma unroll
          for (int nb = 0; nb < 2; ++nb)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float& x = s[nb][2 * e + q];
              x = ex2(fmaf(x, p.scale_log2, up));
              sum += x;
            }
          l[e] = l[e] * alpha[e] + sum;
          m[e] = m_new;
        }
        pf[0] = kv_pack2<F16>(s[0][0], s[0][1]);
        pf[1] = kv_pack2<F16>(s[0][2], s[0][3]);
        pf[2] = kv_pack2<F16>(s[1][0], s[1][1]);
        pf[3] = kv_pack2<F16>(s[1][2], s[1][3]);
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int d = 0; d < 16; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] *= alpha[e >> 1];
        }
        const int vrow = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);  // ldmatrix row of V
        if (key0 + 16 > at.s.kv) {
          // Behind the last key a block holds anything, and 0 x NaN is NaN: clear those rows.
          for (int i = lane; i < 256; i += 32) {
            const int r = i >> 4, ch = i & 15;
            if (key0 + r >= at.s.kv)
              *reinterpret_cast<uint4*>(smem + st * kRStageBytes + (2 + (ch >> 3)) * kRHalf + (warp * 16 + r) * 128 +
                                        ((ch & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();  // before a later TMA write to the same bytes
          __syncwarp();
        }
#pragma unroll
        for (int np = 0; np < 8; ++np) {
          uint32_t b[4];
          const int ch = (np & 3) * 2 + (lane >> 4);
          ldsm4t(vb + (np >> 2) * kRHalf + vrow * 128 + ((ch ^ (vrow & 7)) << 4), b);
          mma16816<F16>(o[2 * np], pf, b[0], b[1]);
          mma16816<F16>(o[2 * np + 1], pf, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // Join the four warps: weights 2^(m_w - M), sums over w in order.
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[e];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if (x != x) m[e] = x;  // scores that are NaN do not raise the maximum: the row is NaN, not empty
      if ((lane & 3) == 0) s_ml[warp][g + e * 8] = make_float2(m[e], x);
    }
    named_sync(1, 128);  // also: all Q fragments, and every stage, have been read
    if constexpr (DIRECT) {
      if (cluster > 1) {
        kv_rows_join_cluster<F16>(p, at, smem, s_ml, o, cluster, rank, t0, rows);
        return;
      }
    }
    float w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = g + e * 8;
      const float M = max_nan(max_nan(s_ml[0][r].x, s_ml[1][r].x), max_nan(s_ml[2][r].x, s_ml[3][r].x));
      w[e] = M == -INFINITY ? 0.f : ex2(m[e] - M);
    }
    const bool whole = first == 0 && n == at.n_tiles;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (first == 0 ? 1 : 0);
    // The sums meet in shared memory, 32 columns a round, or all at once where the unit is
    // the CTA's only one and the stages are free.  Row r of a warp's sums has its 8-column
    // groups at places ^ (r & 3), so that the four rows of a half warp's stores lie in
    // different banks.
    constexpr int ROUNDS = DIRECT ? 1 : 4, DC = 128 / ROUNDS;
    float* jf = reinterpret_cast<float*>(DIRECT ? smem : join);  // [warp][R][DC]
    const int r = tid >> 3, c4 = (tid & 7) * 4;
    const float M = max_nan(max_nan(s_ml[0][r].x, s_ml[1][r].x), max_nan(s_ml[2][r].x, s_ml[3][r].x));
    float L = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) L += M == -INFINITY ? 0.f : s_ml[k][r].y * ex2(s_ml[k][r].x - M);
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    const int tok = p.row_token(r), hh = r - tok * p.group;
    uint16_t* dst = p.out + static_cast<int64_t>(t0 + tok) * p.ld_out + (static_cast<int64_t>(at.h) * p.group + hh) * 128 + c4;
    if (!whole && r < rows && c4 == 0) p.part_ml[slot * R + r] = make_float2(M, L);
#pragma unroll
    for (int rd = 0; rd < ROUNDS; ++rd) {
#pragma unroll
      for (int d = 0; d < DC / 8; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(jf + (warp * R + g + e * 8) * DC + ((d ^ (g & 3)) << 3) + cq) =
              make_float2(o[rd * (DC / 8) + d][2 * e] * w[e], o[rd * (DC / 8) + d][2 * e + 1] * w[e]);
      named_sync(1, 128);
      if (r < rows) {
#pragma unroll
        for (int cc = 0; cc < DC; cc += 32) {
          const int at_c = cc + (((c4 >> 3) ^ (r & 3)) << 3) + (c4 & 4);
          float4 a = *reinterpret_cast<const float4*>(jf + r * DC + at_c);
#pragma unroll
          for (int k = 1; k < 4; ++k) {
            const float4 b = *reinterpret_cast<const float4*>(jf + (k * R + r) * DC + at_c);
            a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
          }
          const int col = rd * DC + cc;
          if (whole)
            *reinterpret_cast<uint2*>(dst + col) = make_uint2(kv_pack2<F16>(a.x * inv, a.y * inv), kv_pack2<F16>(a.z * inv, a.w * inv));
          else
            *reinterpret_cast<float4*>(p.part_o + (slot * R + r) * 128 + col + c4) = a;
        }
      }
      if (!DIRECT) named_sync(1, 128);
    }
    left -= n;
    if (DIRECT || left <= 0 || !kv_next_unit<kRKT>(p, at)) break;
  }
}

// ------------------------------------------------------------ joining parts
// A unit in the parts f .. l has its partial sums in slot 2 f + 1 (it starts there)
// and 2 k, k = f + 1 .. l.  They are summed in the order of the parts, so the result
// does not depend on which CTA finished first.  What this costs is latency, so the
// work is spread wide: the blocks of all of a unit's cuts (and their y blocks) share
// its rows, four to a group whose loads go out together; a group is one warp's, or,
// for a unit in eight parts or more, a block's whose warps take every eighth part each.
// From 32 parts on the block takes a single row and each warp four of its parts at a
// time (1 request of 30k keys, 8 heads over 1, in 235 parts: 24.2 -> 15.1 us in all).
constexpr int kJThreads = 256;
constexpr int kJWarps = kJThreads / 32;
constexpr int kJPer = 4;  // rows of a group

__device__ __forceinline__ void join_fma(float4& s, float w, const float4& a) {
  if (w != 0.f) {  // a part of weight 0 may not have written its sums
    s.x = fmaf(w, a.x, s.x); s.y = fmaf(w, a.y, s.y);
    s.z = fmaf(w, a.z, s.z); s.w = fmaf(w, a.w, s.w);
  }
}

template <bool F16>
__device__ __forceinline__ void join_store(const KvAttnArgs& p, const KvCut& cut, int r, int c4, const float4& a, float by) {
  const int tok = p.row_token(r), hh = r - tok * p.group;
  uint16_t* dst = p.out + static_cast<int64_t>(cut.tok0 + tok) * p.ld_out + (cut.head0 + hh) * 128 + c4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(kv_pack2<F16>(a.x * by, a.y * by), kv_pack2<F16>(a.z * by, a.w * by));
}

template <bool F16>
__global__ void __launch_bounds__(kJThreads, 3) kv_join_kernel(const __grid_constant__ KvAttnArgs p, int R) {
  __shared__ float4 s_sum[kJWarps][kJPer][32];
  __shared__ float2 s_ml[kJWarps][kJPer];
  const int c = blockIdx.x + 1;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const KvCut cut = p.cuts[c];
  if (cut.rows == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c4 = lane * 4;
  const int parts = cut.last - cut.first + 1;
  // This block among those of the unit's parts - 1 cuts.
  const int block = (c - cut.first - 1) * gridDim.y + blockIdx.y, blocks = (parts - 1) * gridDim.y;
  const int groups = (cut.rows + kJPer - 1) / kJPer;
  const int64_t slot0 = 2 * static_cast<int64_t>(cut.first) * R;
  auto at = [&](int i, int r) { return slot0 + (i == 0 ? 1 : 2 * i) * static_cast<int64_t>(R) + r; };  // part i of the unit, row r
  if (parts < kJWarps) {
    for (int g = block * kJWarps + warp; g < groups; g += blocks * kJWarps) {
      const int r0 = g * kJPer;
      // Lane 8 q + i: the maximum and sum of row q in part i; their weights from them.
      const int mi = lane & 7, mq = lane >> 3;
      const float2 ml = mi < parts && r0 + mq < cut.rows ? p.part_ml[at(mi, r0 + mq)] : make_float2(-INFINITY, 0.f);
      float4 s[kJPer], a[2][kJPer];
#pragma unroll
      for (int q = 0; q < kJPer; ++q) {
        s[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        // In bounds for every row of the unit's slot; the first two parts always exist.
        a[0][q] = *reinterpret_cast<const float4*>(p.part_o + at(0, min(r0 + q, cut.rows - 1)) * 128 + c4);
        a[1][q] = *reinterpret_cast<const float4*>(p.part_o + at(1, min(r0 + q, cut.rows - 1)) * 128 + c4);
      }
      float M = ml.x;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, o));
      float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      float L = w * ml.y;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
      w = L != 0.f ? w / L : 0.f;
      for (int i = 0; i < parts; i += 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int q = 0; q < kJPer; ++q) {
            if (i > 0 && i + e < parts)
              a[e][q] = *reinterpret_cast<const float4*>(p.part_o + at(i + e, min(r0 + q, cut.rows - 1)) * 128 + c4);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int q = 0; q < kJPer; ++q) join_fma(s[q], __shfl_sync(0xffffffffu, w, q * 8 + min(i + e, 7)), a[e][q]);
      }
#pragma unroll
      for (int q = 0; q < kJPer; ++q)
        if (r0 + q < cut.rows) join_store<F16>(p, cut, r0 + q, c4, s[q], 1.0f);
    }
    return;
  }
  // A warp's four sums in flight: of four rows, or, where parts are many, of one row.
  const bool many = parts >= kJWarps * kJPer;
  const int per = many ? 1 : kJPer, step = many ? kJWarps * kJPer : kJWarps;
  for (int g = block; g * per < cut.rows; g += blocks) {
    const int r0 = g * per;
    float m[kJPer], l[kJPer];
    float4 s[kJPer];
#pragma unroll
    for (int q = 0; q < kJPer; ++q) {
      m[q] = -INFINITY;
      l[q] = 0.f;
      s[q] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i = warp; i < parts; i += step) {
      float2 ml[kJPer];
      float4 a[kJPer];
#pragma unroll
      for (int q = 0; q < kJPer; ++q) {
        const int part = many ? i + q * kJWarps : i;
        const int64_t k = at(min(part, parts - 1), many ? r0 : min(r0 + q, cut.rows - 1));
        ml[q] = part < parts ? p.part_ml[k] : make_float2(-INFINITY, 0.f);
        a[q] = *reinterpret_cast<const float4*>(p.part_o + k * 128 + c4);
      }
#pragma unroll
      for (int q = 0; q < kJPer; ++q) {
        const float M = max_nan(m[q], ml[q].x);
        if (M == -INFINITY) continue;
        const float keep = ex2(m[q] - M), w = ml[q].x == -INFINITY ? 0.f : ex2(ml[q].x - M);
        l[q] = l[q] * keep + w * ml[q].y;
        s[q].x *= keep; s[q].y *= keep; s[q].z *= keep; s[q].w *= keep;
        join_fma(s[q], w, a[q]);
        m[q] = M;
      }
    }
    __syncthreads();  // the group before has been read
#pragma unroll
    for (int q = 0; q < kJPer; ++q) {
      s_sum[warp][q][lane] = s[q];
      if (lane == 0) s_ml[warp][q] = make_float2(m[q], l[q]);
    }
    __syncthreads();
    if (warp >= per || r0 + warp >= cut.rows) continue;
    // Warp q adds up sums q of all warps, or warp 0 all sums of all warps.
    float M = -INFINITY, L = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const int q0 = warp, q1 = many ? kJPer : warp + 1;
    for (int q = q0; q < q1; ++q)
#pragma unroll
      for (int w = 0; w < kJWarps; ++w) M = max_nan(M, s_ml[w][q].x);
    for (int q = q0; q < q1; ++q)
#pragma unroll
      for (int w = 0; w < kJWarps; ++w) {
        const float2 ml = s_ml[w][q];
        const float k = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
        L += k * ml.y;
        join_fma(sum, k, s_sum[w][q][lane]);
      }
    join_store<F16>(p, cut, r0 + warp, c4, sum, L != 0.f ? 1.0f / L : 0.f);
  }
}

// ------------------------------------------------------------------ host
template <bool F16, bool DIRECT>
cudaError_t launch_rows_t(const KvCacheView& c, KvAttnArgs a, int grid, int cluster, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(kv_rows_kernel<F16, DIRECT>, kRSmem, done);
  if (e != cudaSuccess) return e;
  a.box_rows = std::min(c.block_size, kRKT);
  CUtensorMap mk, mv;
  e = kv_cache_map(&mk, c, c.k, a.box_rows);
  if (e == cudaSuccess) e = kv_cache_map(&mv, c, c.v, a.box_rows);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kRThreads);
  cfg.dynamicSmemBytes = kRSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = DIRECT ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kv_rows_kernel<F16, DIRECT>, mk, mv, a);
}

template <bool F16>
cudaError_t launch_rows(const KvCacheView& c, const KvAttnArgs& a, int grid, int cluster, cudaStream_t s) {
  return a.direct ? launch_rows_t<F16, true>(c, a, grid, cluster, s)
                  : launch_rows_t<F16, false>(c, a, grid, 1, s);
}

template <bool F16>
cudaError_t launch_join(const KvAttnArgs& a, int rows, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.grid - 1, std::max(1, rows / (kJPer * kJWarps * 2)));
  cfg.blockDim = dim3(kJThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  // May start while the main kernel runs; waits for its end before it reads anything of it.
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_join_kernel<F16>, a, rows);
}

}  // namespace

namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* q = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      q = nullptr;
    return reinterpret_cast<EncodeTiledFn>(q);
  }();
  return fn;
}

}  // namespace

// One cache plane: {channel, token of the block, head, block}, boxes of 64 channels x box_rows tokens.
cudaError_t kv_cache_map(CUtensorMap* m, const KvCacheView& c, const void* base, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t bs = static_cast<cuuint64_t>(c.block_size);
  cuuint64_t dims[4] = {128, bs, static_cast<cuuint64_t>(c.heads_kv), static_cast<cuuint64_t>(c.n_blocks)};
  cuuint64_t strides[3] = {256, bs * 256, static_cast<cuuint64_t>(c.block_stride) * 2};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r =
      fn(m, c.f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims,
         strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t kv_query_map(CUtensorMap* m, const KvAttnArgs& a, bool f16, int box_tokens) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(a.heads), static_cast<cuuint64_t>(a.tokens)};
  cuuint64_t strides[2] = {256, static_cast<cuuint64_t>(a.ld_q) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r =
      fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t*>(a.q), dims,
         strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

KvAttnPlan kv_attention_plan(int heads, int heads_kv, int64_t max_new, int num_sms) {
  const int group = heads / heads_kv;
  KvAttnPlan pl{};
  // Measured, 16 requests of 4 tokens x 8 heads a group over 4000 keys: 33.5 us on 32 rows of
  // the first kernel's kind, 27.1 us on the second; 64 such requests 73.4 / 53.6 us.
  if (max_new <= kRRows && max_new * group <= kRRows) {
    pl.unit_rows = kRRows;
    pl.unit_tokens = kRRows / group;
    pl.grid = 2 * num_sms;
  } else {
    pl.unit_rows = kTcRows;
    pl.unit_tokens = 2 * (kTcRows / 2 / group);
    pl.grid = num_sms;
  }
  const size_t part_rows = 2 * static_cast<size_t>(pl.grid) * pl.unit_rows;
  pl.cut_bytes = static_cast<size_t>(pl.grid) * sizeof(KvCut);
  pl.ml_bytes = part_rows * sizeof(float2);  // all multiples of 16
  pl.bytes = pl.cut_bytes + pl.ml_bytes + part_rows * 128 * sizeof(float);
  return pl;
}

cudaError_t launch_kv_attention(const KvCacheView& c, KvAttnArgs a, const KvAttnPlan& plan, void* workspace,
                                cudaStream_t s) {
  a.unit_tokens = plan.unit_tokens;
  a.group_inv = (65536 + a.group - 1) / a.group;
  a.unit_shift = -1;
  for (int i = 0; i <= 8; ++i)
    if (1 << i == plan.unit_tokens) a.unit_shift = i;
  a.grid = plan.grid;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.cuts = reinterpret_cast<KvCut*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + plan.cut_bytes);
  a.part_o = reinterpret_cast<float*>(ws + plan.cut_bytes + plan.ml_bytes);
  const KvAttnForm form = kv_attention_form(a, plan);
  a.direct = form.direct;
  const bool tc = plan.unit_rows == kTcRows;
  const int ctas = form.ctas, cluster = form.cluster;
  cudaError_t e;
  if (tc)
    e = launch_kv_tc(c, a, ctas, cluster, s);
  else
    e = c.f16 ? launch_rows<true>(c, a, ctas, cluster, s) : launch_rows<false>(c, a, ctas, cluster, s);
  if (e != cudaSuccess || a.direct) return e;
  return c.f16 ? launch_join<true>(a, plan.unit_rows, s) : launch_join<false>(a, plan.unit_rows, s);
}

}  // namespace dcpp
