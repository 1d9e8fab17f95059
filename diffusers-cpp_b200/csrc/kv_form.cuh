// Which form the paged attention takes: tiles and units of its two kernels, and whether
// their units are cut into equal parts or given to a CTA, or a cluster of CTAs, each
// (direct).  Host arithmetic on what the call knows: sizes, not lengths.
#pragma once

#include <algorithm>

#include "kv_cache.cuh"

namespace dcpp {

// The kernel for few query rows (kv_attention.cu).
constexpr int kRRows = 16;  // query rows of a unit
constexpr int kRKT = 64;    // keys of a tile
// Longest share of a CTA in the direct form.  4 requests of up to 1500 keys, 32 heads over 8:
// 9.1 us direct, 14.5 us cut; 1 of 12k keys, 8 heads over 1 (24 tiles to a CTA): 25.1 us
// direct, 12.1 us cut.
constexpr int kRDirectTiles = 12;
// Most units of the direct form, in grids of CTAs that fit at once (two to an SM): a CTA
// starts anew for every unit, and for the units of requests without rows too (some 0.9 us
// each).  Cut / direct, 300 keys, 32 heads over 8: 40 requests (1.1 grids) 14.4 / 12.8 us, 128
// (3.5) 30.8 / 29.6 us, 300 (8.1) 61.0 / 61.6 us, 4000 606 / 723 us, 4000 of which 120 have a
// row 51 / 148 us.
constexpr int kRDirectGrids = 4;

// The tcgen05 kernel for many (kv_attention_tc.cu).
constexpr int kTcKT = 128;           // keys of a tile
constexpr int kTcRows = 256;         // query rows of a unit: two tiles of 128
constexpr int kTcMinTiles = 4;       // fewest key tiles of a part
constexpr int kTcDirectTiles = 8;    // longest unit of the direct form
constexpr int kTcClusterTiles = 16;  // longest share of a CTA in a cluster
// As above (one CTA to an SM).  Every request counts with the units of the one with most new
// tokens, and one that does not exist takes 1.9 us.  Cut / direct, one prompt among single
// tokens over up to 1000 keys: 40 requests, prompt of 128 (4.3 grids) 51 / 39 us, of 256
// (8.6) 49 / 48 us, of 500 (17) 47 / 65 us; over up to 250 keys 23 / 26 us (4.3), 21 / 30 us
// (6.5); 1000 requests, prompt of 500 (432) 627 / 1372 us.
constexpr int kTcDirectGrids = 6;

struct KvAttnForm {
  int direct;   // > 0: the direct form, units of a request at most
  int cluster;  // CTAs that share a unit
  int ctas;
};

// `a`: max_new, batch, heads_kv, group and max_kv of the call.
inline KvAttnForm kv_attention_form(const KvAttnArgs& a, const KvAttnPlan& plan) {
  // Short units (by the table's width, all that the host knows of the lengths) are not
  // cut at all: a CTA for each, no search for its share and no second kernel.  Measured,
  // cut / direct: 1 request x 517 keys 12.9 / 6.8 us, 4 ragged prompts of up to
  // 512 tokens 36.0 / 27.9 us.
  const bool tc = plan.unit_rows == kTcRows;
  const int64_t longest = (a.max_kv + (tc ? kTcKT : kRKT) - 1) / (tc ? kTcKT : kRKT);
  const int64_t units = (a.max_new + plan.unit_tokens - 1) / plan.unit_tokens;
  const int64_t all = units * a.batch * a.heads_kv;
  // Few units: a cluster of CTAs for each, as large as still fits the GPU at once (clusters
  // of 8 one to an SM do not fill every SM).
  int cluster = 1;
  const int64_t at_once = tc ? plan.grid - plan.grid / 8 : plan.grid;
  const bool two = tc && std::min<int64_t>(a.max_new, plan.unit_tokens) * a.group > kTcRows / 2;
  while (cluster < 8 && 2 * cluster * all <= at_once && (two ? 4 * cluster <= longest : cluster < longest)) cluster *= 2;
  // How long a CTA's share may be.  tcgen05 kernel, in clusters: not much longer than the
  // cut form's (one of kTcMinTiles or a balanced one); joining units of two row tiles takes
  // longer.  Measured, cut / clusters: 1 request x 4 tokens x 8 heads a group over 4000 keys
  // 20.5 / 13.7 us, over 11000 keys 20.5 / 24.4 us; 16 such requests over 4000 keys 26.7 /
  // 21.5 us, over 7500 keys 34.9 / 32.0 us; 32 tokens over 8000 keys 22.7 / 25.3 us.
  int64_t most = tc ? kTcDirectTiles : kRDirectTiles;
  if (tc && cluster > 1)
    most = std::min<int64_t>(kTcClusterTiles, std::max<int64_t>(kTcMinTiles, all * longest / plan.grid) + (two ? 2 : 4));
  if (longest <= most * cluster && all <= static_cast<int64_t>(tc ? kTcDirectGrids : kRDirectGrids) * plan.grid)
    return {static_cast<int>(units), cluster, static_cast<int>(all) * cluster};
  return {0, 1, plan.grid};
}

}  // namespace dcpp
