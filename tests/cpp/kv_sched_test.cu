// The arithmetic by which the paged attention kernels share out their work, run on
// the host against counting tile by tile.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "kv_sched.cuh"

using namespace dcpp;

#define REQUIRE(x, ...)                                       \
    do {                                                      \
        if (!(x)) {                                           \
            std::printf("line %d: %s: ", __LINE__, #x);       \
            std::printf(__VA_ARGS__);                         \
            std::printf("\n");                                \
            return 1;                                         \
        }                                                     \
    } while (0)

// Tiles of unit u, from the definition: the keys up to the unit's last token, one tile at least.
template <int KT>
int tiles_of(const KvAttnArgs& p, const KvSeq& s, int u) {
    int64_t keys = s.kv;
    if (p.causal) keys = std::min<int64_t>(keys, static_cast<int64_t>(s.off) + static_cast<int64_t>(u + 1) * p.unit_tokens);
    int n = 0;
    for (int64_t k = 0; k < keys; k += KT) ++n;
    return std::max(n, 1);
}

template <int KT>
int check(int unit_tokens, int causal, int q_len, int kv) {
    KvAttnArgs p{};
    p.unit_tokens = unit_tokens;
    p.unit_shift = -1;
    for (int i = 0; i <= 8; ++i)
        if (1 << i == unit_tokens) p.unit_shift = i;
    p.causal = causal;
    KvSeq s{};
    s.q_len = q_len;
    s.kv = kv;
    s.off = kv - q_len;
    s.units = (q_len + unit_tokens - 1) / unit_tokens;
    int64_t sum = 0;
    for (int u = 0; u <= s.units; ++u) {
        const int64_t got = kv_units_before<KT>(p, s, u);
        REQUIRE(got == sum, "KT %d unit %d causal %d q_len %d kv %d u %d: %lld, not %lld", KT, unit_tokens, causal, q_len, kv, u,
                static_cast<long long>(got), static_cast<long long>(sum));
        if (u < s.units) {
            REQUIRE(kv_unit_tiles<KT>(p, s, u) == tiles_of<KT>(p, s, u), "KT %d unit %d causal %d q_len %d kv %d u %d", KT,
                    unit_tokens, causal, q_len, kv, u);
            sum += tiles_of<KT>(p, s, u);
        }
    }
    return 0;
}

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); };
    // Every unit size that a group of 1 .. 128 heads gives: 16 / group, and 2 (128 / group).
    for (int group = 1; group <= 128; ++group) {
        for (int k = 0; k < 60; ++k) {
            const int q_len = k < 8 ? k : pick(0, k % 3 ? 600 : 9000);
            const int kv = k % 4 == 0 ? q_len : k % 4 == 1 ? pick(0, 300) : k % 4 == 2 ? q_len + pick(0, 20000) : pick(0, q_len + 1);
            for (int causal = 0; causal < 2; ++causal) {
                if (group <= 16 && check<64>(16 / group, causal, q_len, kv)) return 1;
                if (check<128>(2 * (128 / group), causal, q_len, kv)) return 1;
            }
        }
    }
    // Long ones: no intermediate value overflows (the last unit ends at the last key).
    for (int group : {1, 3, 8, 12, 100, 128}) {
        KvAttnArgs p{};
        p.unit_tokens = 2 * (128 / group);
        p.unit_shift = -1;
        for (int i = 0; i <= 8; ++i)
            if (1 << i == p.unit_tokens) p.unit_shift = i;
        p.causal = 1;
        KvSeq s{};
        s.q_len = 1 << 24;
        s.kv = 2147483392;
        s.off = s.kv - s.q_len;
        s.units = (s.q_len + p.unit_tokens - 1) / p.unit_tokens;
        int64_t sum = 0;
        for (int u = 0; u < s.units; ++u) sum += kv_unit_tiles<128>(p, s, u);
        REQUIRE(kv_units_before<128>(p, s, s.units) == sum, "group %d", group);
    }
    // Division by the group.
    for (int group = 1; group <= 128; ++group) {
        KvAttnArgs p{};
        p.group_inv = (65536 + group - 1) / group;
        for (int row = 0; row < 256; ++row) REQUIRE(p.row_token(row) == row / group, "group %d row %d", group, row);
    }
    // The cuts: every tile in one part, parts of equal size but for one tile, and each
    // tile's part found again.
    for (int k = 0; k < 2000; ++k) {
        KvRange r{};
        r.total = pick(1, k % 2 ? 500 : 100000);
        r.parts = std::min<int64_t>(pick(1, 296), r.total);
        r.each = r.total / r.parts;
        r.more = static_cast<int>(r.total - r.each * r.parts);
        REQUIRE(kv_cut(r, 0) == 0 && kv_cut(r, r.parts) == r.total, "total %lld parts %d", static_cast<long long>(r.total), r.parts);
        for (int i = 0; i < r.parts; ++i) {
            const int64_t a = kv_cut(r, i), b = kv_cut(r, i + 1);
            REQUIRE(b - a == r.each || b - a == r.each + 1, "part %d", i);
            REQUIRE(kv_part_of(r, a) == i && kv_part_of(r, b - 1) == i, "part %d of %d", i, r.parts);
        }
    }
    std::printf("ok\n");
    return 0;
}
