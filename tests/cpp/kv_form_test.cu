// The choice between the paged attention's forms, on the host: what a call launches
// stays in proportion to the GPU, whatever its sizes.
#include <cstdio>
#include <random>

#include "kv_form.cuh"

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

constexpr int kSms = 148;

// As kv_attention_plan has it.
KvAttnPlan plan_of(int group, int64_t max_new) {
    KvAttnPlan pl{};
    const bool few = max_new * group <= kRRows;
    pl.unit_rows = few ? kRRows : kTcRows;
    pl.unit_tokens = few ? kRRows / group : 2 * (kTcRows / 2 / group);
    pl.grid = few ? 2 * kSms : kSms;
    return pl;
}

KvAttnForm form(int batch, int heads_kv, int group, int max_new, int64_t max_kv) {
    KvAttnArgs a{};
    a.batch = batch;
    a.heads_kv = heads_kv;
    a.group = group;
    a.max_new = max_new;
    a.max_kv = max_kv;
    return kv_attention_form(a, plan_of(group, max_new));
}

int main() {
    std::mt19937 rng(5);
    auto pick = [&](int bits) { return 1 + static_cast<int>(rng() % (1u << (rng() % bits))); };
    for (int k = 0; k < 200000; ++k) {
        const int batch = pick(21), heads_kv = pick(8), group = std::min(pick(8), 128), max_new = pick(25);
        const int64_t max_kv = 16 * static_cast<int64_t>(pick(27));
        const KvAttnPlan pl = plan_of(group, max_new);
        const KvAttnForm f = form(batch, heads_kv, group, max_new, max_kv);
        REQUIRE(f.ctas > 0 && f.ctas <= 6 * 2 * kSms, "batch %d heads_kv %d group %d max_new %d max_kv %lld: %d CTAs", batch, heads_kv,
                group, max_new, static_cast<long long>(max_kv), f.ctas);
        REQUIRE(f.cluster == 1 || f.cluster == 2 || f.cluster == 4 || f.cluster == 8, "cluster %d", f.cluster);
        if (f.direct) {
            // Every unit that may exist has its CTAs.
            const int64_t units = (max_new + pl.unit_tokens - 1) / pl.unit_tokens;
            REQUIRE(f.direct == units && f.ctas == units * batch * heads_kv * f.cluster, "%d units, %d CTAs", f.direct, f.ctas);
        } else {
            REQUIRE(f.cluster == 1 && f.ctas == pl.grid, "cluster %d, %d CTAs", f.cluster, f.ctas);
        }
    }
    // A prompt among many single tokens: 128000 units that may exist, some 8000 that do.
    REQUIRE(form(1000, 8, 4, 1024, 1024).direct == 0, "mixed step");
    REQUIRE(form(4000, 8, 4, 1, 320).direct == 0, "many single tokens");
    // What the forms are for.
    REQUIRE(form(1, 8, 4, 1, 560).cluster == 8, "one short request");
    REQUIRE(form(4, 8, 4, 512, 560).direct == 8, "ragged prompts");
    REQUIRE(form(64, 8, 4, 1, 8048).direct == 0, "long single tokens");
    std::printf("ok\n");
    return 0;
}
