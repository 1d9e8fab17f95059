// The paged key / value cache through include/dcpp.hpp.
//   kv_test cpu   entry points without a context
//   kv_test gpu   one step of two requests
#include <cstdio>
#include <cstring>
#include <vector>

#include "dcpp.hpp"

#define REQUIRE(x)                                              \
    do {                                                        \
        if (!(x)) {                                             \
            std::fprintf(stderr, "line %d: %s\n", __LINE__, #x); \
            return 1;                                           \
        }                                                       \
    } while (0)

static int cpu() {
    dcpp_kv_cache c{};
    size_t n = 0;
    REQUIRE(dcpp_kv_plan(nullptr, &c, 1, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1, nullptr, nullptr, 0, nullptr,
                         nullptr) == DCPP_ERR_INVALID_ARG);
    REQUIRE(dcpp_kv_store(nullptr, &c, 1, 1, nullptr, 0, nullptr, nullptr, 0, DCPP_ROPE_NONE, 1, nullptr, nullptr, nullptr, 0) ==
            DCPP_ERR_INVALID_ARG);
    REQUIRE(dcpp_kv_attention_workspace(nullptr, &c, 1, 1, &n) == DCPP_ERR_INVALID_ARG);
    REQUIRE(dcpp_kv_attention(nullptr, &c, 1, 1, 1, nullptr, 0, nullptr, nullptr, nullptr, 1, 1, 1, 1.0f, nullptr, 0, nullptr,
                              0) == DCPP_ERR_INVALID_ARG);
    return 0;
}

template <class T>
static T* device(dcpp::CudaRuntime& rt, const std::vector<T>& v) {
    T* p = static_cast<T*>(rt.alloc(v.size() * sizeof(T)));
    rt.memcpy(p, v.data(), v.size() * sizeof(T));
    return p;
}

static int gpu() {
    dcpp::CudaRuntime rt(0);
    const int64_t heads = 4, heads_kv = 2, block = 16, n_blocks = 6, width = 3, tokens = 20, cols = (heads + 2 * heads_kv) * 128;
    std::vector<uint16_t> zeros(n_blocks * heads_kv * block * 128, 0), qkv(tokens * cols), q(tokens * heads * 128), out(q.size(), 1);
    for (size_t i = 0; i < qkv.size(); ++i) qkv[i] = static_cast<uint16_t>(0x3F00 + (i * 37) % 251);  // bf16, 0.5 .. 1.97
    dcpp_kv_cache c{};
    c.type = DCPP_TYPE_BF16;
    c.block_size = block;
    c.n_blocks = n_blocks;
    c.heads_kv = heads_kv;
    c.head_dim = 128;
    c.d_k = device(rt, zeros);
    c.d_v = device(rt, zeros);
    auto* cached = device<int32_t>(rt, {0, 0});
    auto* n_new = device<int32_t>(rt, {1, 19});
    auto* ring = device<int32_t>(rt, {5, 3, 1, 0, 2, 4});
    auto* counters = device<int64_t>(rt, {0, 6});
    auto* table = device<int32_t>(rt, std::vector<int32_t>(2 * width, -1));
    auto* seq = device<int32_t>(rt, {0, 0});
    auto* cu = device<int32_t>(rt, {0, 0, 0});
    auto* slots = device<int32_t>(rt, std::vector<int32_t>(tokens));
    auto* pos = device<int32_t>(rt, std::vector<int32_t>(tokens));
    auto* dqkv = device(rt, qkv);
    auto* dq = device(rt, q);
    auto* dout = device(rt, out);
    rt.kv_plan(c, 2, cached, n_new, ring, counters, counters, table, width, seq, cu, tokens, slots, pos);
    rt.kv_store(c, tokens, heads, dqkv, nullptr, nullptr, 1e-6f, DCPP_ROPE_NEOX, 1e6f, pos, slots, dq);
    const size_t bytes = rt.kv_attention_workspace(c, heads, 19);
    void* ws = rt.alloc(bytes);
    rt.kv_attention(c, 2, tokens, heads, dq, cu, seq, table, width, 19, true, 0.088388f, ws, bytes, dout);
    rt.synchronize();
    std::vector<int32_t> got(2 * width);
    rt.memcpy(got.data(), table, got.size() * 4);
    REQUIRE(got[0] == 5 && got[1] == -1 && got[3] == 3 && got[4] == 1 && got[5] == -1);
    rt.memcpy(out.data(), dout, out.size() * 2);
    // Both requests' first tokens attend to themselves alone: their output is their value row.
    for (int64_t t : {0, 1})
        for (int64_t h = 0; h < heads; ++h)
            REQUIRE(std::memcmp(&out[(t * heads + h) * 128], &qkv[t * cols + (heads + heads_kv + h / 2) * 128], 256) == 0);
    bool refused = false;
    try {
        rt.kv_attention(c, 2, tokens, heads, dq, cu, seq, table, width, 19, true, 0.088388f, ws, bytes - 16, dout);
    } catch (const dcpp::Error& e) {
        refused = e.status == DCPP_ERR_INVALID_ARG;
    }
    REQUIRE(refused);
    for (void* p : {c.d_k, c.d_v, static_cast<void*>(cached), static_cast<void*>(n_new), static_cast<void*>(ring),
                    static_cast<void*>(counters), static_cast<void*>(table), static_cast<void*>(seq), static_cast<void*>(cu),
                    static_cast<void*>(slots), static_cast<void*>(pos), static_cast<void*>(dqkv), static_cast<void*>(dq),
                    static_cast<void*>(dout), ws})
        rt.free(p);
    return 0;
}

int main(int argc, char** argv) {
    if (argc != 2) return 2;
    try {
        return std::strcmp(argv[1], "gpu") == 0 ? gpu() : cpu();
    } catch (const std::exception& e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
}
