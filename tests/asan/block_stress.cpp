// block_stress.cpp -- drives the host code of the attention block's entry points (aikit_amd/csrc/attention_block.hip)
// for the host AddressSanitizer build (tests/asan/Makefile), as abi_stress.cpp does for the rest: bias tables and maps of
// every size, adapters at ragged shapes, device calls of every form with the scratch grown, capped and shared by 8
// threads, every argument-error path, releases and a close with handles still open. Numerics are checked elsewhere
// (tests/test_gpu_*.py); here results are only checked to be finite.
// Exit status 0 when every check holds; AddressSanitizer aborts on a memory error.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <random>
#include <string>
#include <thread>
#include <vector>

#include "enchip.h"

static int g_fail = 0;

#define CHECK(cond, ...)                                                   \
    do {                                                                   \
        if (!(cond)) {                                                     \
            std::fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__);      \
            std::fprintf(stderr, __VA_ARGS__);                             \
            std::fprintf(stderr, "\n");                                    \
            ++g_fail;                                                      \
        }                                                                  \
    } while (0)

static std::vector<float> randf(std::mt19937 &g, size_t n, float sd = 1.0f) {
    std::normal_distribution<float> d(0.0f, sd);
    std::vector<float> v(n);
    for (auto &x : v) x = d(g);
    return v;
}

// A device copy of host values, for the life of the object.
template <class T>
struct Dev {
    T *p = nullptr;
    size_t n;
    explicit Dev(const std::vector<T> &v) : n(v.size()) {
        CHECK(hipMalloc((void **)&p, n * sizeof(T) + 16) == hipSuccess, "hipMalloc");
        CHECK(hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice) == hipSuccess, "upload");
    }
    Dev(const Dev &) = delete;
    ~Dev() { (void)hipFree(p); }
    bool finite() const {
        std::vector<T> v(n);
        CHECK(hipDeviceSynchronize() == hipSuccess, "synchronize");
        CHECK(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost) == hipSuccess, "download");
        for (auto x : v)
            if (!std::isfinite((double)x)) return false;
        return true;
    }
};

// Tables by the logarithm and by maps, and what is refused of them.
static void tables(enchip_ctx *ctx, std::mt19937 &g) {
    const int64_t shapes[][3] = {{4, 1, 2}, {32, 12, 128}, {16, 7, 1000}, {64, 3, 1 << 16}, {8, 400, 5}};
    for (auto &s : shapes) {
        const int64_t buckets = s[0], heads = s[1], reach = s[2];
        auto t = randf(g, (size_t)(buckets * heads));
        t[0] = -std::numeric_limits<float>::infinity();
        enchip_relpos b = 0, m = 0;
        CHECK(enchip_relpos_create(ctx, t.data(), buckets, heads, reach, &b) == ENCHIP_OK && b, "relpos: %s", enchip_last_error(ctx));
        std::vector<int32_t> map((size_t)(2 * reach + 1));
        for (auto &x : map) x = (int32_t)(g() % buckets);
        CHECK(enchip_relpos_create_map(ctx, t.data(), buckets, heads, map.data(), reach, &m) == ENCHIP_OK && m, "map");
        map.back() = (int32_t)buckets;
        enchip_relpos bad = 7;
        CHECK(enchip_relpos_create_map(ctx, t.data(), buckets, heads, map.data(), reach, &bad) == ENCHIP_ERR_ARG && bad == 0, "bucket");
        t.back() = std::nanf("");
        CHECK(enchip_relpos_create(ctx, t.data(), buckets, heads, reach, &bad) == ENCHIP_ERR_ARG, "NaN");
        CHECK(enchip_relpos_release(ctx, b) == ENCHIP_OK && enchip_relpos_release(ctx, b) == ENCHIP_ERR_HANDLE, "release");
        CHECK(enchip_relpos_release(ctx, m) == ENCHIP_OK, "release map");
    }
    auto t = randf(g, 64);
    int32_t one = 0;
    enchip_relpos b = 0;
    CHECK(enchip_relpos_create_map(ctx, t.data(), 1, 64, &one, 0, &b) == ENCHIP_OK, "reach 0");  // left for the close
    CHECK(enchip_relpos_create(ctx, t.data(), 7, 2, 20, &b) == ENCHIP_ERR_ARG, "odd buckets");
    CHECK(enchip_relpos_create(ctx, t.data(), 8, 2, 2, &b) == ENCHIP_ERR_ARG, "short reach");
    CHECK(enchip_relpos_create(ctx, t.data(), 8, 2, (int64_t)1 << 40, &b) == ENCHIP_ERR_ARG, "long reach");
    CHECK(enchip_relpos_create(ctx, t.data(), 8, (int64_t)1 << 60, 20, &b) == ENCHIP_ERR_ARG, "heads");
    CHECK(enchip_relpos_create(ctx, nullptr, 8, 2, 20, &b) == ENCHIP_ERR_ARG, "null");
    CHECK(enchip_relpos_create(ctx, t.data(), 8, 2, 20, nullptr) == ENCHIP_ERR_ARG, "null out");
    CHECK(enchip_relpos_create_map(ctx, t.data(), 8, 2, nullptr, 3, &b) == ENCHIP_ERR_ARG, "null map");
    CHECK(enchip_relpos_create_map(ctx, t.data(), 8, 2, &one, -1, &b) == ENCHIP_ERR_ARG, "reach -1");
}

// Head norms, attention in every form, pooling of spans.
static void attention(enchip_ctx *ctx, std::mt19937 &g) {
    const int64_t shapes[][5] = {  // heads, key heads, head_dim, rows, sequences
        {3, 3, 32, 1, 1}, {4, 2, 64, 70, 3}, {8, 1, 128, 300, 2}, {2, 2, 64, 3000, 1}, {32, 32, 64, 700, 2}, {12, 12, 64, 40, 90}};
    for (auto &s : shapes) {
        const int64_t H = s[0], KV = s[1], hd = s[2], L = s[3], S = s[4], W = (H + 2 * KV) * hd, rows = S * L;
        Dev<float> x(randf(g, (size_t)(rows * W))), out(std::vector<float>((size_t)(rows * H * hd)));
        Dev<float> gain(randf(g, (size_t)hd)), pooled(std::vector<float>((size_t)(S * H * hd)));
        std::vector<int32_t> sp, pos((size_t)rows);
        for (int64_t z = 0; z < S; ++z) {
            const int32_t n = (int32_t)(g() % (L + 1));
            sp.push_back((int32_t)(z * L));
            sp.push_back((int32_t)(z * L) + (z ? n : (int32_t)L));
        }
        for (int64_t i = 0; i < rows; ++i) pos[(size_t)i] = (int32_t)(i % L);
        Dev<int32_t> spans(sp), dpos(pos);
        auto t = randf(g, (size_t)(32 * H));
        enchip_relpos b = 0;
        enchip_rope r = 0;
        CHECK(enchip_relpos_create(ctx, t.data(), 32, H, 128, &b) == ENCHIP_OK, "relpos");
        CHECK(enchip_rope_create(ctx, hd, 10000.0, ENCHIP_ROPE_NONE, 1.0, 0, &r) == ENCHIP_OK, "rope: %s", enchip_last_error(ctx));
        for (enchip_rope rope : {r, (enchip_rope)0})
            CHECK(enchip_head_norm_rope_rows_dev(ctx, rope, ENCHIP_ROPE_HALF, x.p, W, x.p, W, S, L, H, KV, hd, gain.p, gain.p, 1e-6,
                                                 dpos.p, 0, nullptr) == ENCHIP_OK, "head norm: %s", enchip_last_error(ctx));
        const float scale = 1.0f / std::sqrt((float)hd);
        for (int i = 0; i < 4; ++i) {
            const bool by_spans = i & 1;
            CHECK(enchip_attention_bias_dev(ctx, i & 2 ? b : 0, x.p, W, x.p + H * hd, W, x.p + (H + KV) * hd, W, out.p, H * hd,
                                            by_spans ? spans.p : nullptr, S, by_spans ? rows : L, H, KV, hd, scale, nullptr) == ENCHIP_OK,
                  "attention: %s", enchip_last_error(ctx));
            CHECK(out.finite(), "attention %d", i);
        }
        CHECK(enchip_pool_mean_l2_spans_dev(ctx, out.p, H * hd, rows, spans.p, S, H * hd, pooled.p, H * hd, nullptr) == ENCHIP_OK, "pool");
        CHECK(pooled.finite(), "pooled");
        CHECK(enchip_attention_bias_dev(ctx, 12345, x.p, W, x.p, W, x.p, W, out.p, H * hd, nullptr, S, L, H, KV, hd, scale, nullptr) ==
                  ENCHIP_ERR_HANDLE, "handle");
        CHECK(enchip_attention_bias_dev(ctx, b, x.p, W, x.p, W, x.p, W, out.p, H * hd, nullptr, S, L, H + 1, KV, hd, scale, nullptr) ==
                  ENCHIP_ERR_ARG, "heads");
        CHECK(enchip_attention_bias_dev(ctx, b, x.p, W, x.p, W, x.p, W, out.p, H * hd, nullptr, (int64_t)1 << 62, L, H, KV, hd, scale,
                                        nullptr) == ENCHIP_ERR_ARG, "sequences");
        CHECK(enchip_pool_mean_l2_spans_dev(ctx, out.p, H * hd, rows, nullptr, S, H * hd, pooled.p, H * hd, nullptr) == ENCHIP_ERR_ARG, "spans");
        CHECK(enchip_head_norm_rope_rows_dev(ctx, 12345, 0, x.p, W, x.p, W, S, L, H, KV, hd, gain.p, gain.p, 1e-6, nullptr, 0, nullptr) ==
                  ENCHIP_ERR_HANDLE, "rope handle");
        CHECK(enchip_head_norm_rope_rows_dev(ctx, 0, 0, x.p, W, x.p, W, S, L, H, KV, hd, gain.p, gain.p, 0.0, nullptr, 0, nullptr) ==
                  ENCHIP_ERR_ARG, "eps");
        CHECK(enchip_relpos_release(ctx, b) == ENCHIP_OK && enchip_rope_release(ctx, r) == ENCHIP_OK, "release");
    }
    // keys in parts need scratch: declined under a cap, whole again without it
    const int64_t L = 6000, hd = 64;
    Dev<float> x(randf(g, (size_t)(L * 3 * hd))), out(std::vector<float>((size_t)(L * hd)));
    auto call = [&] {
        return enchip_attention_bias_dev(ctx, 0, x.p, 3 * hd, x.p + hd, 3 * hd, x.p + 2 * hd, 3 * hd, out.p, hd, nullptr, 1, L, 1, 1, hd, 0.1f,
                                         nullptr);
    };
    CHECK(call() == ENCHIP_OK, "parts: %s", enchip_last_error(ctx));
    CHECK(enchip_set_scratch_limit(ctx, 1000) == ENCHIP_OK && call() == ENCHIP_ERR_OOM, "parts under a cap");
    CHECK(enchip_set_scratch_limit(ctx, 0) == ENCHIP_OK && call() == ENCHIP_OK && out.finite(), "after the cap");
}

// Sets of adapters at ragged shapes, slots rewritten, both calls.
static void adapters(enchip_ctx *ctx, std::mt19937 &g) {
    const int64_t shapes[][5] = {  // rows, K, N, rank, slots
        {1, 1, 1, 1, 1}, {16, 384, 512, 8, 5}, {33, 100, 70, 7, 3}, {300, 257, 129, 40, 4}, {20, 64, 96, 256, 2}, {9, 4100, 64, 8, 2}};
    for (auto &s : shapes) {
        const int64_t M = s[0], K = s[1], N = s[2], R = s[3], slots = s[4];
        enchip_adapters h = 0;
        CHECK(enchip_adapters_create(ctx, K, N, R, slots, &h) == ENCHIP_OK && h, "create: %s", enchip_last_error(ctx));
        for (int64_t z = 0; z < slots; ++z) {
            auto A = randf(g, (size_t)(R * K), 0.05f), B = randf(g, (size_t)(N * R), 0.05f);
            CHECK(enchip_adapters_set(ctx, h, z, A.data(), B.data(), 0.5f) == ENCHIP_OK, "set: %s", enchip_last_error(ctx));
            CHECK(enchip_adapters_set(ctx, h, slots + z, A.data(), B.data(), 0.5f) == ENCHIP_ERR_ARG, "slot");
            A.back() = INFINITY;
            CHECK(enchip_adapters_set(ctx, h, z, A.data(), B.data(), 0.5f) == ENCHIP_ERR_ARG, "infinite A");
            A.back() = 0.0f;
            CHECK(enchip_adapters_set(ctx, h, z, A.data(), B.data(), INFINITY) == ENCHIP_ERR_ARG, "infinite scale");
            CHECK(enchip_adapters_set(ctx, h, z, nullptr, B.data(), 1.0f) == ENCHIP_ERR_ARG, "null A");
        }
        std::vector<int8_t> wq((size_t)(N * K));
        for (auto &q : wq) q = (int8_t)((int)(g() % 255) - 127);
        std::vector<float> ws((size_t)N, 0.004f);
        enchip_weight w = 0;
        CHECK(enchip_weight_register(ctx, wq.data(), ws.data(), N, K, &w) == ENCHIP_OK, "weight");
        std::vector<int32_t> ids((size_t)M);
        for (auto &i : ids) i = (int32_t)(g() % (slots + 2)) - 1;
        Dev<int32_t> di(ids);
        Dev<float> a(randf(g, (size_t)(M * K))), y(randf(g, (size_t)(M * N)));
        CHECK(enchip_adapters_add_dev(ctx, h, a.p, K, M, di.p, y.p, N, y.p, N, nullptr) == ENCHIP_OK, "add: %s", enchip_last_error(ctx));
        CHECK(y.finite(), "add");
        for (int act : {ENCHIP_ACT_NONE, ENCHIP_ACT_GELU}) {
            CHECK(enchip_w8a8_linear_adapters_dev(ctx, w, h, a.p, M, di.p, nullptr, act, y.p, nullptr) == ENCHIP_OK, "linear: %s",
                  enchip_last_error(ctx));
            CHECK(y.finite(), "linear");
        }
        CHECK(enchip_w8a8_linear_adapters_dev(ctx, w, h, a.p, M, di.p, nullptr, 9, y.p, nullptr) == ENCHIP_ERR_ARG, "act");
        CHECK(enchip_w8a8_linear_adapters_dev(ctx, w, h, a.p, M, nullptr, nullptr, 0, y.p, nullptr) == ENCHIP_ERR_ARG, "null ids");
        CHECK(enchip_w8a8_linear_adapters_dev(ctx, w, 999, a.p, M, di.p, nullptr, 0, y.p, nullptr) == ENCHIP_ERR_HANDLE, "handle");
        CHECK(enchip_adapters_add_dev(ctx, h, a.p, K - 1, M, di.p, y.p, N, y.p, N, nullptr) == ENCHIP_ERR_ARG, "pitch");
        CHECK(enchip_weight_release(ctx, w) == ENCHIP_OK, "release weight");
        CHECK(enchip_adapters_release(ctx, h) == ENCHIP_OK && enchip_adapters_release(ctx, h) == ENCHIP_ERR_HANDLE, "release");
    }
    enchip_adapters h = 0;
    CHECK(enchip_adapters_create(ctx, 64, 64, 4, 2, &h) == ENCHIP_OK, "create");  // left for the close
    CHECK(enchip_adapters_create(ctx, 64, 64, 257, 2, &h) == ENCHIP_ERR_ARG && h == 0, "rank");
    CHECK(enchip_adapters_create(ctx, 131072, 1 << 24, 256, 65536, &h) == ENCHIP_ERR_ARG, "bytes");
    CHECK(enchip_adapters_create(ctx, 64, 64, 4, 2, nullptr) == ENCHIP_ERR_ARG, "null out");
}

// 8 threads on one context: handles made, used and released, and messages of their own failures.
static void threads(enchip_ctx *ctx) {
    std::vector<std::thread> ts;
    std::vector<int> bad(8, 0);
    for (int t = 0; t < 8; ++t)
        ts.emplace_back([ctx, t, &bad] {
            std::mt19937 g(200 + t);
            const int64_t K = 64 + 32 * t, N = 96, M = 40;
            Dev<float> a(randf(g, (size_t)(M * K))), y(randf(g, (size_t)(M * N)));
            Dev<int32_t> ids(std::vector<int32_t>((size_t)M, 0));
            for (int it = 0; it < 10; ++it) {
                enchip_adapters h = 0;
                enchip_relpos b = 0;
                auto A = randf(g, (size_t)(4 * K)), B = randf(g, (size_t)(N * 4)), table = randf(g, 64);
                if (enchip_adapters_create(ctx, K, N, 4, 2, &h) != ENCHIP_OK) bad[t]++;
                if (enchip_adapters_set(ctx, h, 0, A.data(), B.data(), 1.0f) != ENCHIP_OK) bad[t]++;
                if (enchip_adapters_add_dev(ctx, h, a.p, K, M, ids.p, y.p, N, y.p, N, nullptr) != ENCHIP_OK) bad[t]++;
                if (enchip_relpos_create(ctx, table.data(), 32, 2, 50, &b) != ENCHIP_OK) bad[t]++;
                if (enchip_adapters_set(ctx, h, 50 + t, A.data(), B.data(), 1.0f) != ENCHIP_ERR_ARG) bad[t]++;
                if (std::string(enchip_last_error(ctx)).find("slot " + std::to_string(50 + t)) == std::string::npos) bad[t]++;
                if (enchip_relpos_release(ctx, b) != ENCHIP_OK || enchip_adapters_release(ctx, h) != ENCHIP_OK) bad[t]++;
            }
        });
    for (auto &th : ts) th.join();
    for (int t = 0; t < 8; ++t) CHECK(bad[t] == 0, "thread %d: %d failures", t, bad[t]);
}

int main() {
    enchip_ctx *ctx = nullptr;
    if (enchip_open(0, &ctx) != ENCHIP_OK) {
        std::fprintf(stderr, "enchip_open(0) failed: %s\n", enchip_last_error(nullptr));
        return 2;
    }
    void *stream = nullptr;
    CHECK(enchip_stream(ctx, &stream) == ENCHIP_OK && stream && enchip_stream(ctx, nullptr) == ENCHIP_ERR_ARG, "stream");
    std::mt19937 g(11);
    auto part = [&](const char *name, auto fn) {
        std::printf("%s\n", name);
        std::fflush(stdout);
        fn();
        std::printf("%s: %d failures so far\n", name, g_fail);
        std::fflush(stdout);
    };
    part("tables", [&] { tables(ctx, g); });
    part("attention", [&] { attention(ctx, g); });
    part("adapters", [&] { adapters(ctx, g); });
    part("threads", [&] { threads(ctx); });
    CHECK(enchip_close(ctx) == ENCHIP_OK, "close");  // with a table and a set still open
    std::printf("block_stress: %s (%d failures)\n", g_fail ? "FAILED" : "ok", g_fail);
    std::fflush(nullptr);
    std::_Exit(g_fail ? 1 : 0);  // without the exit-time destructors, as abi_stress.cpp says
}
