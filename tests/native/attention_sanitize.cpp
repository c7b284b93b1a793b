// attention_sanitize.cpp -- drives the attention entry points of libtkv_hip's C
// ABI (caches, rotation and append, prompts, paged) with the library's host code
// built with AddressSanitizer and UndefinedBehaviorSanitizer, as host_sanitize.cpp
// does for the rest.  Without a GPU: argument checks and the no-device paths, at
// sizes whose products would overflow.  With one: small calls of every kernel
// choice (any layout, streaming, tiles; split and not), checked where a row sees
// a single key and its output is that key's value.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "../../include/tkv_hip.h"

static int g_fail = 0;
#define CHECK(cond, what)                                                  \
    do {                                                                   \
        if (!(cond)) {                                                     \
            char buf[256];                                                 \
            tkv_hip_last_error(buf, sizeof(buf));                          \
            fprintf(stderr, "attention_sanitize: FAIL %s (last error: %s)\n", what, buf); \
            g_fail = 1;                                                    \
        }                                                                  \
    } while (0)

static const int64_t kHuge = INT64_MAX;

// Refused before any device is touched; no pointer here is read.
static void refusals() {
    int64_t h = 0;
    void* p = reinterpret_cast<void*>(16);
    const int32_t* ip = static_cast<int32_t*>(p);
    const int64_t* lp = static_cast<int64_t*>(p);
    const float* fp = static_cast<float*>(p);
    float* out = static_cast<float*>(p);
    const tkv_hip_rows r = {p, 64, 64}, none = {nullptr, 64, 64};
    const auto create = [&](int32_t type, int64_t pages, int64_t page, int64_t heads, int64_t d, void* k, float* ks) {
        return tkv_hip_kv_create(0, type, pages, page, heads, d, k, k, ks, ks, &h);
    };
    CHECK(create(7, 1, 16, 1, 64, nullptr, nullptr) == TKV_HIP_BAD_ARG, "cache of an unknown type");
    CHECK(create(TKV_HIP_F32, 0, 16, 1, 64, nullptr, nullptr) == TKV_HIP_BAD_ARG, "cache of no pages");
    CHECK(create(TKV_HIP_F32, kHuge, kHuge, 1, 64, nullptr, nullptr) == TKV_HIP_BAD_ARG, "cache of 2^126 slots");
    CHECK(create(TKV_HIP_F32, 1 << 16, 1 << 14, 65535, 64, nullptr, nullptr) == TKV_HIP_BAD_ARG,
          "cache of 2^46 rows");
    CHECK(create(TKV_HIP_F32, 1, 16, 1, 257, nullptr, nullptr) == TKV_HIP_BAD_ARG, "cache of heads of 257");
    CHECK(create(TKV_HIP_I8, 1, 16, 1, 64, p, nullptr) == TKV_HIP_BAD_ARG, "int8 pools without scales");
    CHECK(create(TKV_HIP_F32, 1, 16, 1, 64, p, out) == TKV_HIP_BAD_ARG, "f32 pools with scales");
    CHECK(tkv_hip_kv_create(0, TKV_HIP_F32, 1, 16, 1, 64, nullptr, nullptr, nullptr, nullptr, nullptr) ==
              TKV_HIP_BAD_ARG,
          "cache without an output");
    CHECK(tkv_hip_kv_free(0) == TKV_HIP_OK, "kv_free(0)");
    CHECK(tkv_hip_kv_info(0, nullptr, nullptr, nullptr, nullptr) == TKV_HIP_BAD_ARG, "kv_info(0)");

    const double freq[128] = {1.0};
    for (int64_t rot : {int64_t(0), int64_t(3), int64_t(258), kHuge})
        CHECK(tkv_hip_dev_rope_table(0, 4, rot, freq, 1.0, out) == TKV_HIP_BAD_ARG, "table of a bad rot_dim");
    CHECK(tkv_hip_dev_rope_table(0, kHuge, 64, freq, 1.0, out) == TKV_HIP_BAD_ARG, "table of 2^63 positions");
    CHECK(tkv_hip_dev_rope_table(0, 4, 64, nullptr, 1.0, out) == TKV_HIP_BAD_ARG, "table without frequencies");
    CHECK(tkv_hip_dev_rope_table(0, 0, 64, freq, 1.0, nullptr) == TKV_HIP_OK, "table of no positions");

    const auto append = [&](int32_t in, int64_t tokens, int64_t hq, int64_t hkv, int64_t d, const tkv_hip_rows* q,
                            const float* table, int64_t rot, int32_t layout) {
        return tkv_hip_dev_rope_append(0, in, tokens, hq, hkv, d, q, &r, &r, ip, table, 8, rot, layout, q, nullptr,
                                       TKV_HIP_F32, 0, lp);
    };
    CHECK(append(TKV_HIP_I8, 1, 1, 1, 64, &r, nullptr, 0, 0) == TKV_HIP_BAD_ARG, "append of int8 rows");
    CHECK(append(TKV_HIP_F32, -1, 1, 1, 64, &r, nullptr, 0, 0) == TKV_HIP_BAD_ARG, "append of -1 tokens");
    CHECK(append(TKV_HIP_F32, kHuge, 65535, 65535, 64, &r, nullptr, 0, 0) == TKV_HIP_BAD_ARG,
          "append of 2^63 tokens");
    CHECK(append(TKV_HIP_F32, 1, kHuge, 1, 64, &r, nullptr, 0, 0) == TKV_HIP_BAD_ARG, "append of 2^63 heads");
    CHECK(append(TKV_HIP_F32, 1, 1, 1, 64, &none, nullptr, 0, 0) == TKV_HIP_BAD_ARG, "append of NULL rows");
    CHECK(append(TKV_HIP_F32, 1, 1, 1, 64, &r, fp, 66, 0) == TKV_HIP_BAD_ARG, "rot_dim above the head");
    CHECK(append(TKV_HIP_F32, 1, 1, 1, 64, &r, fp, 64, 9) == TKV_HIP_BAD_ARG, "unknown layout");

    const auto prompt = [&](int64_t tokens, int64_t tokens_k, int64_t hq, int64_t hkv, int64_t d, int64_t seqs,
                            const tkv_hip_rows* q, float scale, int64_t window) {
        return tkv_hip_dev_attention_prompt(0, TKV_HIP_F32, tokens, tokens_k, hq, hkv, d, seqs, q, &r, &r, &r,
                                            TKV_HIP_F32, ip, nullptr, scale, 1, window);
    };
    CHECK(prompt(kHuge, 1, 1, 1, 64, 1, &r, 1.0f, 0) == TKV_HIP_BAD_ARG, "prompt of 2^63 tokens");
    CHECK(prompt(1, kHuge, 1, 1, 64, 1, &r, 1.0f, 0) == TKV_HIP_BAD_ARG, "prompt of 2^63 keys");
    CHECK(prompt(1, 1, 3, 2, 64, 1, &r, 1.0f, 0) == TKV_HIP_BAD_ARG, "prompt of uneven heads");
    CHECK(prompt(1, 1, 1, kHuge, 64, 1, &r, 1.0f, 0) == TKV_HIP_BAD_ARG, "prompt of 2^63 key heads");
    CHECK(prompt(1, 1, 1, 1, 64, kHuge, &r, 1.0f, 0) == TKV_HIP_BAD_ARG, "prompt of 2^63 sequences");
    CHECK(prompt(1, 1, 1, 1, 64, 1, &none, 1.0f, 0) == TKV_HIP_BAD_ARG, "prompt of NULL rows");
    CHECK(prompt(1, 1, 1, 1, 64, 1, &r, -1.0f, 0) == TKV_HIP_BAD_ARG, "prompt of a negative scale");
    CHECK(prompt(1, 1, 1, 1, 64, 1, &r, 1.0f, -1) == TKV_HIP_BAD_ARG, "prompt of a negative window");
    CHECK(tkv_hip_dev_attention_paged(0, TKV_HIP_F32, 1, 1, 0, 1, &r, &r, TKV_HIP_F32, ip, 1, nullptr, ip, 0, 0, 1.0f,
                                      1, 0) == TKV_HIP_BAD_ARG,
          "paged without a cache");
}

static void no_device() {
    int64_t h = 0;
    void* p = reinterpret_cast<void*>(16);
    const tkv_hip_rows r = {p, 64, 64};
    const double freq[32] = {1.0};
    CHECK(tkv_hip_kv_create(0, TKV_HIP_F32, 1, 16, 1, 64, nullptr, nullptr, nullptr, nullptr, &h) ==
              TKV_HIP_NO_DEVICE,
          "cache without a device");
    CHECK(tkv_hip_dev_rope_table(0, 4, 64, freq, 1.0, static_cast<float*>(p)) == TKV_HIP_NO_DEVICE,
          "table without a device");
    CHECK(tkv_hip_dev_rope_append(0, TKV_HIP_F32, 1, 1, 0, 64, &r, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, &r,
                                  nullptr, TKV_HIP_F32, 0, nullptr) == TKV_HIP_NO_DEVICE,
          "append without a device");
    CHECK(tkv_hip_dev_attention_prompt(0, TKV_HIP_F32, 1, 1, 1, 1, 64, 1, &r, &r, &r, &r, TKV_HIP_F32,
                                       static_cast<int32_t*>(p), nullptr, 1.0f, 1, 0) == TKV_HIP_NO_DEVICE,
          "prompt without a device");
}

template <typename T>
static T* put(int64_t ctx, const std::vector<T>& x) {
    void* p = nullptr;
    CHECK(tkv_hip_malloc(ctx, (int64_t)(x.size() * sizeof(T)), &p) == TKV_HIP_OK, "malloc");
    CHECK(tkv_hip_memcpy_h2d(ctx, p, x.data(), (int64_t)(x.size() * sizeof(T))) == TKV_HIP_OK, "upload");
    return static_cast<T*>(p);
}

static void on_device() {
    int64_t ctx = 0;
    CHECK(tkv_hip_ctx_create(0, &ctx) == TKV_HIP_OK, "ctx_create");
    const int hq = 4, hkv = 2, page = 16, pages = 200;
    for (int d : {64, 20})
        for (int32_t type : {TKV_HIP_F32, TKV_HIP_I8}) {
            // `keys` tokens appended one behind the other, the last `n` of them queried
            // with a window of one: each output is its own token's value
            const int keys = 3000, row = (hq + 2 * hkv) * d;
            std::vector<float> x((size_t)keys * row);
            for (size_t i = 0; i < x.size(); i++) x[i] = (float)((int)(i * 37 % 255) - 127);
            // int8: a row whose largest element is 127 has codes that are its elements,
            // times a scale within an ulp of 1
            for (int t = 0; t < keys; t++)
                for (int h = 0; h < hq + 2 * hkv; h++) x[(size_t)t * row + h * d] = 127.0f;
            std::vector<int64_t> slots(keys);
            std::vector<int32_t> table(pages), lens = {keys}, pos(keys);
            for (int t = 0; t < keys; t++) slots[t] = t, pos[t] = t;
            for (int i = 0; i < pages; i++) table[i] = i;
            float* dx = put(ctx, x);
            int64_t* ds = put(ctx, slots);
            int32_t *dt = put(ctx, table), *dl = put(ctx, lens), *dp = put(ctx, pos);
            int64_t cache = 0;
            CHECK(tkv_hip_kv_create(ctx, type, pages, page, hkv, d, nullptr, nullptr, nullptr, nullptr, &cache) ==
                      TKV_HIP_OK,
                  "kv_create");
            const tkv_hip_rows q = {dx, row, d}, k = {dx + hq * d, row, d}, v = {dx + (hq + hkv) * d, row, d};
            CHECK(tkv_hip_dev_rope_append(ctx, TKV_HIP_F32, keys, hq, hkv, d, &q, &k, &v, nullptr, nullptr, 0, 0, 0,
                                          nullptr, nullptr, TKV_HIP_F32, cache, ds) == TKV_HIP_OK,
                  "append");
            for (int n : {1, 5, 100, 1500}) {
                std::vector<int32_t> cu = {0, n};
                int32_t* dc = put(ctx, cu);
                float* dy = put(ctx, std::vector<float>((size_t)n * hq * d, -1.0f));
                const tkv_hip_rows qn = {dx + (size_t)(keys - n) * row, row, d}, y = {dy, hq * d, d};
                for (int64_t window : {int64_t(1), int64_t(0)})
                    CHECK(tkv_hip_dev_attention_paged(ctx, TKV_HIP_F32, n, hq, cache, 1, &qn, &y, TKV_HIP_F32, dt,
                                                      pages, n > 1 ? dc : nullptr, dl, n, keys, 0.01f, 1,
                                                      1 - window) == TKV_HIP_OK,
                          "attention_paged");
                std::vector<float> got((size_t)n * hq * d);
                CHECK(tkv_hip_memcpy_d2h(ctx, got.data(), dy, (int64_t)(got.size() * 4)) == TKV_HIP_OK, "download");
                float worst = 0.0f;
                for (int t = 0; t < n; t++)
                    for (int h = 0; h < hq; h++)
                        for (int e = 0; e < d; e++) {
                            const float want = x[(size_t)(keys - n + t) * row + (hq + hkv + h / (hq / hkv)) * d + e];
                            const float off = got[((size_t)t * hq + h) * d + e] - want;
                            worst = off < 0 ? (worst > -off ? worst : -off) : (worst > off ? worst : off);
                        }
                CHECK(worst <= 127.0f * 0x1p-21f, "a row that sees one key has its value");
                CHECK(tkv_hip_free(ctx, dc) == TKV_HIP_OK && tkv_hip_free(ctx, dy) == TKV_HIP_OK, "free");
            }
            const std::vector<int32_t> cu = {0, 1000, 1000, keys};
            int32_t* dc = put(ctx, cu);
            float* dy = put(ctx, std::vector<float>((size_t)keys * hq * d, -1.0f));
            const tkv_hip_rows y = {dy, hq * d, d};
            CHECK(tkv_hip_dev_attention_prompt(ctx, TKV_HIP_F32, keys, keys, hq, hkv, d, 3, &q, &k, &v, &y,
                                               TKV_HIP_F32, dc, nullptr, 0.01f, 1, 1) == TKV_HIP_OK,
                  "attention_prompt");
            std::vector<double> freq(d / 2, 0.5);
            float* tab = put(ctx, std::vector<float>((size_t)keys * d, 0.0f));
            CHECK(tkv_hip_dev_rope_table(ctx, keys, d, freq.data(), 1.0, tab) == TKV_HIP_OK, "rope_table");
            CHECK(tkv_hip_dev_rope_append(ctx, TKV_HIP_F32, keys, hq, hkv, d, &q, &k, nullptr, dp, tab, keys, d,
                                          TKV_HIP_ROPE_PAIRS, &q, &k, TKV_HIP_F32, 0, nullptr) == TKV_HIP_OK,
                  "rotation in place");
            CHECK(tkv_hip_ctx_synchronize(ctx) == TKV_HIP_OK, "synchronize");
            CHECK(tkv_hip_kv_free(cache) == TKV_HIP_OK, "kv_free");
            for (void* p : {(void*)dx, (void*)ds, (void*)dt, (void*)dl, (void*)dp, (void*)dc, (void*)dy, (void*)tab})
                CHECK(tkv_hip_free(ctx, p) == TKV_HIP_OK, "free");
        }
    CHECK(tkv_hip_ctx_destroy(ctx) == TKV_HIP_OK, "ctx_destroy");
}

int main() {
    refusals();
    const int devices = tkv_hip_device_count();
    if (devices < 1) no_device();
    else on_device();
    if (g_fail) return 1;
    printf("attention_sanitize: all checks passed (%s)\n", devices < 1 ? "no device" : "device 0");
    return 0;
}
