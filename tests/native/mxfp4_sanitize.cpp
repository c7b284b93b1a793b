// mxfp4_sanitize.cpp -- drives the 4-bit entry points and the norms with rotation of
// libtkv_hip's C ABI with the library's host code built with AddressSanitizer and
// UndefinedBehaviorSanitizer, as host_sanitize.cpp and attention_sanitize.cpp do for
// the rest.  Without a GPU: argument checks and the no-device paths, at sizes whose
// products would overflow.  With one: small calls of every kernel choice, of values
// that 4 bits hold, so that the outputs are whole numbers known beforehand.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "../../include/tkv_hip.h"

static int g_fail = 0;
#define CHECK(cond, what)                                                  \
    do {                                                                   \
        if (!(cond)) {                                                     \
            char buf[256];                                                 \
            tkv_hip_last_error(buf, sizeof(buf));                          \
            fprintf(stderr, "mxfp4_sanitize: FAIL %s (last error: %s)\n", what, buf); \
            g_fail = 1;                                                    \
        }                                                                  \
    } while (0)

static const int64_t kHuge = INT64_MAX;

// Refused before any device is touched; no pointer here is read.
static void refusals() {
    int64_t h = 0;
    void* p = reinterpret_cast<void*>(64);
    uint8_t* b = static_cast<uint8_t*>(p);
    for (int64_t rows : {int64_t(-1), int64_t(1) << 31, kHuge})
        CHECK(tkv_hip_dev_quantize_mxfp4(0, TKV_HIP_F32, p, 32, rows, 32, b, b) == TKV_HIP_BAD_ARG, "rows out of range");
    for (int64_t cols : {int64_t(0), int64_t(-5), int64_t(1) << 31, kHuge})
        CHECK(tkv_hip_dev_dequantize_mxfp4(0, b, b, 1, cols, TKV_HIP_F32, p, kHuge) == TKV_HIP_BAD_ARG,
              "cols out of range");
    CHECK(tkv_hip_dev_quantize_mxfp4(0, TKV_HIP_F32, p, INT64_MIN, 2, 32, b, b) == TKV_HIP_BAD_ARG, "negative stride");
    CHECK(tkv_hip_dev_quantize_mxfp4(0, TKV_HIP_F32, nullptr, 0, 0, 32, nullptr, nullptr) == TKV_HIP_OK, "no rows");
    CHECK(tkv_hip_dev_matmul_mxfp4(0, b, b, b, b, kHuge, 1, 32, nullptr, TKV_HIP_F32, p, kHuge) == TKV_HIP_UNSUPPORTED,
          "product of 2^63 rows");
    CHECK(tkv_hip_dev_matmul_mxfp4(0, b, b, b, b, 1, kHuge, 32, nullptr, TKV_HIP_F32, p, kHuge) == TKV_HIP_UNSUPPORTED,
          "product of 2^63 columns");
    CHECK(tkv_hip_dev_matmul_mxfp4(0, b, b, b, b, 1, 1, kHuge, nullptr, TKV_HIP_F32, p, 1) == TKV_HIP_UNSUPPORTED,
          "product of 2^63 terms");
    CHECK(tkv_hip_dev_matmul_mxfp4(0, b, b, b, b, 1, 1, -1, nullptr, TKV_HIP_F32, p, 1) == TKV_HIP_BAD_ARG,
          "product of -1 terms");
    CHECK(tkv_hip_dev_matmul_mxfp4(0, b, b, b, b, 1, 1, 32, reinterpret_cast<float*>(66), TKV_HIP_F32, p, 1) ==
              TKV_HIP_BAD_ARG,
          "unaligned bias");
    CHECK(tkv_hip_weight_create_mxfp4(0, nullptr, b, 1, 32, nullptr, &h) == TKV_HIP_BAD_ARG, "weight without codes");
    CHECK(tkv_hip_weight_create_mxfp4(0, b, b, 1, 32, nullptr, nullptr) == TKV_HIP_BAD_ARG, "weight without an output");
    CHECK(tkv_hip_linear_forward_typed(0, 0, TKV_HIP_F32, p, 1, 1, TKV_HIP_F32, p, 1) == TKV_HIP_BAD_ARG,
          "linear without a weight");

    const tkv_hip_rows r = {p, 64, 64};
    uint8_t axes[32] = {};
    const auto rotate = [&](const tkv_hip_head_norm* norm, const tkv_hip_rope* rope, int64_t tokens) {
        return tkv_hip_dev_norm_rope_append(0, TKV_HIP_F32, tokens, 1, 0, 64, &r, nullptr, nullptr, norm, rope, &r, nullptr,
                                            TKV_HIP_F32, 0, nullptr);
    };
    const float* f = static_cast<float*>(p);
    const int32_t* pos = static_cast<int32_t*>(p);
    for (float eps : {0.0f, -1.0f, 1.0f / 0.0f * 0.0f}) {
        const tkv_hip_head_norm norm = {eps, f, f};
        CHECK(rotate(&norm, nullptr, 1) == TKV_HIP_BAD_ARG, "eps");
    }
    const tkv_hip_head_norm norm = {1e-6f, nullptr, nullptr};
    for (int64_t tokens : {int64_t(-1), int64_t(1) << 31, kHuge})
        CHECK(rotate(&norm, nullptr, tokens) == TKV_HIP_BAD_ARG, "tokens out of range");
    for (int64_t rot : {int64_t(0), int64_t(63), int64_t(66), kHuge}) {
        const tkv_hip_rope rope = {f, 4, rot, 0, 2, pos, 1, axes};
        CHECK(rotate(&norm, &rope, 1) == TKV_HIP_BAD_ARG, "rot_dim");
    }
    for (int32_t n : {0, -1, 5, INT32_MAX}) {
        const tkv_hip_rope rope = {f, 4, 64, 0, n, pos, 1, axes};
        CHECK(rotate(&norm, &rope, 1) == TKV_HIP_BAD_ARG, "number of axes");
    }
    axes[31] = 2;
    const tkv_hip_rope two = {f, 4, 64, 0, 2, pos, 1, axes};
    CHECK(rotate(&norm, &two, 1) == TKV_HIP_BAD_ARG, "a pair's axis beyond the axes");
    const tkv_hip_rope none = {nullptr, 4, 64, 0, 1, pos, 1, nullptr};
    CHECK(rotate(&norm, &none, 1) == TKV_HIP_BAD_ARG, "rotation without a table");
}

static void no_device() {
    int64_t h = 0;
    void* p = reinterpret_cast<void*>(64);
    uint8_t* b = static_cast<uint8_t*>(p);
    const tkv_hip_rows r = {p, 64, 64};
    const tkv_hip_head_norm norm = {1e-6f, nullptr, nullptr};
    uint8_t axes[32] = {1};
    const tkv_hip_rope rope = {static_cast<float*>(p), 4, 64, 1, 2, static_cast<int32_t*>(p), 1, axes};
    CHECK(tkv_hip_dev_quantize_mxfp4(0, TKV_HIP_F32, p, 32, 1, 32, b, b) == TKV_HIP_NO_DEVICE, "quantize");
    CHECK(tkv_hip_dev_dequantize_mxfp4(0, b, b, 1, 32, TKV_HIP_BF16, p, 32) == TKV_HIP_NO_DEVICE, "dequantize");
    CHECK(tkv_hip_dev_matmul_mxfp4(0, b, b, b, b, 1, 1, 32, nullptr, TKV_HIP_F32, p, 1) == TKV_HIP_NO_DEVICE, "matmul");
    CHECK(tkv_hip_weight_create_mxfp4(0, b, b, 1, 32, nullptr, &h) == TKV_HIP_NO_DEVICE, "weight");
    CHECK(tkv_hip_dev_norm_rope_append(0, TKV_HIP_F32, 1, 1, 0, 64, &r, nullptr, nullptr, &norm, &rope, &r, nullptr,
                                       TKV_HIP_F32, 0, nullptr) == TKV_HIP_NO_DEVICE,
          "norm and rotation");
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
    // values of +-1, 2, 3, 4 in every block with a 4: held exactly
    for (int m : {1, 5, 20, 50, 100, 700})
        for (int k : {32, 300, 4200}) {
            const int n = 130, blocks = (k + 31) / 32;
            std::vector<float> x((size_t)m * k), w((size_t)n * k), bias(n);
            for (size_t i = 0; i < x.size(); i++) x[i] = (float)((int)(i * 7 % 9) - 4);
            for (size_t i = 0; i < w.size(); i++) w[i] = (float)((int)(i * 5 % 9) - 4);
            for (int i = 0; i < n; i++) bias[i] = (float)(i % 17);
            float *dx = put(ctx, x), *dw = put(ctx, w), *db = put(ctx, bias);
            float* dy = put(ctx, std::vector<float>((size_t)m * n, -1.0f));
            uint8_t* codes = put(ctx, std::vector<uint8_t>((size_t)m * blocks * 16));
            uint8_t* scales = put(ctx, std::vector<uint8_t>((size_t)m * blocks));
            float* dv = put(ctx, std::vector<float>((size_t)m * k, -1.0f));
            CHECK(tkv_hip_dev_quantize_mxfp4(ctx, TKV_HIP_F32, dx, k, m, k, codes, scales) == TKV_HIP_OK, "quantize");
            CHECK(tkv_hip_dev_dequantize_mxfp4(ctx, codes, scales, m, k, TKV_HIP_F32, dv, k) == TKV_HIP_OK,
                  "dequantize");
            std::vector<float> back((size_t)m * k), got((size_t)m * n);
            CHECK(tkv_hip_memcpy_d2h(ctx, back.data(), dv, (int64_t)(back.size() * 4)) == TKV_HIP_OK, "download");
            CHECK(memcmp(back.data(), x.data(), back.size() * 4) == 0, "values held exactly");
            int64_t weight = 0;
            CHECK(tkv_hip_weight_create(ctx, dw, n, k, db, TKV_HIP_WEIGHT_MXFP4, &weight) == TKV_HIP_OK, "weight_create");
            void* wc = nullptr;
            float* ws = nullptr;
            int64_t wn = 0, wk = 0;
            int32_t format = 0;
            CHECK(tkv_hip_weight_info(weight, &wc, &ws, nullptr, &wn, &wk, &format) == TKV_HIP_OK && wn == n &&
                      wk == blocks * 32 && format == TKV_HIP_WEIGHT_MXFP4,
                  "weight_info");
            for (int form = 0; form < 3; form++) {
                CHECK(tkv_hip_memset(ctx, dy, 0xff, (int64_t)m * n * 4) == TKV_HIP_OK, "memset");
                const int rc = form == 0 ? tkv_hip_linear_forward(ctx, weight, dx, m, TKV_HIP_ACT_PER_TOKEN, dy)
                               : form == 1
                                   ? tkv_hip_linear_forward_typed(ctx, weight, TKV_HIP_F32, dx, k, m, TKV_HIP_F32, dy, n)
                                   : tkv_hip_dev_matmul_mxfp4(ctx, codes, scales, static_cast<uint8_t*>(wc),
                                                              reinterpret_cast<uint8_t*>(ws), m, n, k, db, TKV_HIP_F32,
                                                              dy, n);
                CHECK(rc == TKV_HIP_OK, "product");
                CHECK(tkv_hip_memcpy_d2h(ctx, got.data(), dy, (int64_t)(got.size() * 4)) == TKV_HIP_OK, "download");
                int wrong = 0;
                for (int i = 0; i < m; i += 1 + i / 3)
                    for (int j = 0; j < n; j++) {
                        double sum = bias[j];
                        for (int e = 0; e < k; e++) sum += (double)x[(size_t)i * k + e] * w[(size_t)j * k + e];
                        wrong += got[(size_t)i * n + j] != (float)sum;
                    }
                CHECK(wrong == 0, "whole numbers multiplied exactly");
            }
            CHECK(tkv_hip_weight_free(weight) == TKV_HIP_OK, "weight_free");
            for (void* p : {(void*)dx, (void*)dw, (void*)db, (void*)dy, (void*)codes, (void*)scales, (void*)dv})
                CHECK(tkv_hip_free(ctx, p) == TKV_HIP_OK, "free");
        }
    // heads of +-c: their norm is c, so that with eps beside nothing they become +-1,
    // and without a turn (an angle of 0) stay so
    for (int d : {64, 20})
        for (int tokens : {1, 300, 9000}) {
            const int hq = 3, hkv = 2, row = (hq + 2 * hkv) * d, pages = (tokens + 15) / 16;
            std::vector<float> x((size_t)tokens * row), gain(d, 2.0f), table((size_t)4 * d);
            for (size_t i = 0; i < x.size(); i++) x[i] = i % 3 ? 1024.0f : -1024.0f;
            for (size_t i = 0; i < table.size(); i += 2) table[i] = 1.0f;
            std::vector<int32_t> pos((size_t)2 * tokens, 3);
            std::vector<int64_t> slots(tokens);
            for (int t = 0; t < tokens; t++) slots[t] = t;
            float *dx = put(ctx, x), *dg = put(ctx, gain), *dt = put(ctx, table);
            float* dq = put(ctx, std::vector<float>((size_t)tokens * hq * d, -7.0f));
            int32_t* dp = put(ctx, pos);
            int64_t *ds = put(ctx, slots), cache = 0;
            CHECK(tkv_hip_kv_create(ctx, TKV_HIP_F32, pages, 16, hkv, d, nullptr, nullptr, nullptr, nullptr, &cache) ==
                      TKV_HIP_OK,
                  "kv_create");
            std::vector<uint8_t> axes(d / 2);
            for (int i = 0; i < d / 2; i++) axes[i] = (uint8_t)(i % 2);
            const tkv_hip_rows q = {dx, row, d}, k = {dx + hq * d, row, d}, v = {dx + (hq + hkv) * d, row, d};
            const tkv_hip_rows out = {dq, hq * d, d};
            const tkv_hip_head_norm norm = {1e-6f, dg, nullptr};
            const tkv_hip_rope rope = {dt, 4, d, TKV_HIP_ROPE_PAIRS, 2, dp, tokens, axes.data()};
            CHECK(tkv_hip_dev_norm_rope_append(ctx, TKV_HIP_F32, tokens, hq, hkv, d, &q, &k, &v, &norm, &rope, &out, nullptr,
                                               TKV_HIP_F32, cache, ds) == TKV_HIP_OK,
                  "norm_rope_append");
            std::vector<float> got((size_t)tokens * hq * d), kept((size_t)pages * hkv * 16 * d);
            void *kp = nullptr, *vp = nullptr;
            CHECK(tkv_hip_kv_info(cache, &kp, &vp, nullptr, nullptr) == TKV_HIP_OK, "kv_info");
            CHECK(tkv_hip_memcpy_d2h(ctx, got.data(), dq, (int64_t)(got.size() * 4)) == TKV_HIP_OK, "download");
            CHECK(tkv_hip_memcpy_d2h(ctx, kept.data(), kp, (int64_t)(kept.size() * 4)) == TKV_HIP_OK, "download");
            float worst = 0.0f;
            const auto off = [&](float a, float b) {
                const float e = a < b ? b - a : a - b;
                worst = e > worst ? e : worst;
            };
            for (int t = 0; t < tokens; t++)
                for (int e = 0; e < d; e++) {
                    for (int h = 0; h < hq; h++)
                        off(got[((size_t)t * hq + h) * d + e], x[(size_t)t * row + h * d + e] / 512.0f);
                    for (int h = 0; h < hkv; h++)
                        off(kept[(((size_t)(t / 16) * hkv + h) * 16 + t % 16) * d + e],
                            x[(size_t)t * row + (hq + h) * d + e] / 1024.0f);
                }
            CHECK(worst <= 0x1p-18f, "heads of one magnitude become ones");
            CHECK(tkv_hip_kv_free(cache) == TKV_HIP_OK, "kv_free");
            for (void* p : {(void*)dx, (void*)dg, (void*)dt, (void*)dq, (void*)dp, (void*)ds})
                CHECK(tkv_hip_free(ctx, p) == TKV_HIP_OK, "free");
        }
    CHECK(tkv_hip_ctx_destroy(ctx) == TKV_HIP_OK, "ctx_destroy");
}

int main() {
    refusals();
    const int devices = tkv_hip_device_count();
    if (devices < 1) no_device();
    else on_device();
    if (!g_fail) printf("mxfp4_sanitize: all checks passed (%s)\n", devices < 1 ? "no device" : "device 0");
    // Out without the exit handlers: the GPU runtime's free memory there, which can make
    // the sanitizer give device memory out of its quarantine back to that runtime, gone
    // by then, and it fails for that ("dev_runtime_unloaded").
    fflush(stdout);
    fflush(stderr);
    std::_Exit(g_fail ? 1 : 0);
}
