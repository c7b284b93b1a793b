// rope.hip -- the paged cache's handle, rotation tables, and the kernel that
// takes the new tokens' queries, keys and values from the projection to the
// attention: rotate, convert, append.
#include <math.h>

#include <new>

#include "attn.h"

namespace tkv {

// table[p][i] = amplitude * (cos, sin)(p * inv_freq[i]).  The product is rounded
// once in f64, 2^-53 of itself (10^-7 rad at position 2^29), and sincos reduces it
// there: the entries are right to f32 rounding, where an f32 angle would be off by
// 2^-24 of itself (0.006 rad at position 100000).
struct Freqs {
    double f[128];
};

__global__ __launch_bounds__(256) void k_rope_table(Freqs fr, int half, int64_t n, double amplitude,
                                                    float2* __restrict__ table) {
    const int64_t t = wide_block() * 256 + threadIdx.x;
    if (t >= n) return;
    const int64_t p = t / half;
    double s, c;
    sincos((double)p * fr.f[t - p * half], &s, &c);
    table[t] = make_float2((float)(amplitude * c), (float)(amplitude * s));
}

struct RopeArgs {
    const void *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    void *qo, *ko;
    int64_t qo_st, qo_sh, ko_st, ko_sh;
    void *kc, *vc;       // the cache's pools, or null
    float *ks, *vs;      // I8
    const int64_t* slots;
    int64_t n_slots;
    FastDiv page, heads;  // heads: q, k and v rows of a token
    const int32_t* positions;
    const float2* table;
    int64_t table_len;
    int64_t tokens;
    int32_t hq, hkv, d, rot, pairs;
    int32_t lanes_log2;  // lanes of a head row
};

template <typename T>
struct alignas(16) Vec8 {
    T e[8];
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const Vec8<T> v = *reinterpret_cast<const Vec8<T>*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_f32(v.e[i]);
}
// 16-bit chunks are stored past the L2's reuse: the lanes of a row write whole
// lines (8192 tokens of 48 heads of 128: 50.6 -> 45.1 us).  f32 chunks are half
// lines per store and lose by it.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < 8; i++) v.e[i] = from_f32<T>(x[i]);
    if constexpr (sizeof(T) == 2) {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        u32x4 w;
        __builtin_memcpy(&w, &v, 16);
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
    } else {
        *reinterpret_cast<Vec8<T>*>(p) = v;
    }
}
// codes of a row from its max |x| (over 1 << lanes lanes), as bits: a NaN's are
// above every number's, so a row that has one gets a NaN for its scale, and values
// of NaN, where f32's maximum would leave it out and code it as 0
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float row_max(unsigned m, int lanes) {
    for (int o = 1 << lanes >> 1; o; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o));
    return __uint_as_float(m);
}
// By the rounded reciprocal, as elementwise tensor libraries divide by a constant:
// within an ulp of max / 127, and the same codes as their operations give.
__device__ __forceinline__ float scale_of(float m) { return (m < 1e-8f ? 1e-8f : m) * (1.0f / 127.0f); }
__device__ __forceinline__ int8_t code_of(float x, float inv) {
    const float y = __builtin_rintf(x * inv);
    return y != y ? (int8_t)0 : (int8_t)(int)fminf(fmaxf(y, -127.0f), 127.0f);
}

// Chunks of 8 elements: a lane takes two of a head row's, in the half layout those
// that are rotated with each other, so that neighbouring lanes have neighbouring
// chunks; 2^lanes lanes per head row, and `HEADS` heads of its token in turn, all
// their loads in flight together, so that each element is read once and a table
// entry once per HEADS heads.  Head index and with it the role (q, k or v) are the
// workgroup's.  HBM bound: 8192 tokens of 32 + 8 heads of 128, bf16, 45.7 us, 4.5
// TB/s, where a large copy reaches 5.1; 32 tokens of 12 + 12 heads of 64 take 3.4 us,
// one launch.
template <typename TI, typename TO, typename C, int HEADS>
__global__ __launch_bounds__(256) void k_rope_rows(RopeArgs a) {
    const int64_t t64 = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> a.lanes_log2;
    if (t64 >= a.tokens) return;  // whole groups: the rows' lanes stay together
    const int tok = (int)t64, i = (int)threadIdx.x & ((1 << a.lanes_log2) - 1);
    const int chunks = a.d >> 3;
    const int turns = a.pairs ? 0 : a.rot >> 4;  // chunk pairs rotated with each other
    const int rest = chunks - 2 * turns, j = i - turns;
    const int c0 = i < turns ? i : j < (rest + 1) / 2 ? 2 * turns + j : chunks;
    const int c1 = i < turns ? i + turns : c0 < chunks ? c0 + (rest + 1) / 2 : chunks;
    const bool in0 = c0 < chunks, in1 = c1 < chunks;
    const int pos = a.table ? a.positions[tok] : 0;
    const bool pad = a.table && (pos < 0 || pos >= a.table_len);
    int64_t slot = -1;
    if (a.kc && !pad) slot = a.slots[tok];
    const bool put = slot >= 0 && slot < a.n_slots;
    const uint32_t s32 = put ? (uint32_t)slot : 0, pg = div_by(a.page, s32);
    // (cos, sin): of the 8 pairs of a chunk pair, or the 4 of either chunk
    const bool turn0 = a.pairs ? c0 < a.rot >> 3 : i < turns, turn1 = a.pairs ? c1 < a.rot >> 3 : i < turns;
    float2 w[8];
    const auto entries = [&](int at, float2* to) {
        const float4* cs = reinterpret_cast<const float4*>(a.table + (int64_t)pos * (a.rot >> 1) + at);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float4 v = cs[k];
            to[2 * k] = make_float2(v.x, v.y);
            to[2 * k + 1] = make_float2(v.z, v.w);
        }
    };
    if (turn0 && !pad) entries(a.pairs ? 4 * c0 : 8 * i, w);
    if (turn1 && !pad) entries(a.pairs ? 4 * c1 : 8 * i + 4, w + 4);
    const int first = blockIdx.y * HEADS;
    float x0[HEADS][8], x1[HEADS][8];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int row = min(first + u, (int)a.heads.d - 1);
        const bool isq = row < a.hq, isv = row >= a.hq + a.hkv;
        const int h = row - (isq ? 0 : isv ? a.hq + a.hkv : a.hq);
        const TI* src = static_cast<const TI*>(isq ? a.q : isv ? a.v : a.k) +
                        (int64_t)h * (isq ? a.q_sh : isv ? a.v_sh : a.k_sh) +
                        (int64_t)tok * (isq ? a.q_st : isv ? a.v_st : a.k_st);
#pragma unroll
        for (int k = 0; k < 8; k++) x0[u][k] = x1[u][k] = 0.0f;
        if (in0 && !pad) load8(src + 8 * c0, x0[u]);
        if (in1 && !pad) load8(src + 8 * c1, x1[u]);
    }
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int row = first + u;
        if (row >= (int)a.heads.d) break;
        const bool isq = row < a.hq, isv = row >= a.hq + a.hkv;
        const int h = row - (isq ? 0 : isv ? a.hq + a.hkv : a.hq);
        if (!isv && !pad) {
            // each product and sum is rounded by itself (no contraction in this
            // library): the same bits as separate elementwise operations
            if (a.pairs) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (!(k < 4 ? turn0 : turn1)) continue;
                    float* x = k < 4 ? x0[u] : x1[u];
                    const int e = 2 * (k & 3);
                    const float p = x[e], q = x[e + 1];
                    x[e] = p * w[k].x - q * w[k].y;
                    x[e + 1] = q * w[k].x + p * w[k].y;
                }
            } else if (turn0) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float p = x0[u][k], q = x1[u][k];
                    x0[u][k] = p * w[k].x - q * w[k].y;
                    x1[u][k] = q * w[k].x + p * w[k].y;
                }
            }
        }
        if (!isv && (isq ? a.qo : a.ko)) {
            TO* dst = static_cast<TO*>(isq ? a.qo : a.ko) + (int64_t)tok * (isq ? a.qo_st : a.ko_st) +
                      (int64_t)h * (isq ? a.qo_sh : a.ko_sh);
            if (in0) store8(dst + 8 * c0, x0[u]);
            if (in1) store8(dst + 8 * c1, x1[u]);
        }
        if (isq || !a.kc) continue;
        const int64_t at = ((int64_t)pg * a.hkv + h) * a.page.d + (s32 - pg * a.page.d);
        if constexpr (sizeof(C) == 1) {
            unsigned most = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) most = max(most, max(abs_bits(x0[u][k]), abs_bits(x1[u][k])));
            const float m = row_max(most, a.lanes_log2);
            if (!put) continue;
            const float scale = scale_of(m), inv = 1.0f / scale;
            if (i == 0) (isv ? a.vs : a.ks)[at] = scale;
            int8_t* dst = static_cast<int8_t*>(isv ? a.vc : a.kc) + at * a.d;
            int8_t z[8];
#pragma unroll
            for (int half = 0; half < 2; half++) {
#pragma unroll
                for (int k = 0; k < 8; k++) z[k] = code_of(half ? x1[u][k] : x0[u][k], inv);
                uint2 v;
                __builtin_memcpy(&v, z, 8);
                if (half ? in1 : in0) *reinterpret_cast<uint2*>(dst + 8 * (half ? c1 : c0)) = v;
            }
        } else if (put) {
            C* dst = static_cast<C*>(isv ? a.vc : a.kc) + at * a.d;
            if (in0) store8(dst + 8 * c0, x0[u]);
            if (in1) store8(dst + 8 * c1, x1[u]);
        }
    }
}

// Any head size, rotation and alignment: one head row per 2^lanes lanes, 8
// elements a lane, one by one; the element that one is rotated with is loaded
// again, so that it is bound by its load instructions.
template <typename TI, typename TO, typename C>
__global__ __launch_bounds__(256) void k_rope_any(RopeArgs a) {
    const int64_t t = wide_block() * 256 + threadIdx.x;
    const int64_t r64 = t >> a.lanes_log2;
    if (r64 >= a.tokens * a.heads.d) return;  // whole groups: the rows' lanes stay together
    const uint32_t r = (uint32_t)r64;
    const int e0 = 8 * ((int)threadIdx.x & ((1 << a.lanes_log2) - 1));
    const uint32_t tok = div_by(a.heads, r);
    int h = (int)(r - tok * a.heads.d);
    const bool isq = h < a.hq, isv = h >= a.hq + a.hkv;
    h -= isq ? 0 : isv ? a.hq + a.hkv : a.hq;
    const TI* src = static_cast<const TI*>(isq ? a.q : isv ? a.v : a.k) +
                    (int64_t)tok * (isq ? a.q_st : isv ? a.v_st : a.k_st) +
                    (int64_t)h * (isq ? a.q_sh : isv ? a.v_sh : a.k_sh);
    const int pos = a.table ? a.positions[tok] : 0;
    const bool pad = a.table && (pos < 0 || pos >= a.table_len);
    int64_t slot = -1;
    if (!isq && a.kc && !pad) slot = a.slots[tok];
    const int half = a.rot >> 1;
    const float2* cs = a.table + (int64_t)pos * half;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = e0 + i;
        x[i] = e < a.d && !pad ? to_f32(src[e]) : 0.0f;
        if (e < a.rot && !isv && !pad) {
            const bool low = a.pairs ? !(e & 1) : e < half;
            const int mate = a.pairs ? e ^ 1 : low ? e + half : e - half;
            const float2 w = cs[a.pairs ? e >> 1 : low ? e : e - half];
            const float o = to_f32(src[mate]);
            x[i] = low ? x[i] * w.x - o * w.y : x[i] * w.x + o * w.y;
        }
    }
    if (!isv && (isq ? a.qo : a.ko)) {
        // a row may be rotated in place: its lanes are one wave's, and all have
        // loaded before the first stores
        __builtin_amdgcn_wave_barrier();
        TO* dst = static_cast<TO*>(isq ? a.qo : a.ko) + (int64_t)tok * (isq ? a.qo_st : a.ko_st) +
                  (int64_t)h * (isq ? a.qo_sh : a.ko_sh);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (e0 + i < a.d) dst[e0 + i] = from_f32<TO>(x[i]);
    }
    const bool put = slot >= 0 && slot < a.n_slots;
    const uint32_t s32 = put ? (uint32_t)slot : 0, pg = div_by(a.page, s32);
    const int64_t at = ((int64_t)pg * a.hkv + h) * a.page.d + (s32 - pg * a.page.d);
    if constexpr (sizeof(C) == 1) {
        unsigned most = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) most = max(most, abs_bits(x[i]));
        const float m = row_max(most, a.lanes_log2);
        if (!put) return;
        const float scale = scale_of(m), inv = 1.0f / scale;
        if (e0 == 0) (isv ? a.vs : a.ks)[at] = scale;
        int8_t* dst = static_cast<int8_t*>(isv ? a.vc : a.kc) + at * a.d;
        for (int i = 0; i < 8; i++)
            if (e0 + i < a.d) dst[e0 + i] = code_of(x[i], inv);
    } else if (put) {
        C* dst = static_cast<C*>(isv ? a.vc : a.kc) + at * a.d;
        for (int i = 0; i < 8; i++)
            if (e0 + i < a.d) dst[e0 + i] = from_f32<C>(x[i]);
    }
}

template <typename TI, typename TO, typename C>
static void launch_rope(Ctx* c, RopeArgs a, bool vec) {
    const int64_t heads = a.heads.d;
    int rows_log2 = 0;
    while (16 << rows_log2 < a.d) rows_log2++;
    // (a dimension of the grid holds 2^28 tokens of heads of 256)
    if (!vec || (a.tokens << rows_log2) + 255 > kGridItems) {
        while (8 << a.lanes_log2 < a.d) a.lanes_log2++;
        k_rope_any<TI, TO, C><<<wide_grid(ceil_div(a.tokens * heads << a.lanes_log2, 256)), 256, 0, c->stream>>>(a);
        return;
    }
    a.lanes_log2 = rows_log2;
    const int64_t blocks = ceil_div(a.tokens << a.lanes_log2, 256);
    // four heads per lane where that still leaves eight workgroups per CU
    if (blocks * ceil_div(heads, 4) >= 8 * c->num_cus)
        k_rope_rows<TI, TO, C, 4><<<dim3((unsigned)blocks, (unsigned)ceil_div(heads, 4)), 256, 0, c->stream>>>(a);
    else
        k_rope_rows<TI, TO, C, 1><<<dim3((unsigned)blocks, (unsigned)heads), 256, 0, c->stream>>>(a);
}

template <typename TI, typename TO>
static void launch_rope_to(Ctx* c, const RopeArgs& a, bool i8, bool vec) {
    if (i8) launch_rope<TI, TO, int8_t>(c, a, vec);
    else launch_rope<TI, TO, TO>(c, a, vec);
}

template <typename TI>
static void launch_rope_from(Ctx* c, const RopeArgs& a, int type_out, bool i8, bool vec) {
    if (type_out == TKV_HIP_F32) launch_rope_to<TI, float>(c, a, i8, vec);
    else if (type_out == TKV_HIP_F16) launch_rope_to<TI, _Float16>(c, a, i8, vec);
    else launch_rope_to<TI, __bf16>(c, a, i8, vec);
}

static bool rows_aligned(const tkv_hip_rows* r, int64_t bytes) {
    return !r || (aligned(r->data, 16) && r->stride_token * bytes % 16 == 0 &&
                  r->stride_head * bytes % 16 == 0);
}

static void kv_release(KvCache* kv) {
    if (!kv) return;
    if (kv->owned) {
        // Teardown: errors here leave nothing the caller can act on.
        (void)hipSetDevice(kv->device);
        (void)hipDeviceSynchronize();
        if (kv->k) (void)hipFree(kv->k);
        if (kv->v) (void)hipFree(kv->v);
        if (kv->ks) (void)hipFree(kv->ks);
        if (kv->vs) (void)hipFree(kv->vs);
    }
    delete kv;
}

}  // namespace tkv

using namespace tkv;

extern "C" {

int32_t tkv_hip_kv_create(int64_t ctx, int32_t type, int64_t num_pages, int64_t page_size,
                          int64_t heads, int64_t head_dim, void* k, void* v, float* k_scales,
                          float* v_scales, int64_t* handle_out) {
    const bool i8 = type == TKV_HIP_I8;
    if (!handle_out || num_pages <= 0 || page_size <= 0 || heads <= 0 || head_dim <= 0 ||
        head_dim > 256 || heads > 65535)
        return set_error(TKV_HIP_BAD_ARG, "kv_create: sizes out of range or NULL output");
    if (!i8 && !float_type(type)) return set_error(TKV_HIP_BAD_ARG, "kv_create: unknown type");
    if (page_size >= (1ll << 31) || num_pages >= (1ll << 31) ||
        num_pages * page_size >= (1ll << 31) || num_pages * page_size * heads >= (1ll << 32))
        return set_error(TKV_HIP_BAD_ARG,
                         "kv_create: num_pages * page_size >= 2^31, or 2^32 with the heads");
    if (!!k != !!v || (k && i8) != !!k_scales || (k && i8) != !!v_scales)
        return set_error(TKV_HIP_BAD_ARG,
                         "kv_create: give both pools or none, and scales with int8 pools only");
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    if (!k && c->capturing)
        return set_error(TKV_HIP_BAD_ARG, "kv_create: allocates, not inside a stream capture");
    KvCache* kv = new (std::nothrow) KvCache();
    if (!kv) return set_error(TKV_HIP_OOM, "kv_create: host allocation failed");
    kv->device = c->device;
    kv->type = type;
    kv->pages = num_pages;
    kv->page = (int)page_size;
    kv->heads = (int)heads;
    kv->d = (int)head_dim;
    kv->k = k;
    kv->v = v;
    kv->ks = k_scales;
    kv->vs = v_scales;
    if (!k) {
        kv->owned = true;
        const int64_t rows = num_pages * heads * page_size;
        const int64_t bytes = rows * head_dim * type_bytes(type);
        void** at[4] = {&kv->k, &kv->v, reinterpret_cast<void**>(&kv->ks),
                        reinterpret_cast<void**>(&kv->vs)};
        for (int i = 0; i < (i8 ? 4 : 2); i++) {
            const int64_t b = i < 2 ? bytes : rows * 4;
            const hipError_t e = hipMalloc(at[i], (size_t)b);
            int rc = e == hipSuccess ? TKV_HIP_OK : fail_hip(e, "hipMalloc(cache)", __FILE__, __LINE__);
            if (rc == TKV_HIP_OOM) (void)hipGetLastError();
            if (rc == TKV_HIP_OK) rc = launch_fill(c, *at[i], 0, b);
            if (rc != TKV_HIP_OK) {
                kv_release(kv);
                return rc;
            }
        }
        // the handle is any context's of this device, and its pointers the caller's:
        // what they write must not meet the fill on this context's stream
        const hipError_t e = hipStreamSynchronize(c->stream);
        if (e != hipSuccess) {
            const int rc = fail_hip(e, "hipStreamSynchronize(cache)", __FILE__, __LINE__);
            kv_release(kv);
            return rc;
        }
    }
    *handle_out = reinterpret_cast<int64_t>(kv);
    return TKV_HIP_OK;
}

int32_t tkv_hip_kv_free(int64_t handle) {
    kv_release(reinterpret_cast<KvCache*>(handle));
    return TKV_HIP_OK;
}

int32_t tkv_hip_kv_info(int64_t handle, void** k, void** v, float** k_scales, float** v_scales) {
    const KvCache* kv = reinterpret_cast<const KvCache*>(handle);
    if (!kv) return set_error(TKV_HIP_BAD_ARG, "NULL cache handle");
    if (k) *k = kv->k;
    if (v) *v = kv->v;
    if (k_scales) *k_scales = kv->ks;
    if (v_scales) *v_scales = kv->vs;
    return TKV_HIP_OK;
}

int32_t tkv_hip_dev_rope_table(int64_t ctx, int64_t positions, int64_t rot_dim,
                               const double* inv_freq, double amplitude, float* table) {
    if (positions < 0 || positions >= (1ll << 31) || rot_dim < 2 || rot_dim > 256 || rot_dim % 2 ||
        !inv_freq || (positions > 0 && !table) || !aligned(table, 8))
        return set_error(TKV_HIP_BAD_ARG, "rope_table: bad arguments (rot_dim even, 2 .. 256; table 8-byte aligned)");
    if (positions == 0) return TKV_HIP_OK;
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    const int half = (int)(rot_dim / 2);
    const int64_t n = positions * half;
    Freqs fr;
    for (int i = 0; i < 128; i++) fr.f[i] = i < half ? inv_freq[i] : 0.0;
    k_rope_table<<<wide_grid(ceil_div(n, 256)), 256, 0, c->stream>>>(fr, half, n, amplitude,
                                                                     reinterpret_cast<float2*>(table));
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

int32_t tkv_hip_dev_rope_append(int64_t ctx, int32_t type_in, int64_t tokens, int64_t heads_q,
                                int64_t heads_kv, int64_t head_dim, const tkv_hip_rows* q,
                                const tkv_hip_rows* k, const tkv_hip_rows* v,
                                const int32_t* positions, const float* table, int64_t table_len,
                                int64_t rot_dim, int32_t layout, const tkv_hip_rows* q_out,
                                const tkv_hip_rows* k_out, int32_t type_out, int64_t cache,
                                const int64_t* slots) {
    const KvCache* kv = reinterpret_cast<const KvCache*>(cache);
    if (!float_type(type_in) || !float_type(type_out))
        return set_error(TKV_HIP_BAD_ARG, "rope_append: types are F32, F16 or BF16");
    if (tokens < 0 || tokens >= (1ll << 31) || heads_q < 0 || heads_kv < 0 || heads_q > 65535 || heads_kv > 65535 ||
        head_dim <= 0 || head_dim > 256)
        return set_error(TKV_HIP_BAD_ARG, "rope_append: sizes out of range (head_dim 1 .. 256)");
    if (table && (rot_dim < 2 || rot_dim > head_dim || rot_dim % 2 || table_len < 0 || !positions ||
                  !aligned(table, 8) || (layout != TKV_HIP_ROPE_HALF && layout != TKV_HIP_ROPE_PAIRS)))
        return set_error(TKV_HIP_BAD_ARG,
                         "rope_append: a table takes positions, an even rot_dim in 2 .. head_dim and a known layout");
    const bool has_q = q && heads_q > 0, has_k = k && heads_kv > 0, has_v = v && heads_kv > 0;
    if ((heads_q > 0 && !has_q) || (heads_kv > 0 && !has_k) || (has_q && !q->data) ||
        (has_k && !k->data) || (has_v && !v->data))
        return set_error(TKV_HIP_BAD_ARG, "rope_append: NULL rows with a positive head count");
    if ((q_out && (!has_q || !q_out->data)) || (k_out && (!has_k || !k_out->data)))
        return set_error(TKV_HIP_BAD_ARG, "rope_append: an output without its rows");
    if (kv) {
        if (!has_k || !has_v || !slots)
            return set_error(TKV_HIP_BAD_ARG, "rope_append: a cache takes k, v and slots");
        if (kv->heads != heads_kv || kv->d != head_dim)
            return set_error(TKV_HIP_BAD_ARG, "rope_append: the cache has other heads");
        if (kv->type != type_out && kv->type != TKV_HIP_I8)
            return set_error(TKV_HIP_BAD_ARG, "rope_append: the cache's type is neither type_out nor I8");
    }
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    if (kv && kv->device != c->device)
        return set_error(TKV_HIP_BAD_ARG, "rope_append: the cache is on another device");
    RopeArgs a = {};
    // without a cache the values have nowhere to go: no rows for them
    const int64_t heads = heads_q + heads_kv + (kv ? heads_kv : 0);
    if (tokens == 0 || heads == 0) return TKV_HIP_OK;
    if (tokens * heads >= (1ll << 31))
        return set_error(TKV_HIP_UNSUPPORTED, "rope_append: tokens * heads >= 2^31");
    if (has_q) a.q = q->data, a.q_st = q->stride_token, a.q_sh = q->stride_head;
    if (has_k) a.k = k->data, a.k_st = k->stride_token, a.k_sh = k->stride_head;
    if (has_v) a.v = v->data, a.v_st = v->stride_token, a.v_sh = v->stride_head;
    if (q_out) a.qo = q_out->data, a.qo_st = q_out->stride_token, a.qo_sh = q_out->stride_head;
    if (k_out) a.ko = k_out->data, a.ko_st = k_out->stride_token, a.ko_sh = k_out->stride_head;
    if (kv) {
        a.kc = kv->k;
        a.vc = kv->v;
        a.ks = kv->ks;
        a.vs = kv->vs;
        a.slots = slots;
        a.n_slots = kv->pages * kv->page;
        a.page = fast_div((uint32_t)kv->page);
    } else {
        a.page = fast_div(1);
    }
    a.heads = fast_div((uint32_t)heads);
    a.positions = positions;
    a.table = reinterpret_cast<const float2*>(table);
    a.table_len = table_len;
    a.tokens = tokens;
    a.hq = (int32_t)heads_q;
    a.hkv = (int32_t)heads_kv;
    a.d = (int32_t)head_dim;
    a.rot = table ? (int32_t)rot_dim : 0;
    a.pairs = layout == TKV_HIP_ROPE_PAIRS;
    const int64_t bi = type_bytes(type_in), bo = type_bytes(type_out);
    const bool vec = head_dim % 8 == 0 && a.rot % (a.pairs ? 8 : 16) == 0 && aligned(table, 16) &&
                     heads < 65536 && rows_aligned(has_q ? q : nullptr, bi) &&
                     rows_aligned(has_k ? k : nullptr, bi) && rows_aligned(has_v ? v : nullptr, bi) &&
                     rows_aligned(q_out, bo) && rows_aligned(k_out, bo) &&
                     (!kv || (aligned(kv->k, 16) && aligned(kv->v, 16)));
    const bool i8 = kv && kv->type == TKV_HIP_I8;
    if (type_in == TKV_HIP_F32) launch_rope_from<float>(c, a, type_out, i8, vec);
    else if (type_in == TKV_HIP_F16) launch_rope_from<_Float16>(c, a, type_out, i8, vec);
    else launch_rope_from<__bf16>(c, a, type_out, i8, vec);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

}  // extern "C"
