// rope.hip -- the paged cache's handle, rotation tables, and the kernel that
// takes the new tokens' queries, keys and values from the projection to the
// attention: rotate, convert, append.
#include <math.h>

#include <new>

#include "attn.h"

namespace tkv {

// table[p][i] = amplitude * (cos, sin)(p * inv_freq[i]).  The product of a
// position below 2^29 and a frequency of 24 significant bits is exact in f64,
// and sincos reduces it there: the table is right to f32 rounding at any
// position, where an f32 angle would be off by 2^-24 of itself (0.006 rad at
// position 100000).
struct Freqs {
    double f[128];
};

__global__ __launch_bounds__(256) void k_rope_table(Freqs fr, int half, int64_t n, double amplitude,
                                                    float2* __restrict__ table) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
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
    int64_t rows;        // tokens * heads
    int32_t hq, hkv, d, rot, pairs;
    int32_t lanes_log2;  // lanes of a head row, 8 elements each
};

template <typename T>
struct alignas(16) Vec8 {
    T e[8];
};

// 8 elements of a row from e0 on: one or two 16-byte loads (VEC), else those
// below d one by one.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int e0, int d, float (&x)[8]) {
    if constexpr (VEC) {
        const Vec8<T> v = *reinterpret_cast<const Vec8<T>*>(row + e0);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(v.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = e0 + i < d ? to_f32(row[e0 + i]) : 0.0f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int e0, int d, const float (&x)[8]) {
    if constexpr (VEC) {
        Vec8<T> v;
#pragma unroll
        for (int i = 0; i < 8; i++) v.e[i] = from_f32<T>(x[i]);
        *reinterpret_cast<Vec8<T>*>(row + e0) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (e0 + i < d) row[e0 + i] = from_f32<T>(x[i]);
    }
}

// One head row (of q, k or v) per 2^lanes_log2 lanes, 8 elements per lane, one
// row per thread group and no loop: HBM bound, each input element read from it
// once.  A lane also loads the 8 elements that its own are rotated with (they
// are another lane's, so the second load hits the cache; a shuffle of 8 f32
// through LDS costs more) and the 8 or 4 table entries, which the token's other
// heads read too.
//
// VEC: 16-byte aligned rows, d and rot / 2 multiples of 8.
template <typename TI, typename TO, typename C, bool VEC>
__global__ __launch_bounds__(256) void k_rope_append(RopeArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r64 = t >> a.lanes_log2;
    if (r64 >= a.rows) return;  // whole groups: the rows' lanes stay together
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
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const bool live = e0 < a.d;
    if (live && !pad) {
        load8<TI, VEC>(src, e0, a.d, x);
        if (a.table && !isv && e0 < a.rot) {
            const int half = a.rot >> 1;
            const float2* cs = a.table + (int64_t)pos * half;
            // each product and sum is rounded by itself (no contraction in
            // this library): the same bits as separate elementwise operations
            if (VEC && a.pairs) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 w = cs[(e0 >> 1) + i];
                    const float u = x[2 * i], y = x[2 * i + 1];
                    x[2 * i] = u * w.x - y * w.y;
                    x[2 * i + 1] = y * w.x + u * w.y;
                }
            } else if (VEC) {
                const bool low = e0 < half;
                float o[8];
                load8<TI, VEC>(src, low ? e0 + half : e0 - half, a.d, o);
                const float2* w = cs + (low ? e0 : e0 - half);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float c = w[i].x, s = w[i].y;
                    x[i] = low ? x[i] * c - o[i] * s : x[i] * c + o[i] * s;
                }
            } else {
                for (int i = 0; i < 8; i++) {
                    const int e = e0 + i;
                    if (e >= a.rot) break;
                    const bool low = a.pairs ? !(e & 1) : e < half;
                    const int mate = a.pairs ? e ^ 1 : low ? e + half : e - half;
                    const float2 w = cs[a.pairs ? e >> 1 : low ? e : e - half];
                    const float o = to_f32(src[mate]);
                    x[i] = low ? x[i] * w.x - o * w.y : x[i] * w.x + o * w.y;
                }
            }
        }
    }
    if (live && isq && a.qo)
        store8<TO, VEC>(static_cast<TO*>(a.qo) + (int64_t)tok * a.qo_st + (int64_t)h * a.qo_sh, e0, a.d, x);
    if (live && !isq && !isv && a.ko)
        store8<TO, VEC>(static_cast<TO*>(a.ko) + (int64_t)tok * a.ko_st + (int64_t)h * a.ko_sh, e0, a.d, x);
    const bool put = slot >= 0 && slot < a.n_slots;
    const uint32_t s32 = put ? (uint32_t)slot : 0, pg = div_by(a.page, s32);
    const int64_t at = ((int64_t)pg * a.hkv + h) * a.page.d + (s32 - pg * a.page.d);
    if constexpr (sizeof(C) == 1) {
        // max |x| of the row over its lanes (NaN skipped), then its codes
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));
        for (int o = 1 << a.lanes_log2 >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        if (!put) return;
        const float scale = fmaxf(m, 1e-8f) / 127.0f, inv = 1.0f / scale;
        if (e0 == 0) (isv ? a.vs : a.ks)[at] = scale;
        if (!live) return;
        int8_t* dst = static_cast<int8_t*>(isv ? a.vc : a.kc) + at * a.d + e0;
        int8_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = __builtin_rintf(x[i] * inv);
            q[i] = y != y ? (int8_t)0 : (int8_t)(int)fminf(fmaxf(y, -127.0f), 127.0f);
        }
        if constexpr (VEC) {
            uint2 w;
            __builtin_memcpy(&w, q, 8);
            *reinterpret_cast<uint2*>(dst) = w;
        } else {
            for (int i = 0; i < 8; i++)
                if (e0 + i < a.d) dst[i] = q[i];
        }
    } else if (put && live) {
        store8<C, VEC>(static_cast<C*>(isv ? a.vc : a.kc) + at * a.d, e0, a.d, x);
    }
}

template <typename TI, typename TO>
static void launch_rope(Ctx* c, const RopeArgs& a, bool i8, bool vec) {
    const dim3 grid((unsigned)ceil_div(a.rows << a.lanes_log2, 256));
    if (i8) {
        if (vec) k_rope_append<TI, TO, int8_t, true><<<grid, 256, 0, c->stream>>>(a);
        else k_rope_append<TI, TO, int8_t, false><<<grid, 256, 0, c->stream>>>(a);
    } else {
        if (vec) k_rope_append<TI, TO, TO, true><<<grid, 256, 0, c->stream>>>(a);
        else k_rope_append<TI, TO, TO, false><<<grid, 256, 0, c->stream>>>(a);
    }
}

template <typename TI>
static void launch_rope_to(Ctx* c, const RopeArgs& a, int type_out, bool i8, bool vec) {
    if (type_out == TKV_HIP_F32) launch_rope<TI, float>(c, a, i8, vec);
    else if (type_out == TKV_HIP_F16) launch_rope<TI, _Float16>(c, a, i8, vec);
    else launch_rope<TI, __bf16>(c, a, i8, vec);
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
    if (ceil_div(n, 256) >= (1ll << 31))
        return set_error(TKV_HIP_UNSUPPORTED, "rope_table: too many entries");
    k_rope_table<<<(unsigned)ceil_div(n, 256), 256, 0, c->stream>>>(fr, half, n, amplitude,
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
    if (tokens < 0 || heads_q < 0 || heads_kv < 0 || heads_q > 65535 || heads_kv > 65535 ||
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
    a.rows = tokens * heads;
    a.hq = (int32_t)heads_q;
    a.hkv = (int32_t)heads_kv;
    a.d = (int32_t)head_dim;
    a.rot = table ? (int32_t)rot_dim : 0;
    a.pairs = layout == TKV_HIP_ROPE_PAIRS;
    while (8 << a.lanes_log2 < head_dim) a.lanes_log2++;
    const int64_t bi = type_bytes(type_in), bo = type_bytes(type_out);
    const bool vec = head_dim % 8 == 0 && (a.rot / 2) % 8 == 0 && rows_aligned(has_q ? q : nullptr, bi) &&
                     rows_aligned(has_k ? k : nullptr, bi) && rows_aligned(has_v ? v : nullptr, bi) &&
                     rows_aligned(q_out, bo) && rows_aligned(k_out, bo) &&
                     (!kv || (aligned(kv->k, 16) && aligned(kv->v, 16)));
    const bool i8 = kv && kv->type == TKV_HIP_I8;
    if (type_in == TKV_HIP_F32) launch_rope_to<float>(c, a, type_out, i8, vec);
    else if (type_in == TKV_HIP_F16) launch_rope_to<_Float16>(c, a, type_out, i8, vec);
    else launch_rope_to<__bf16>(c, a, type_out, i8, vec);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

}  // extern "C"
