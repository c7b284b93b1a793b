// rope.hip -- the paged cache's handle, rotation tables, and the kernel that
// takes the new tokens' queries, keys and values from the projection to the
// attention: rotate, convert, append.
#include <math.h>

#include <new>
#include <string>

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
    // the kernels with NORM or AXES (below) alone
    int32_t normed;
    float eps, inv_d;
    const float *qg, *kg;     // gains, or null
    int32_t axes;
    int64_t axis_stride;      // of the positions
    uint32_t pair_axis[8];    // two bits a pair
};
constexpr int kMaxAxes = 4;

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
// 1 / sqrt(mean of the squares + eps), from their sum over a row's lanes.  Lanes are
// exchanged within rows of 16 without LDS: neighbours, pairs, then halves of 8 and
// of 16 mirrored, whose lanes hold the same sums by then.  (A row of 32 lanes, which
// only the kernel for any size has, takes one exchange more.)
template <int CTRL>
__device__ __forceinline__ float swapped(float x) {
    return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_sum(float s, int lanes) {
    if (lanes > 0) s += swapped<0xb1>(s);   // quad_perm 1 0 3 2
    if (lanes > 1) s += swapped<0x4e>(s);   // quad_perm 2 3 0 1
    if (lanes > 2) s += swapped<0x141>(s);  // row_half_mirror
    if (lanes > 3) s += swapped<0x140>(s);  // row_mirror
    if (lanes > 4) s += __shfl_xor(s, 16);
    return s;
}
// v_rsq_f32, an ulp off at most, which takes no subnormals: those are scaled.
__device__ __forceinline__ float inv_norm(float sum, float inv_d, float eps) {
    float v = sum * inv_d + eps;
    const bool tiny = v < 0x1p-100f;
    v = tiny ? v * 0x1p64f : v;
    const float r = __builtin_amdgcn_rsqf(v);
    return tiny ? r * 0x1p32f : r;
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

// A chunk as it is in memory.
template <typename T>
struct alignas(16) Raw8 {
    unsigned v[2 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ void from_raw(const Raw8<T>& r, float (&x)[8]) {
    unsigned v[2 * sizeof(T)];
#pragma unroll
    for (int k = 0; k < (int)(2 * sizeof(T)); k++) {
        v[k] = r.v[k];
        asm volatile("" : "+v"(v[k]));
    }
    Vec8<T> e;
    __builtin_memcpy(&e, v, sizeof(e));
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = to_f32(e.e[k]);
}
__device__ __forceinline__ void norm_turn(float& p, float& q, float2 w, float r, bool turn) {
    // (the products are chosen, not their factor: 0 times an infinity beside an element
    // that is not rotated would make that a NaN)
    const float c = turn ? w.x * r : r, s = w.y * r, a = p, b = q;
    const float bs = turn ? b * s : 0.0f, as = turn ? a * s : 0.0f;
    p = __builtin_fmaf(a, c, -bs);
    q = __builtin_fmaf(b, c, as);
}

// The same with norms per head, positions on several axes, or both: a lane's two
// chunks of `HEADS` heads in flight as they are in memory, and converted one head at
// a time.  A pair's entry is in the table's row of its own axis' position.
//   Normed rows: the squares' sum goes over the row's lanes; with r the inverse norm
// and g the gains, y_a = (a g_a)(r c) - (b g_b)(r s), the second product added by an
// fma.  Others are rotated as above, each product and sum rounded by itself.
//   HBM bound, and by what it computes beside: 8192 tokens of 32 + 8 heads of 128 in
// bf16 take 46.4 us (46.2 without norms, by the kernel above), 4.4 TB/s; with three
// axes, whose entries are 8 bytes from rows of their own, 46.9.
template <typename TI, typename TO, typename C, int HEADS>
__global__ __launch_bounds__(256) void k_norm_rope_rows(RopeArgs a) {
    const int64_t t64 = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> a.lanes_log2;
    if (t64 >= a.tokens) return;  // whole groups: the rows' lanes stay together
    const int tok = (int)t64, i = (int)threadIdx.x & ((1 << a.lanes_log2) - 1);
    const int chunks = a.d >> 3;
    const int turns = a.pairs ? 0 : a.rot >> 4;  // chunk pairs rotated with each other
    const int rest = chunks - 2 * turns, j = i - turns;
    const int c0 = i < turns ? i : j < (rest + 1) / 2 ? 2 * turns + j : chunks;
    const int c1 = i < turns ? i + turns : c0 < chunks ? c0 + (rest + 1) / 2 : chunks;
    const bool in0 = c0 < chunks, in1 = c1 < chunks;
    const int first = blockIdx.y * HEADS;

    // positions; the rows themselves do not wait for them
    int at_axis[kMaxAxes] = {0, 0, 0, 0};
    bool pad = false;
    if (a.table) {
#pragma unroll
        for (int x = 0; x < kMaxAxes; x++)
            if (x < a.axes) at_axis[x] = a.positions[x * a.axis_stride + tok];
    }
    int64_t slot = a.kc ? a.slots[tok] : -1;
    Raw8<TI> raw[HEADS][2];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int row = min(first + u, (int)a.heads.d - 1);
        const bool isq = row < a.hq, isv = row >= a.hq + a.hkv;
        const int h = row - (isq ? 0 : isv ? a.hq + a.hkv : a.hq);
        const TI* src = static_cast<const TI*>(isq ? a.q : isv ? a.v : a.k) +
                        (int64_t)h * (isq ? a.q_sh : isv ? a.v_sh : a.k_sh) +
                        (int64_t)tok * (isq ? a.q_st : isv ? a.v_st : a.k_st);
        raw[u][0] = raw[u][1] = Raw8<TI>{};
        if (in0) raw[u][0] = *reinterpret_cast<const Raw8<TI>*>(src + 8 * c0);
        if (in1) raw[u][1] = *reinterpret_cast<const Raw8<TI>*>(src + 8 * c1);
    }
    float g0[8], g1[8];
    const float* have = first < a.hq ? a.qg : a.kg;
    const auto load_gains = [&]() {
#pragma unroll
        for (int k = 0; k < 8; k++) g0[k] = g1[k] = 1.0f;
        if (have && in0) load8(have + 8 * c0, g0);
        if (have && in1) load8(have + 8 * c1, g1);
    };
    load_gains();
    if (a.table) {
#pragma unroll
        for (int x = 0; x < kMaxAxes; x++)
            if (x < a.axes) pad = pad || at_axis[x] < 0 || at_axis[x] >= a.table_len;
    }
    if (pad) slot = -1;
    const bool put = slot >= 0 && slot < a.n_slots;
    const uint32_t s32 = put ? (uint32_t)slot : 0, pg = div_by(a.page, s32);
    // (cos, sin): of the 8 pairs of a chunk pair, or the 4 of either chunk
    const bool turn0 = a.pairs ? c0 < a.rot >> 3 : i < turns, turn1 = a.pairs ? c1 < a.rot >> 3 : i < turns;
    float2 w[8];
    const auto entries = [&](int at, float2* to) {
        const int half = a.rot >> 1;
        if (a.axes > 1) {
            const uint32_t which = a.pair_axis[at >> 4] >> (2 * (at & 15));
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int x = (which >> (2 * k)) & 3;
                const int p = x == 0 ? at_axis[0] : x == 1 ? at_axis[1] : x == 2 ? at_axis[2] : at_axis[3];
                to[k] = a.table[(int64_t)p * half + at + k];
            }
        } else {
            const float4* cs = reinterpret_cast<const float4*>(a.table + (int64_t)at_axis[0] * half + at);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float4 v = cs[k];
                to[2 * k] = make_float2(v.x, v.y);
                to[2 * k + 1] = make_float2(v.z, v.w);
            }
        }
    };
    if (turn0 && !pad) entries(a.pairs ? 4 * c0 : 8 * i, w);
    if (turn1 && !pad) entries(a.pairs ? 4 * c1 : 8 * i + 4, w + 4);

#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        const int row = first + u;
        if (row >= (int)a.heads.d) break;
        const bool isq = row < a.hq, isv = row >= a.hq + a.hkv;
        const int h = row - (isq ? 0 : isv ? a.hq + a.hkv : a.hq);
        // (a head's conversions stay behind the heads before it: done at once they
        // hold twice the registers)
        float x0[8], x1[8];
        from_raw(raw[u][0], x0);
        from_raw(raw[u][1], x1);
        if (pad) {
#pragma unroll
            for (int k = 0; k < 8; k++) x0[k] = x1[k] = 0.0f;
        }
        if (!isv && a.normed) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) sum = __builtin_fmaf(x1[k], x1[k], __builtin_fmaf(x0[k], x0[k], sum));
            const float r = inv_norm(row_sum(sum, a.lanes_log2), a.inv_d, a.eps);
            const float* gain = isq ? a.qg : a.kg;
            if (u > 0 && gain != have) {
                have = gain;
                load_gains();
            }
            if (gain) {
#pragma unroll
                for (int k = 0; k < 8; k++) x0[k] *= g0[k], x1[k] *= g1[k];
            }
            if (a.pairs) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    norm_turn(x0[2 * k], x0[2 * k + 1], w[k], r, turn0);
                    norm_turn(x1[2 * k], x1[2 * k + 1], w[4 + k], r, turn1);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) norm_turn(x0[k], x1[k], w[k], r, turn0);
            }
            if (pad) {  // zeros whatever the gains
#pragma unroll
                for (int k = 0; k < 8; k++) x0[k] = x1[k] = 0.0f;
            }
        } else if (!isv && !pad) {
            if (a.pairs) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (!(k < 4 ? turn0 : turn1)) continue;
                    float* x = k < 4 ? x0 : x1;
                    const int e = 2 * (k & 3);
                    const float p = x[e], q = x[e + 1];
                    x[e] = p * w[k].x - q * w[k].y;
                    x[e + 1] = q * w[k].x + p * w[k].y;
                }
            } else if (turn0) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float p = x0[k], q = x1[k];
                    x0[k] = p * w[k].x - q * w[k].y;
                    x1[k] = q * w[k].x + p * w[k].y;
                }
            }
        }
        if (!isv && (isq ? a.qo : a.ko)) {
            TO* dst = static_cast<TO*>(isq ? a.qo : a.ko) + (int64_t)tok * (isq ? a.qo_st : a.ko_st) +
                      (int64_t)h * (isq ? a.qo_sh : a.ko_sh);
            if (in0) store8(dst + 8 * c0, x0);
            if (in1) store8(dst + 8 * c1, x1);
        }
        if (isq || !a.kc) continue;
        const int64_t at = ((int64_t)pg * a.hkv + h) * a.page.d + (s32 - pg * a.page.d);
        if constexpr (sizeof(C) == 1) {
            unsigned most = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) most = max(most, max(abs_bits(x0[k]), abs_bits(x1[k])));
            const float m = row_max(most, a.lanes_log2);
            if (!put) continue;
            const float scale = scale_of(m), inv = 1.0f / scale;
            if (i == 0) (isv ? a.vs : a.ks)[at] = scale;
            int8_t* dst = static_cast<int8_t*>(isv ? a.vc : a.kc) + at * a.d;
            int8_t z[8];
#pragma unroll
            for (int half = 0; half < 2; half++) {
#pragma unroll
                for (int k = 0; k < 8; k++) z[k] = code_of(half ? x1[k] : x0[k], inv);
                uint2 v;
                __builtin_memcpy(&v, z, 8);
                if (half ? in1 : in0) *reinterpret_cast<uint2*>(dst + 8 * (half ? c1 : c0)) = v;
            }
        } else if (put) {
            C* dst = static_cast<C*>(isv ? a.vc : a.kc) + at * a.d;
            if (in0) store8(dst + 8 * c0, x0);
            if (in1) store8(dst + 8 * c1, x1);
        }
    }
}

// Any head size, rotation and alignment: one head row per 2^lanes lanes, 8
// elements a lane, one by one; the element that one is rotated with is loaded
// again, so that it is bound by its load instructions.
template <typename TI, typename TO, typename C, bool MORE>
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
    bool pad = a.table && (pos < 0 || pos >= a.table_len);
    if (MORE && a.table)
        for (int x = 1; x < a.axes; x++) {
            const int p = a.positions[x * a.axis_stride + tok];
            pad = pad || p < 0 || p >= a.table_len;
        }
    int64_t slot = -1;
    if (!isq && a.kc && !pad) slot = a.slots[tok];
    const int half = a.rot >> 1;
    const float2* cs = a.table + (int64_t)pos * half;
    const bool normed = MORE && a.normed && !isv;
    const float* gain = isq ? a.qg : a.kg;
    float inv = 1.0f;
    if (MORE && a.normed) {  // every lane of the wave takes part in the sum
        float sum = 0.0f;
        for (int i = 0; i < 8; i++) {
            const float e = e0 + i < a.d && !pad ? to_f32(src[e0 + i]) : 0.0f;
            sum += e * e;
        }
        inv = inv_norm(row_sum(sum, a.lanes_log2), a.inv_d, a.eps);
    }
    const auto element = [&](int e) {
        const float v = to_f32(src[e]);
        return normed ? v * inv * (gain ? gain[e] : 1.0f) : v;
    };
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = e0 + i;
        x[i] = e < a.d && !pad ? element(e) : 0.0f;
        if (e < a.rot && !isv && !pad) {
            const bool low = a.pairs ? !(e & 1) : e < half;
            const int mate = a.pairs ? e ^ 1 : low ? e + half : e - half;
            const int pair = a.pairs ? e >> 1 : low ? e : e - half;
            const float2* from = cs;
            if (MORE && a.axes > 1) {
                const int axis = (a.pair_axis[pair >> 4] >> (2 * (pair & 15))) & 3;
                from = a.table + (int64_t)a.positions[axis * a.axis_stride + tok] * half;
            }
            const float2 w = from[pair];
            const float o = element(mate);
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

template <typename TI, typename TO, typename C, bool MORE>
static void launch_rope(Ctx* c, RopeArgs a, bool vec) {
    const int64_t heads = a.heads.d;
    int rows_log2 = 0;
    while (16 << rows_log2 < a.d) rows_log2++;
    // (a dimension of the grid holds 2^28 tokens of heads of 256)
    if (!vec || (a.tokens << rows_log2) + 255 > kGridItems) {
        while (8 << a.lanes_log2 < a.d) a.lanes_log2++;
        k_rope_any<TI, TO, C, MORE>
            <<<wide_grid(ceil_div(a.tokens * heads << a.lanes_log2, 256)), 256, 0, c->stream>>>(a);
        return;
    }
    a.lanes_log2 = rows_log2;
    const int64_t blocks = ceil_div(a.tokens << a.lanes_log2, 256);
    // four heads per lane where that still leaves eight workgroups per CU, with norms
    // two (5001 tokens of 12 + 12 heads of 64 12.1 us, of one head 14.5; 2000 of 32 + 8
    // of 128 11.9 and 14.2; with one per CU 700 of those 7.3 and 6.4)
    const bool four = blocks * ceil_div(heads, 4) >= (MORE ? 2 : 8) * c->num_cus;
    const dim3 grid((unsigned)blocks, (unsigned)(four ? ceil_div(heads, 4) : heads));
    if constexpr (MORE) {
        if (four) k_norm_rope_rows<TI, TO, C, 4><<<grid, 256, 0, c->stream>>>(a);
        else k_norm_rope_rows<TI, TO, C, 1><<<grid, 256, 0, c->stream>>>(a);
    } else {
        if (four) k_rope_rows<TI, TO, C, 4><<<grid, 256, 0, c->stream>>>(a);
        else k_rope_rows<TI, TO, C, 1><<<grid, 256, 0, c->stream>>>(a);
    }
}

template <typename TI, typename TO>
static void launch_rope_to(Ctx* c, const RopeArgs& a, bool i8, bool vec) {
    if (a.normed || a.axes > 1) {
        if (i8) launch_rope<TI, TO, int8_t, true>(c, a, vec);
        else launch_rope<TI, TO, TO, true>(c, a, vec);
    } else {
        if (i8) launch_rope<TI, TO, int8_t, false>(c, a, vec);
        else launch_rope<TI, TO, TO, false>(c, a, vec);
    }
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

// Both entry points: checks, arguments, launch.  norm and rope may be null.
static int rope_append(const char* who, int64_t ctx, int32_t type_in, int64_t tokens, int64_t heads_q,
                       int64_t heads_kv, int64_t head_dim, const tkv_hip_rows* q, const tkv_hip_rows* k,
                       const tkv_hip_rows* v, const tkv_hip_head_norm* norm, const tkv_hip_rope* rope,
                       const tkv_hip_rows* q_out, const tkv_hip_rows* k_out, int32_t type_out, int64_t cache,
                       const int64_t* slots) {
    const auto bad = [&](const char* what) { return set_error(TKV_HIP_BAD_ARG, std::string(who) + ": " + what); };
    const KvCache* kv = reinterpret_cast<const KvCache*>(cache);
    if (!float_type(type_in) || !float_type(type_out)) return bad("types are F32, F16 or BF16");
    if (tokens < 0 || tokens >= (1ll << 31) || heads_q < 0 || heads_kv < 0 || heads_q > 65535 || heads_kv > 65535 ||
        head_dim <= 0 || head_dim > 256)
        return bad("sizes out of range (head_dim 1 .. 256)");
    if (rope && (rope->rot_dim < 2 || rope->rot_dim > head_dim || rope->rot_dim % 2 || rope->table_len < 0 ||
                 !rope->positions || !aligned(rope->table, 8) ||
                 (rope->layout != TKV_HIP_ROPE_HALF && rope->layout != TKV_HIP_ROPE_PAIRS)))
        return bad("a table takes positions, an even rot_dim in 2 .. head_dim and a known layout");
    if (rope && (rope->axes < 1 || rope->axes > kMaxAxes || (rope->axes > 1 && !rope->pair_axis)))
        return bad("1 to 4 axes, several with the axis of each pair");
    if (rope && rope->axes > 1)
        for (int64_t i = 0; i < rope->rot_dim / 2; i++)
            if (rope->pair_axis[i] >= rope->axes) return bad("a pair's axis is not among the axes");
    if (norm && !(norm->eps > 0.0f && norm->eps <= 3.402823466e38f)) return bad("eps: positive and finite");
    if (norm && (!aligned(norm->q_gain, 4) || !aligned(norm->k_gain, 4))) return bad("unaligned gains");
    const bool has_q = q && heads_q > 0, has_k = k && heads_kv > 0, has_v = v && heads_kv > 0;
    if ((heads_q > 0 && !has_q) || (heads_kv > 0 && !has_k) || (has_q && !q->data) ||
        (has_k && !k->data) || (has_v && !v->data))
        return bad("NULL rows with a positive head count");
    if ((q_out && (!has_q || !q_out->data)) || (k_out && (!has_k || !k_out->data)))
        return bad("an output without its rows");
    if (kv) {
        if (!has_k || !has_v || !slots) return bad("a cache takes k, v and slots");
        if (kv->heads != heads_kv || kv->d != head_dim) return bad("the cache has other heads");
        if (kv->type != type_out && kv->type != TKV_HIP_I8)
            return bad("the cache's type is neither type_out nor I8");
    }
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    if (kv && kv->device != c->device) return bad("the cache is on another device");
    RopeArgs a = {};
    // without a cache the values have nowhere to go: no rows for them
    const int64_t heads = heads_q + heads_kv + (kv ? heads_kv : 0);
    if (tokens == 0 || heads == 0) return TKV_HIP_OK;
    if (tokens * heads >= (1ll << 31))
        return set_error(TKV_HIP_UNSUPPORTED, std::string(who) + ": tokens * heads >= 2^31");
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
    a.tokens = tokens;
    a.hq = (int32_t)heads_q;
    a.hkv = (int32_t)heads_kv;
    a.d = (int32_t)head_dim;
    a.axes = 1;
    if (rope) {
        a.positions = rope->positions;
        a.table = reinterpret_cast<const float2*>(rope->table);
        a.table_len = rope->table_len;
        a.rot = (int32_t)rope->rot_dim;
        a.pairs = rope->layout == TKV_HIP_ROPE_PAIRS;
        a.axes = rope->axes;
        a.axis_stride = rope->stride_axis;
        for (int i = 0; a.axes > 1 && i < a.rot / 2; i++)
            a.pair_axis[i >> 4] |= (uint32_t)rope->pair_axis[i] << (2 * (i & 15));
    }
    if (norm) {
        a.normed = 1;
        a.eps = norm->eps;
        a.inv_d = 1.0f / (float)head_dim;
        a.qg = norm->q_gain;
        a.kg = norm->k_gain;
    }
    const int64_t bi = type_bytes(type_in), bo = type_bytes(type_out);
    const bool vec = head_dim % 8 == 0 && a.rot % (a.pairs ? 8 : 16) == 0 && aligned(a.table, 16) &&
                     aligned(a.qg, 16) && aligned(a.kg, 16) && heads < 65536 &&
                     rows_aligned(has_q ? q : nullptr, bi) && rows_aligned(has_k ? k : nullptr, bi) &&
                     rows_aligned(has_v ? v : nullptr, bi) && rows_aligned(q_out, bo) && rows_aligned(k_out, bo) &&
                     (!kv || (aligned(kv->k, 16) && aligned(kv->v, 16)));
    const bool i8 = kv && kv->type == TKV_HIP_I8;
    if (type_in == TKV_HIP_F32) launch_rope_from<float>(c, a, type_out, i8, vec);
    else if (type_in == TKV_HIP_F16) launch_rope_from<_Float16>(c, a, type_out, i8, vec);
    else launch_rope_from<__bf16>(c, a, type_out, i8, vec);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
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
    const tkv_hip_rope r = {table, table_len, rot_dim, layout, 1, positions, 0, nullptr};
    return rope_append("rope_append", ctx, type_in, tokens, heads_q, heads_kv, head_dim, q, k, v, nullptr,
                       table ? &r : nullptr, q_out, k_out, type_out, cache, slots);
}

int32_t tkv_hip_dev_norm_rope_append(int64_t ctx, int32_t type_in, int64_t tokens, int64_t heads_q,
                                     int64_t heads_kv, int64_t head_dim, const tkv_hip_rows* q,
                                     const tkv_hip_rows* k, const tkv_hip_rows* v,
                                     const tkv_hip_head_norm* norm, const tkv_hip_rope* rope,
                                     const tkv_hip_rows* q_out, const tkv_hip_rows* k_out,
                                     int32_t type_out, int64_t cache, const int64_t* slots) {
    if (rope && !rope->table) return set_error(TKV_HIP_BAD_ARG, "norm_rope_append: a rotation without its table");
    return rope_append("norm_rope_append", ctx, type_in, tokens, heads_q, heads_kv, head_dim, q, k, v, norm, rope,
                       q_out, k_out, type_out, cache, slots);
}

}  // extern "C"
