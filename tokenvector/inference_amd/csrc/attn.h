// attn.h -- what the attention operators share: element types, the cache's
// handle, arguments of the kernels and the sequences' bounds.
#pragma once

#include <hip/hip_runtime.h>

#include "tkv_internal.h"

namespace tkv {

// A paged cache (tkv_hip_kv_create): K and V [pages, heads, page, d], scales
// [pages, heads, page].  A page of one head is contiguous, so that the
// attention of a head reads runs of page * d elements.
struct KvCache {
    int device = 0;
    int type = TKV_HIP_F32;
    int64_t pages = 0;
    int page = 0, heads = 0, d = 0;
    void *k = nullptr, *v = nullptr;
    float *ks = nullptr, *vs = nullptr;  // I8
    bool owned = false;
};

inline int64_t type_bytes(int type) {
    return type == TKV_HIP_F32 ? 4 : type == TKV_HIP_I8 ? 1 : 2;
}
inline bool float_type(int type) {
    return type == TKV_HIP_F32 || type == TKV_HIP_F16 || type == TKV_HIP_BF16;
}

// HIP takes fewer than 2^32 work items in a dimension of a grid: 2^24 workgroups of
// 256.  Kernels that may need more number them over two.
constexpr int64_t kGridItems = (1ll << 32) - 1;
constexpr int64_t kWideX = 1 << 22;
constexpr int64_t kWideBlocks = kWideX * 65535;
inline dim3 wide_grid(int64_t blocks) {
    const int64_t x = blocks < kWideX ? blocks : kWideX;
    return dim3((unsigned)x, (unsigned)ceil_div(blocks, x));
}
__device__ __forceinline__ int64_t wide_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// n / d for n < 2^31 by a multiplication, (mulhi(m, n) + n) >> l: the method of
// Granlund and Montgomery, "Division by invariant integers using multiplication" (1994).
struct FastDiv {
    uint32_t d, m, l;
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t l = 0;
    while ((1ull << l) < d) l++;
    return {d, (uint32_t)((((1ull << l) - d) << 32) / d + 1), l};
}
__device__ __forceinline__ uint32_t div_by(FastDiv f, uint32_t n) {
    return (__umulhi(f.m, n) + n) >> f.l;
}

// Element conversions, one rounding (to nearest even) on the way down.
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(int8_t x) { return (float)x; }
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
    return (T)x;
}

// Attention of one call, as its kernels take it.  Strides in elements.
struct AttnArgs {
    const void* q;
    int64_t q_st, q_sh;
    void* out;
    int64_t o_st, o_sh;
    // packed keys and values, or a cache's pools
    const void *k, *v;
    int64_t k_st, k_sh, v_st, v_sh;
    const float *ks, *vs;
    const int32_t* pages;  // page table, null where keys are packed
    int64_t pages_st;
    int64_t pool_pages;
    FastDiv page;
    const int32_t *cu_q, *cu_k, *kv_lens;
    int64_t tokens, tokens_k;
    int32_t seqs, hq, hkv, g, d;
    int32_t causal;
    int64_t window;    // 0: none
    float scale_log2;  // scale * log2(e) > 0: weights are exp2(s * scale_log2 - m)
    int32_t out_f32;
    FastDiv gdiv;      // g
    // split over the keys: arrival counts [units][hkv][1 + kJoin], and the sums,
    // sum_bytes for every workgroup of the grid (and, above kJoin splits, for
    // every kJoin of them)
    int32_t splits, units;
    int32_t narrow;  // 128-row tiles: the kernel with 32 keys a tile, where there is one
    char* sums;
    int64_t sum_bytes;
    unsigned* arrivals;
};

// Keys of a sequence, at most.  The kernels number keys, and round their ends up to
// tiles, in 32 bits.
constexpr int kMaxKeys = 0x7fffff00;

// The rows of sequence i, clamped to what there is.
struct Seq {
    int q0, n;       // query rows q0 .. q0 + n
    int64_t k0;      // first packed key row
    int len;         // keys
};

__device__ __forceinline__ int clamp_to(int v, int64_t hi) {
    return v < 0 ? 0 : (int64_t)v > hi ? (int)hi : v;
}

template <bool PAGED>
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int i) {
    Seq s;
    if (PAGED && !a.cu_q) {
        s.q0 = i;
        s.n = 1;
    } else {
        s.q0 = clamp_to(a.cu_q[i], a.tokens);
        const int end = clamp_to(a.cu_q[i + 1], a.tokens);
        s.n = end > s.q0 ? end - s.q0 : 0;
    }
    if (PAGED) {
        s.k0 = 0;
        const int64_t held = a.pages_st * (int64_t)a.page.d;
        s.len = clamp_to(a.kv_lens[i], held < kMaxKeys ? held : kMaxKeys);
    } else {
        const int32_t* cu = a.cu_k ? a.cu_k : a.cu_q;
        const int k0 = clamp_to(cu[i], a.tokens_k);
        const int end = clamp_to(cu[i + 1], a.tokens_k);
        s.k0 = k0;
        s.len = end > k0 ? end - k0 : 0;
    }
    return s;
}

// First key after the last one, and first key, that the query at position pos sees.
__device__ __forceinline__ int seen_end(const AttnArgs& a, int pos, int len) {
    return a.causal ? (pos + 1 < len ? pos + 1 : len) : len;
}
__device__ __forceinline__ int seen_begin(const AttnArgs& a, int pos) {
    if (a.window <= 0) return 0;
    const int64_t b = (int64_t)pos + 1 - a.window;
    return b > 0 ? (b > 0x7fffffff ? 0x7fffffff : (int)b) : 0;
}

// The last sequence that begins at or before query row `row`, which is the one
// that has it if any does.
__device__ __forceinline__ int seq_at(const AttnArgs& a, int64_t row) {
    if (!a.cu_q) return (int)row;
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_q[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}
// Element offset of key (or value) row j of a sequence; *srow, where paged, the
// row of its scale.
template <bool PAGED>
__device__ __forceinline__ int64_t kv_row(const AttnArgs& a, const Seq& s, const int32_t* table,
                                          int kvh, int j, int64_t st, int64_t sh, int64_t* srow) {
    if (!PAGED) return (s.k0 + j) * st + kvh * sh;
    const uint32_t pg = div_by(a.page, (uint32_t)j), slot = (uint32_t)j - pg * a.page.d;
    uint32_t id = (uint32_t)table[pg];
    id = (int64_t)id < a.pool_pages ? id : 0;
    const int64_t row = ((int64_t)id * a.hkv + kvh) * a.page.d + slot;
    *srow = row;
    return row * a.d;
}

// One query row (qr) over the keys [j0, j1) by one wave: a key per lane for the
// logits, an element of the head per lane for the sums (lane + 64 e in acc[e]).
// Keys outside the range are not read.  *m in log2 units.
template <typename T, typename C, bool PAGED>
__device__ __forceinline__ void attend_row(const AttnArgs& a, const Seq& s, const int32_t* table,
                                           int kvh, const T* qr, int j0, int j1, float* mo,
                                           float* lo, float (&acc)[4]) {
    const int lane = threadIdx.x & 63;
    const C* kp = static_cast<const C*>(a.k);
    const C* vp = static_cast<const C*>(a.v);
    float m = -__builtin_inff(), l = 0.0f;
    for (int e = 0; e < 4; e++) acc[e] = 0.0f;
    for (int j = j0; j < j1; j += 64) {
        const bool seen = j + lane < j1;
        float x = -__builtin_inff(), vs = 1.0f;
        if (seen) {
            int64_t sr = 0;
            const C* kr = kp + kv_row<PAGED>(a, s, table, kvh, j + lane, a.k_st, a.k_sh, &sr);
            float dot = 0.0f;
            for (int e = 0; e < a.d; e++) dot = fmaf(to_f32(qr[e]), to_f32(kr[e]), dot);
            if (sizeof(C) == 1) {
                dot *= a.ks[sr];
                vs = a.vs[sr];
            }
            x = dot * a.scale_log2;
        }
        float top = x;
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float mn = fmaxf(m, top), base = mn == -__builtin_inff() ? 0.0f : mn;
        const float p = seen ? exp2f(x - base) : 0.0f, fix = exp2f(m - base);
        float sum = p;
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        l = l * fix + sum;
        for (int e = 0; e < 4; e++) acc[e] *= fix;
        m = mn;
        const int n = j1 - j < 64 ? j1 - j : 64;
        for (int t = 0; t < n; t++) {
            int64_t sr = 0;
            const float w = __shfl(p * vs, t);
            const C* vr = vp + kv_row<PAGED>(a, s, table, kvh, j + t, a.v_st, a.v_sh, &sr);
            for (int e = 0; e < 4; e++)
                if (lane + 64 * e < a.d) acc[e] = fmaf(w, to_f32(vr[lane + 64 * e]), acc[e]);
        }
    }
    *mo = m;
    *lo = l;
}

// The head size that a matrix kernel is built for.
inline int64_t padded_head(int64_t d, bool f32) {
    return d <= 64 ? 64 : d <= 96 && !f32 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256;
}

// attn_any.hip: any head size up to 256, any strides and alignment.
int launch_attn_any(Ctx* c, const AttnArgs& a, int type, int kv_type);
// attn_tile_*.hip: many query rows per sequence and head, on the matrix units.
// 16-byte rows.
int launch_attn_tile_bf16(Ctx* c, const AttnArgs& a, bool i8);
int launch_attn_tile_f16(Ctx* c, const AttnArgs& a, bool i8);
int launch_attn_tile_f32(Ctx* c, const AttnArgs& a, bool i8);
// attn_few_*.hip: up to 32 query rows per sequence and key / value head, over a
// cache (int8 ones with d a multiple of 16).
int launch_attn_few_bf16(Ctx* c, const AttnArgs& a, bool i8, int blocks_of_16);
int launch_attn_few_f16(Ctx* c, const AttnArgs& a, bool i8, int blocks_of_16);
int launch_attn_few_f32(Ctx* c, const AttnArgs& a, bool i8, int blocks_of_16);
// Sums that one level of the splits' join reads; the most splits.
constexpr int kJoin = 16;
constexpr int kMaxSplits = kJoin * kJoin;
// Query rows (of all heads of one key / value head) that a workgroup takes.
constexpr int kTileRows = 128;

}  // namespace tkv
