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

// n / d for n < 2^31 by a multiplication: (mulhi(m, n) + n) >> l.
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
    float scale_log2;  // scale * log2(e): weights are exp2(s * scale_log2 - m)
    int32_t out_f32;
};

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
        s.len = clamp_to(a.kv_lens[i], a.pages_st * (int64_t)a.page.d);
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

// attn_any.hip: any head size up to 256, any strides and alignment.
int launch_attn_any(Ctx* c, const AttnArgs& a, int type, int kv_type);

}  // namespace tkv
