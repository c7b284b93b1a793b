// attn_any.hip -- attention for any head size, stride and alignment.
//
// One wave per (query row, query head): 64 keys a step, a key per lane for the
// logits, an element of the head per lane for the sums (up to four of them),
// the running maximum and sum of the softmax in f32.  Every key row is read by
// one lane at a time, so this form is bound by its scattered loads; the layouts
// that the matrix kernels take (16-byte rows) never come here.
#include "attn.h"

namespace tkv {

template <typename C, bool PAGED>
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

template <typename T, typename C, bool PAGED>
__global__ __launch_bounds__(256) void k_attn_any(AttnArgs a) {
    __shared__ float qs[4][256];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
    const int64_t row = unit / a.hq;
    const int h = (int)(unit - row * a.hq), kvh = h / a.g;
    if (row >= a.tokens) return;
    // the last sequence that begins at or before the row
    int lo = 0, hi = a.seqs;
    if (PAGED && !a.cu_q) {
        lo = (int)row;
        hi = lo + 1;
    }
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_q[mid] <= row) lo = mid; else hi = mid;
    }
    if (lo >= a.seqs) return;
    const Seq s = seq_of<PAGED>(a, lo);
    const int i = (int)row - s.q0;
    if (i < 0 || i >= s.n) return;  // no sequence covers the row
    const T* qr = static_cast<const T*>(a.q) + row * a.q_st + h * a.q_sh;
    for (int e = lane; e < a.d; e += 64) qs[wave][e] = to_f32(qr[e]);
    __builtin_amdgcn_wave_barrier();

    const int pos = s.len - s.n + i;
    const int j0 = seen_begin(a, pos), j1 = seen_end(a, pos, s.len);
    const int32_t* table = PAGED ? a.pages + lo * a.pages_st : nullptr;
    const C* kp = static_cast<const C*>(a.k);
    const C* vp = static_cast<const C*>(a.v);
    float m = -__builtin_inff(), l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = j0; j < j1; j += 64) {
        const bool seen = j + lane < j1;
        float x = -__builtin_inff(), vs = 1.0f;
        if (seen) {
            int64_t sr = 0;
            const C* kr = kp + kv_row<C, PAGED>(a, s, table, kvh, j + lane, a.k_st, a.k_sh, &sr);
            float dot = 0.0f;
            for (int e = 0; e < a.d; e++) dot = fmaf(qs[wave][e], to_f32(kr[e]), dot);
            if (a.ks) {
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
            const C* vr = vp + kv_row<C, PAGED>(a, s, table, kvh, j + t, a.v_st, a.v_sh, &sr);
            for (int e = 0; e < 4; e++)
                if (lane + 64 * e < a.d) acc[e] = fmaf(w, to_f32(vr[lane + 64 * e]), acc[e]);
        }
    }
    const int64_t at = row * a.o_st + h * a.o_sh;
    for (int e = 0; e < 4; e++) {
        const int x = lane + 64 * e;
        if (x >= a.d) continue;
        const float y = l == 0.0f ? 0.0f : acc[e] / l;
        if (a.out_f32) static_cast<float*>(a.out)[at + x] = y;
        else static_cast<T*>(a.out)[at + x] = from_f32<T>(y);
    }
}

template <typename T, typename C>
static void launch_any(Ctx* c, const AttnArgs& a) {
    const dim3 grid((unsigned)ceil_div(a.tokens * a.hq, 4));
    if (a.pages) k_attn_any<T, C, true><<<grid, 256, 0, c->stream>>>(a);
    else k_attn_any<T, C, false><<<grid, 256, 0, c->stream>>>(a);
}

int launch_attn_any(Ctx* c, const AttnArgs& a, int type, int kv_type) {
    if (ceil_div(a.tokens * a.hq, 4) >= (1ll << 31))
        return set_error(TKV_HIP_UNSUPPORTED, "attention: too many rows");
    const bool i8 = kv_type == TKV_HIP_I8;
    if (type == TKV_HIP_F32) i8 ? launch_any<float, int8_t>(c, a) : launch_any<float, float>(c, a);
    else if (type == TKV_HIP_F16)
        i8 ? launch_any<_Float16, int8_t>(c, a) : launch_any<_Float16, _Float16>(c, a);
    else i8 ? launch_any<__bf16, int8_t>(c, a) : launch_any<__bf16, __bf16>(c, a);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

}  // namespace tkv
