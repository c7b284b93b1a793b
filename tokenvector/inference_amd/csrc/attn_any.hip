// attn_any.hip -- attention for any head size, stride and alignment.
//
// One wave per (query row, query head): 64 keys a step, a key per lane for the
// logits, an element of the head per lane for the sums (up to four of them),
// the running maximum and sum of the softmax in f32.  Every key row is read by
// one lane at a time, so this form is bound by its scattered loads: 1000 tokens of
// 4 heads of 33, bf16, 267 us, 1.0 TFLOP/s.  Layouts that the matrix kernels take
// (16-byte rows) come here only where a call has more units than a grid takes.
#include "attn.h"

namespace tkv {

template <typename T, typename C, bool PAGED>
__global__ __launch_bounds__(256) void k_attn_any(AttnArgs a) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t unit = wide_block() * 4 + wave;
    const int64_t row = unit / a.hq;
    const int h = (int)(unit - row * a.hq), kvh = h / a.g;
    if (row >= a.tokens) return;
    const int lo = seq_at(a, row);
    const Seq s = seq_of<PAGED>(a, lo);
    const int i = (int)row - s.q0;
    if (i < 0 || i >= s.n) return;  // no sequence covers the row
    const T* qr = static_cast<const T*>(a.q) + row * a.q_st + h * a.q_sh;

    const int pos = s.len - s.n + i;
    float m, l, acc[4];
    attend_row<T, C, PAGED>(a, s, PAGED ? a.pages + lo * a.pages_st : nullptr, kvh, qr,
                            seen_begin(a, pos), seen_end(a, pos, s.len), &m, &l, acc);
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
    const dim3 grid = wide_grid(ceil_div(a.tokens * a.hq, 4));
    if (a.pages) k_attn_any<T, C, true><<<grid, 256, 0, c->stream>>>(a);
    else k_attn_any<T, C, false><<<grid, 256, 0, c->stream>>>(a);
}

int launch_attn_any(Ctx* c, const AttnArgs& a, int type, int kv_type) {
    if (ceil_div(a.tokens * a.hq, 4) > kWideBlocks)
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
