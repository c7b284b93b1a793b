// mxfp4_few.hip -- products and linears of few rows with a 4-bit weight: the
// weight is streamed once, and its bytes are what bounds them.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 with the weight's rows as its rows and the
// tokens as its columns.  A lane's operand is a block of a row, 16 bytes and a
// scale byte, straight from memory: lanes of a row take the chunks of a 128-byte
// line (two instructions, 256 elements).  The waves of a workgroup take
// 256-element slabs of K in turn, each for all of the workgroup's 16 NR rows, and
// their sums are added in LDS in the waves' order.
//
// The linear's form codes the tokens on the way: a lane that multiplies block b of
// token t loads its 32 elements, has their maximum without any other lane, and
// holds the codes as the instruction takes them.  That is done again by every
// workgroup.
#include <type_traits>

#include "mxfp4.h"

namespace tkv {
namespace mx {

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct FewArgs {
    Product p;
    const void* x;  // the linear's rows
    int64_t stride, k;
    int32_t vec;    // rows of 16 bytes
};

template <typename T>
struct Block {
    u32x4 raw[sizeof(T) * 2];
};

// 32 elements from `at` of a row of k, zeros past its end.
template <typename T>
__device__ __forceinline__ Block<T> load_block(const T* row, int64_t at, int64_t k, bool vec) {
    Block<T> b;
    if (vec && at + 32 <= k) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) * 2; i++) b.raw[i] = reinterpret_cast<const u32x4*>(row + at)[i];
    } else {
        T e[32];
#pragma unroll
        for (int i = 0; i < 32; i++) e[i] = at + i < k ? row[at + i] : (T)0.0f;
        __builtin_memcpy(&b, e, sizeof(b));
    }
    return b;
}

// Codes and scale byte of a block held by one lane.  16-bit types: the largest
// magnitude of two at a time as integers (infinities and NaN above all numbers),
// and the conversions that take them.
template <typename T>
__device__ __forceinline__ v4i code_block(const Block<T>& b, unsigned& byte) {
    unsigned most = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) most = max(most, b.raw[i][j] & 0x7fffffffu);
    } else {
        u16x2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, b.raw[i][j] & 0x7fff7fffu));
        const unsigned short one = m.x > m.y ? m.x : m.y;
        if constexpr (std::is_same<T, __bf16>::value)
            most = (unsigned)one << 16;
        else
            most = __float_as_uint((float)__builtin_bit_cast(_Float16, one));
    }
    byte = scale_byte(most);
    if (byte == 255) return v4i{0, 0, 0, 0};
    const float scale = scale_value(byte);
    v4i c;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned w = 0;
        if constexpr (sizeof(T) == 4) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = __uint_as_float(b.raw[2 * i + j / 4][j & 3]);
            w = code8(x, scale);
        } else {
            // (values of their own: the compiler takes a vector's first element for
            // each where a bit cast names an element)
            const unsigned e0 = b.raw[i][0], e1 = b.raw[i][1], e2 = b.raw[i][2], e3 = b.raw[i][3];
            if constexpr (std::is_same<T, __bf16>::value) {
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b16x2, e0), scale, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b16x2, e1), scale, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b16x2, e2), scale, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(b16x2, e3), scale, 3);
            } else {
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h16x2, e0), scale, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h16x2, e1), scale, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h16x2, e2), scale, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(h16x2, e3), scale, 3);
            }
        }
        c[i] = (int)w;
    }
    return c;
}

struct Coded {};      // the tokens come as codes and slabs,
struct CodedRows {};  // or the scales of both as [rows][blocks]

template <typename TI, int NR, int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void k_mx_few(FewArgs a) {
    constexpr bool ROWS = std::is_same<TI, CodedRows>::value, CODED = ROWS || std::is_same<TI, Coded>::value;
    typedef typename std::conditional<CODED, float, TI>::type TX;
    const Product& p = a.p;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int64_t n0 = wide_block() * (16 * NR);
    if (n0 >= p.n) return;
    const uint32_t row_bytes = (uint32_t)p.blocks * 16u;
    const int slabs = (p.blocks + 7) >> 3;

    // rows past the weight's, and tokens past m, read the last one
    const uint8_t* w_row[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const int64_t row = n0 + r * 16 + l16;
        w_row[r] = p.w + (row < p.n ? row : p.n - 1) * row_bytes;
    }
    int64_t token[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) token[t] = t * 16 + l16 < p.m ? t * 16 + l16 : p.m - 1;

    struct Slab {
        v4i w[NR][2];
        v2i ws[NR];
        v4i t[CODED ? MT : 1][2];
        v2i ts[CODED ? MT : 1];
        Block<TX> x[CODED ? 1 : MT][2];
    };
    const auto load = [&](int s, Slab& b) {
        uint32_t at[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            at[h] = (uint32_t)s * 128u + (uint32_t)(h * 64 + g * 16);
            at[h] = at[h] < row_bytes ? at[h] : row_bytes - 16;  // past the row: its scales are 2^-127
        }
#pragma unroll
        for (int r = 0; r < NR; r++) {
#pragma unroll
            for (int h = 0; h < 2; h++) b.w[r][h] = *reinterpret_cast<const v4i*>(w_row[r] + at[h]);
            if constexpr (ROWS) {
                const int64_t row = n0 + r * 16 + l16;
                b.ws[r] = row_scales(p.ws + (row < p.n ? row : p.n - 1) * p.blocks, s, p.blocks);
            } else {
                b.ws[r] = *reinterpret_cast<const v2i*>(p.ws + ((int64_t)s * p.w_rows + n0 + r * 16 + l16) * 8);
            }
        }
#pragma unroll
        for (int t = 0; t < MT; t++) {
            if constexpr (CODED) {
#pragma unroll
                for (int h = 0; h < 2; h++)
                    b.t[t][h] = *reinterpret_cast<const v4i*>(p.a + token[t] * row_bytes + at[h]);
                if constexpr (ROWS) b.ts[t] = row_scales(p.as + token[t] * p.blocks, s, p.blocks);
                else b.ts[t] = *reinterpret_cast<const v2i*>(p.as + ((int64_t)s * p.a_rows + t * 16 + l16) * 8);
            } else {
                // (one lane of a token that is not there does what the last token's does)
                const TX* row = static_cast<const TX*>(a.x) + token[t] * a.stride;
#pragma unroll
                for (int h = 0; h < 2; h++)
                    b.x[t][h] = load_block<TX>(row, ((int64_t)s * 8 + h * 4 + g) * 32, a.k, a.vec);
            }
        }
    };

    v4f acc[NR][MT];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int t = 0; t < MT; t++) acc[r][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    Slab cur;
    if (wave < slabs) load(wave, cur);
    for (int s = wave; s < slabs; s += WAVES) {
        Slab next;
        if (s + WAVES < slabs) load(s + WAVES, next);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v4i tc[MT];
            unsigned tb[MT];
#pragma unroll
            for (int t = 0; t < MT; t++) {
                if constexpr (CODED) {
                    tc[t] = cur.t[t][h];
                    tb[t] = (unsigned)cur.ts[t][h] >> (8 * g);
                } else {
                    tc[t] = code_block<TX>(cur.x[t][h], tb[t]);
                    // (blocks past the row are zeros, and their scale 2^-127)
                }
            }
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const v4i w = cur.w[r][h];
                const unsigned wb = (unsigned)cur.ws[r][h] >> (8 * g);
#pragma unroll
                for (int t = 0; t < MT; t++)
                    acc[r][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        v8i{w.x, w.y, w.z, w.w, 0, 0, 0, 0}, v8i{tc[t].x, tc[t].y, tc[t].z, tc[t].w, 0, 0, 0, 0},
                        acc[r][t], 4, 4, 0, (int)wb, 0, (int)tb[t]);
            }
        }
        cur = next;
    }

    // a lane holds rows 4 g .. 4 g + 3 of 16 for token l16
    __shared__ v4f part[WAVES][NR * MT][64];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int t = 0; t < MT; t++) part[wave][r * MT + t][lane] = acc[r][t];
    __syncthreads();
    for (int i = wave; i < NR * MT; i += WAVES) {
        v4f sum = part[0][i][lane];
#pragma unroll
        for (int w = 1; w < WAVES; w++) sum += part[w][i][lane];
        const int64_t tok = (i % MT) * 16 + l16, n = n0 + (i / MT) * 16 + g * 4;
        if (tok >= p.m) continue;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (n + e >= p.n) break;
            const float y = sum[e] + (p.bias ? p.bias[n + e] : 0.0f);
            const int64_t at = tok * p.ldy + n + e;
            if (p.y_type == TKV_HIP_F32) static_cast<float*>(p.y)[at] = y;
            else if (p.y_type == TKV_HIP_F16) static_cast<_Float16*>(p.y)[at] = from_f32<_Float16>(y);
            else static_cast<__bf16*>(p.y)[at] = from_f32<__bf16>(y);
        }
    }
}

template <typename TI, int MT>
static int launch_few(Ctx* c, const FewArgs& a) {
    constexpr int WAVES = 8;
    const int64_t rows = ceil_div(a.p.n, 16);
    // rows a workgroup: as many as leave a workgroup per CU
    if (rows >= 4 * c->num_cus)
        k_mx_few<TI, 4, MT, WAVES><<<wide_grid(ceil_div(rows, 4)), WAVES * 64, 0, c->stream>>>(a);
    else if (rows >= 2 * c->num_cus)
        k_mx_few<TI, 2, MT, WAVES><<<wide_grid(ceil_div(rows, 2)), WAVES * 64, 0, c->stream>>>(a);
    else
        k_mx_few<TI, 1, MT, WAVES><<<wide_grid(rows), WAVES * 64, 0, c->stream>>>(a);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

}  // namespace mx

using namespace mx;

int launch_mx_few(Ctx* c, const Product& p) {
    FewArgs a = {};
    a.p = p;
    if (p.a_rows == 0) {
        if (p.m <= 16) return launch_few<CodedRows, 1>(c, a);
        if (p.m <= 32) return launch_few<CodedRows, 2>(c, a);
        return launch_few<CodedRows, 4>(c, a);
    }
    if (p.m <= 16) return launch_few<Coded, 1>(c, a);
    if (p.m <= 32) return launch_few<Coded, 2>(c, a);
    return launch_few<Coded, 4>(c, a);
}

int launch_mx_few_linear(Ctx* c, int type, const void* x, int64_t stride, int64_t k, const Product& p) {
    FewArgs a = {};
    a.p = p;
    a.x = x;
    a.stride = stride;
    a.k = k;
    a.vec = aligned(x, 16) && stride * type_bytes(type) % 16 == 0;
    if (type == TKV_HIP_F32) return launch_few<float, 1>(c, a);
    if (type == TKV_HIP_F16) return launch_few<_Float16, 1>(c, a);
    return launch_few<__bf16, 1>(c, a);
}

}  // namespace tkv
