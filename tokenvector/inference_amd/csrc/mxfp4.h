// mxfp4.h -- microscaled 4-bit floating point: its layouts, and what the
// kernels that code, decode and multiply it share.
//
// A row of k elements is ceil(k / 32) blocks of 16 code bytes (element 2i in
// the low half of byte i; the last block's missing elements are zeros) and as
// many scale bytes, 2^(byte - 127), 255 for a block that stands for NaN.
// The matrix kernels take the scales in slabs: [ceil(blocks / 8)][rows rounded
// up to 256][8], so that the scales of a tile's rows and of the 256 elements of
// a K slice are one run, which the copies to LDS and a wave's loads take whole.
// Blocks past the row's last have scale 0: 2^-127 on either side, products
// below 2^-240, which add nothing to an f32 sum.
#pragma once

#include <hip/hip_runtime.h>

#include "attn.h"
#include "mxfp4_plan.h"

namespace tkv {
namespace mx {

typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef v4i v4i_any __attribute__((aligned(2)));  // in memory, of any alignment
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kSlabRows = 256;
inline int64_t blocks_of(int64_t k) { return ceil_div(k, 32); }
inline int64_t slabs_of(int64_t k) { return ceil_div(blocks_of(k), 8); }
inline int64_t slab_rows(int64_t rows) { return ceil_div(rows, kSlabRows) * kSlabRows; }
inline size_t slab_bytes(int64_t rows, int64_t k) { return (size_t)(slabs_of(k) * slab_rows(rows) * 8); }

// A product's operands and output.  y rows ldy elements apart, of y_type.
struct Product {
    const uint8_t *a, *as;  // codes [m][blocks][16], scales
    const uint8_t *w, *ws;  // codes [n][blocks][16], scales
    int64_t m, n;
    int64_t a_rows, w_rows;  // of the scales' slabs; 0: they are [rows][blocks]
    int32_t blocks;
    const float* bias;
    void* y;
    int64_t ldy;
    int32_t y_type;
};
inline Shape shape_of(const Ctx* c, const Product& p) {
    return {p.m, p.n, p.blocks, c->num_cus, c->attn_arrivals != nullptr};
}

// The block's scale byte from its largest |x| as bits: floor(log2) - 2 (the
// largest code is 1.5 * 2^2), at least 2^-127, which blocks of zeros and
// subnormals get.
__device__ __forceinline__ unsigned scale_byte(unsigned most) {
    const unsigned e = most >> 23;
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// 2^(byte - 127), byte < 255
__device__ __forceinline__ float scale_value(unsigned byte) {
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
// Eight codes of x / scale: rounded to nearest even and saturated at 6 by
// v_cvt_scalef32_pk_fp4_f32 (the same as comparing with the midpoints for every
// finite float, subnormal scale included).
__device__ __forceinline__ unsigned code8(const float (&x)[8], float scale) {
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
}

// 8 elements as they are in memory.
template <typename T>
struct alignas(16) Quarter {
    unsigned v[2 * sizeof(T)];
};

// Without its first n elements, zeros behind the others.
template <typename T>
__device__ __forceinline__ void drop(Quarter<T>& q, int n) {
    constexpr int D = 2 * (int)sizeof(T);  // dwords
    const auto move = [&](bool is, int by) {
#pragma unroll
        for (int i = 0; i < D; i++) q.v[i] = !is ? q.v[i] : i + by < D ? q.v[i + by] : 0u;
    };
    move(n & 8, D);
    move(n & 4, D / 2);
    move(n & 2, D / 4);
    if constexpr (sizeof(T) == 4) {
        move(n & 1, 1);
    } else if (n & 1) {
#pragma unroll
        for (int i = 0; i < D; i++) q.v[i] = q.v[i] >> 16 | (i + 1 < D ? q.v[i + 1] << 16 : 0u);
    }
}
// 8 elements from `at` of a row of `cols` >= 8, zeros past its end, in two halves: at
// the row's end its last 8 are loaded, and end_quarter, when they are there, drops those
// before `at`.  So no lane's loads differ from the others', and several rows' are in
// flight together (8 x 4095 coded for 4096 outputs 6.5 us, with a branch for the last
// elements 9.3).  Global memory takes wide accesses of any alignment: 10482 x 2861 of
// f32 coded and read back 50 us, element by element 128.  RAGGED: cols is no multiple
// of 8.
template <typename T>
__device__ __forceinline__ Quarter<T> load_quarter(const T* row, int64_t at, int64_t cols) {
    Quarter<T> q;
    __builtin_memcpy(&q, row + (at < cols - 8 ? at : cols - 8), sizeof(q));
    return q;
}
template <typename T, bool RAGGED>
__device__ __forceinline__ void end_quarter(Quarter<T>& q, int64_t at, int64_t cols) {
    const int64_t past = at - (cols - 8);
    if (RAGGED) {
        if (past > 0) drop(q, past < 8 ? (int)past : 8);
    } else if (past >= 8) {
        q = Quarter<T>{};
    }
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));

// The largest of a lane's and its three neighbours' of four.
__device__ __forceinline__ unsigned neighbour_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
    return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}

// The code dword and scale byte of 8 elements, whose block's others are in the
// lane's three neighbours of four.  Of 16-bit types two magnitudes at a time are
// compared, as integers (infinities and NaN above all numbers), and converted as
// they are: the same codes as from f32, which every value of theirs was compared
// with at every scale.
template <typename T>
__device__ __forceinline__ unsigned code_quarter(const Quarter<T>& q, unsigned& byte) {
    unsigned code = 0;
    if constexpr (sizeof(T) == 4) {
        unsigned most = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) most = max(most, q.v[i] & 0x7fffffffu);
        byte = scale_byte(neighbour_max(most));
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __uint_as_float(q.v[i]);
        code = code8(x, scale_value(byte));
    } else {
        u16x2 m = __builtin_bit_cast(u16x2, q.v[0] & 0x7fff7fffu);
#pragma unroll
        for (int i = 1; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, q.v[i] & 0x7fff7fffu));
        unsigned most = neighbour_max(m.x > m.y ? m.x : m.y);
        if constexpr (__is_same(T, __bf16)) {
            byte = scale_byte(most << 16);
            const float scale = scale_value(byte);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(b16x2, q.v[0]), scale, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(b16x2, q.v[1]), scale, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(b16x2, q.v[2]), scale, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(b16x2, q.v[3]), scale, 3);
        } else {
            byte = scale_byte(__float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)most)));
            const float scale = scale_value(byte);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, __builtin_bit_cast(h16x2, q.v[0]), scale, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, __builtin_bit_cast(h16x2, q.v[1]), scale, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, __builtin_bit_cast(h16x2, q.v[2]), scale, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, __builtin_bit_cast(h16x2, q.v[3]), scale, 3);
        }
    }
    return byte == 255 ? 0u : code;
}

// The scales of a row's blocks 8 s .. 8 s + 7 from its [blocks] bytes, those past its
// last 0.  Nothing behind the row is read, and there is no branch on s, so that the
// loads of several s are in flight together.
__device__ __forceinline__ v2i row_scales(const uint8_t* row, int s, int blocks) {
    uint64_t v = 0;
    if (blocks >= 8) {
        const int at = 8 * s < blocks - 8 ? 8 * s : blocks - 8, past = 8 * s - at;
        __builtin_memcpy(&v, row + at, 8);
        v = past < 8 ? v >> (8 * past) : 0;
    } else if (s == 0) {
#pragma unroll
        for (int i = 0; i < 7; i++)
            if (i < blocks) v |= (uint64_t)row[i] << (8 * i);
    }
    return v2i{(int)(uint32_t)v, (int)(uint32_t)(v >> 32)};
}

}  // namespace mx

// A workspace; hipMalloc's error is taken off, or the next launch's check would
// report it.
int mx_room(Ctx* c, int slot, size_t bytes, void** out);
// mxfp4.hip.  x: rows of `cols` elements of `type`, `stride` elements apart.
// Scales to [rows][blocks], or to slabs.
int launch_mx_quantize(Ctx* c, int type, const void* x, int64_t stride, int64_t rows, int64_t cols,
                       uint8_t* codes, uint8_t* scales, bool slabs);
int launch_mx_dequantize(Ctx* c, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                         int64_t cols, int type, void* y, int64_t stride);
// Two operands' scales to slabs (rows_b 0: one's).
int launch_mx_slabs(Ctx* c, int64_t k, const uint8_t* a, int64_t rows_a, uint8_t* slabs_a, const uint8_t* b = nullptr,
                    int64_t rows_b = 0, uint8_t* slabs_b = nullptr);
// mxfp4_tile.hip.  Scales as slabs, or as rows where mx::takes_rows.
int launch_mx_product(Ctx* c, const mx::Product& p);
// mxfp4_few.hip: m <= kFewRows; and the linear that codes its rows itself, where
// mx::codes_few.
int launch_mx_few(Ctx* c, const mx::Product& p);
int launch_mx_few_linear(Ctx* c, int type, const void* x, int64_t stride, int64_t k, const mx::Product& p);
// The linear of a resident weight on float rows (mxfp4.hip).
int launch_mx_linear(Ctx* c, int type, const void* x, int64_t stride, int64_t k, mx::Product p);

}  // namespace tkv
