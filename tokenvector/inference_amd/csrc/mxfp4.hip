// mxfp4.hip -- microscaled 4-bit floating point: rows coded and decoded, the
// scales' slabs, and the entry points.
#include "mxfp4.h"

namespace tkv {
namespace mx {

template <typename T>
struct alignas(16) Chunk {
    T e[8];
};

struct CodeArgs {
    const void* x;
    int64_t stride;
    uint8_t *codes, *scales;
    int64_t slab_rows;
    int64_t rows, cols;
    int32_t blocks, per_row;  // of a row; of a row with the slabs' padding
    FastDiv div;              // per_row
};

// A lane takes 8 elements of a block, so that loads, and the stores of codes,
// are runs of a wave; the block's maximum goes over its 4 lanes.
template <typename T, bool SLABS, bool RAGGED>
__global__ __launch_bounds__(256) void k_mx_code(CodeArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t b = (uint32_t)(t >> 2);
    if (b >= (uint64_t)a.rows * a.per_row) return;  // whole blocks: their lanes stay together
    const uint32_t row = div_by(a.div, b);
    const int block = (int)(b - row * a.per_row), part = (int)threadIdx.x & 3;
    const int64_t at = (int64_t)block * 32 + part * 8;
    unsigned byte;
    const T* from = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
    Quarter<T> x = {};
    if (!RAGGED || a.cols >= 8) {
        x = load_quarter<T>(from, at, a.cols);
        end_quarter<T, RAGGED>(x, at, a.cols);
    } else {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = at + i < a.cols ? from[at + i] : (T)0.0f;
        __builtin_memcpy(&x, e, sizeof(x));
    }
    const unsigned code = code_quarter<T>(x, byte);
    if (block < a.blocks)
        reinterpret_cast<unsigned*>(a.codes)[((int64_t)row * a.blocks + block) * 4 + part] = code;
    if (part == 0) {
        if (SLABS)
            a.scales[((int64_t)(block >> 3) * a.slab_rows + row) * 8 + (block & 7)] =
                block < a.blocks ? (uint8_t)byte : (uint8_t)0;
        else
            a.scales[(int64_t)row * a.blocks + block] = (uint8_t)byte;
    }
}

struct DecodeArgs {
    const uint8_t *codes, *scales;
    void* y;
    int64_t stride;
    int64_t rows, cols;
    int32_t blocks;
    FastDiv div;  // blocks
};

// Each value is its code's times a power of two: exact in f32 but for what
// passes its range, and rounded once to the output's type.  STREAM: the stores go past
// the L2's reuse (16384 x 8192 of bf16 coded and read back 130 -> 110 us, 8001 x 4001
// 34 -> 28); not f32 rows that start anywhere, whose two stores a lane leave parts of
// lines to each other (10482 x 2861 50 -> 70).
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void k_mx_decode(DecodeArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t b = (uint32_t)(t >> 2);
    if (b >= (uint64_t)a.rows * a.blocks) return;
    const uint32_t row = div_by(a.div, b);
    const int block = (int)(b - row * a.blocks), part = (int)threadIdx.x & 3;
    const int64_t at = (int64_t)block * 32 + part * 8;
    if (at >= a.cols) return;
    const unsigned code = reinterpret_cast<const unsigned*>(a.codes)[((int64_t)row * a.blocks + block) * 4 + part];
    const unsigned byte = a.scales[(int64_t)row * a.blocks + block];
    const float scale = byte == 255 ? __uint_as_float(0x7fc00000u) : scale_value(byte);
    float x[8];
    const v2f p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0);
    const v2f p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1);
    const v2f p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2);
    const v2f p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3);
    x[0] = p0[0] * scale, x[1] = p0[1] * scale, x[2] = p1[0] * scale, x[3] = p1[1] * scale;
    x[4] = p2[0] * scale, x[5] = p2[1] * scale, x[6] = p3[0] * scale, x[7] = p3[1] * scale;
    // (a product folded into its conversion to f16 is an fma on +0, which takes the
    // sign off a zero: the values stay apart from it)
#pragma unroll
    for (int i = 0; i < 8; i++) asm("" : "+v"(x[i]));
    T* dst = static_cast<T*>(a.y) + (int64_t)row * a.stride + at;
    if (at + 8 <= a.cols) {
        Chunk<T> v;
#pragma unroll
        for (int i = 0; i < 8; i++) v.e[i] = from_f32<T>(x[i]);
        v4i w[sizeof(T) / 2];
        __builtin_memcpy(w, &v, sizeof(v));
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            if (STREAM) __builtin_nontemporal_store(w[i], reinterpret_cast<v4i_any*>(dst) + i);
            else reinterpret_cast<v4i_any*>(dst)[i] = w[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (at + i < a.cols) dst[i] = from_f32<T>(x[i]);
    }
}

// Row-major scales of one or two operands to slabs: a workgroup takes 32 rows (numbered
// over two dimensions of the grid) of eight slabs, so that loads and stores are both runs of 64 bytes (products of 4096 x 256 of
// 16384 26.2 -> 24.4 us, 1024 x 14336 of 4096 39.1 -> 38.0; before, a row a lane).
struct SlabArgs {
    const uint8_t* scales[2];
    uint8_t* out[2];
    int64_t rows[2];
    int32_t blocks;
    int64_t first;  // groups of 32 rows of the first operand
};
__global__ __launch_bounds__(256) void k_mx_slabs(SlabArgs a) {
    const int64_t group = wide_block();
    const int which = group >= a.first;
    const int64_t row = (group - (which ? a.first : 0)) * 32 + (threadIdx.x >> 3);
    const int64_t rows = which ? a.rows[1] : a.rows[0], padded = (rows + kSlabRows - 1) / kSlabRows * kSlabRows;
    const int g = (int)blockIdx.z * 8 + (threadIdx.x & 7);
    if (row >= rows || g * 8 >= a.blocks) return;
    const uint8_t* from = (which ? a.scales[1] : a.scales[0]) + row * a.blocks;
    uint8_t* out = which ? a.out[1] : a.out[0];
    *reinterpret_cast<v2i*>(out + (g * padded + row) * 8) = row_scales(from, g, a.blocks);
}

// Blocks of one launch, at most: their number is divided in 32 bits, and 4 lanes
// of each fit a dimension of the grid.
constexpr int64_t kLaunchBlocks = 1ll << 29;

template <typename T>
static int code_rows(Ctx* c, const void* x, int64_t stride, int64_t rows, int64_t cols, uint8_t* codes,
                     uint8_t* scales, bool slabs) {
    const int64_t blocks = blocks_of(cols), per_row = slabs ? slabs_of(cols) * 8 : blocks;
    const int64_t step = kLaunchBlocks / per_row;
    for (int64_t r = 0; r < rows; r += step) {
        CodeArgs a;
        a.x = static_cast<const T*>(x) + r * stride;
        a.stride = stride;
        a.codes = codes + r * blocks * 16;
        a.scales = scales + r * (slabs ? 8 : blocks);
        a.slab_rows = slab_rows(rows);
        a.rows = rows - r < step ? rows - r : step;
        a.cols = cols;
        a.blocks = (int32_t)blocks;
        a.per_row = (int32_t)per_row;
        a.div = fast_div((uint32_t)per_row);
        const unsigned grid = (unsigned)ceil_div(a.rows * per_row * 4, 256);
        if (slabs) {
            if (cols % 8) k_mx_code<T, true, true><<<grid, 256, 0, c->stream>>>(a);
            else k_mx_code<T, true, false><<<grid, 256, 0, c->stream>>>(a);
        } else {
            if (cols % 8) k_mx_code<T, false, true><<<grid, 256, 0, c->stream>>>(a);
            else k_mx_code<T, false, false><<<grid, 256, 0, c->stream>>>(a);
        }
        TKV_LAUNCH_CHECK();
    }
    return TKV_HIP_OK;
}

template <typename T>
static int decode_rows(Ctx* c, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* y,
                       int64_t stride) {
    const int64_t blocks = blocks_of(cols), step = kLaunchBlocks / blocks;
    const bool past = sizeof(T) == 2 || (aligned(y, 16) && stride * (int64_t)sizeof(T) % 16 == 0);
    for (int64_t r = 0; r < rows; r += step) {
        DecodeArgs a;
        a.codes = codes + r * blocks * 16;
        a.scales = scales + r * blocks;
        a.y = static_cast<T*>(y) + r * stride;
        a.stride = stride;
        a.rows = rows - r < step ? rows - r : step;
        a.cols = cols;
        a.blocks = (int32_t)blocks;
        a.div = fast_div((uint32_t)blocks);
        const unsigned grid = (unsigned)ceil_div(a.rows * blocks * 4, 256);
        if (past) k_mx_decode<T, true><<<grid, 256, 0, c->stream>>>(a);
        else k_mx_decode<T, false><<<grid, 256, 0, c->stream>>>(a);
        TKV_LAUNCH_CHECK();
    }
    return TKV_HIP_OK;
}

}  // namespace mx

using namespace mx;

int launch_mx_quantize(Ctx* c, int type, const void* x, int64_t stride, int64_t rows, int64_t cols, uint8_t* codes,
                       uint8_t* scales, bool slabs) {
    if (type == TKV_HIP_F32) return code_rows<float>(c, x, stride, rows, cols, codes, scales, slabs);
    if (type == TKV_HIP_F16) return code_rows<_Float16>(c, x, stride, rows, cols, codes, scales, slabs);
    return code_rows<__bf16>(c, x, stride, rows, cols, codes, scales, slabs);
}

int launch_mx_dequantize(Ctx* c, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, int type,
                         void* y, int64_t stride) {
    if (type == TKV_HIP_F32) return decode_rows<float>(c, codes, scales, rows, cols, y, stride);
    if (type == TKV_HIP_F16) return decode_rows<_Float16>(c, codes, scales, rows, cols, y, stride);
    return decode_rows<__bf16>(c, codes, scales, rows, cols, y, stride);
}

int launch_mx_slabs(Ctx* c, int64_t k, const uint8_t* sa, int64_t rows_a, uint8_t* slabs_a, const uint8_t* sb,
                    int64_t rows_b, uint8_t* slabs_b) {
    const int64_t first = ceil_div(rows_a, 32);
    const SlabArgs a = {{sa, sb}, {slabs_a, slabs_b}, {rows_a, rows_b}, (int32_t)blocks_of(k), first};
    dim3 grid = wide_grid(first + ceil_div(rows_b, 32));
    grid.z = (unsigned)ceil_div(slabs_of(k), 8);
    k_mx_slabs<<<grid, 256, 0, c->stream>>>(a);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

int mx_room(Ctx* c, int slot, size_t bytes, void** out) {
    const int rc = ctx_workspace(c, slot, bytes, out);
    if (rc == TKV_HIP_OOM) (void)hipGetLastError();
    return rc;
}

int launch_mx_linear(Ctx* c, int type, const void* x, int64_t stride, int64_t k, Product p) {
    if (codes_few(shape_of(c, p), k)) return launch_mx_few_linear(c, type, x, stride, k, p);
    void *codes, *slabs;
    TKV_RC_TRY(mx_room(c, 0, (size_t)(p.m * p.blocks) * 16, &codes));
    TKV_RC_TRY(mx_room(c, 1, slab_bytes(p.m, k), &slabs));
    TKV_RC_TRY(launch_mx_quantize(c, type, x, stride, p.m, k, static_cast<uint8_t*>(codes),
                                  static_cast<uint8_t*>(slabs), true));
    p.a = static_cast<uint8_t*>(codes);
    p.as = static_cast<uint8_t*>(slabs);
    p.a_rows = slab_rows(p.m);
    return launch_mx_product(c, p);
}

// Sizes that coding and decoding take: a launch's blocks are numbered in 32 bits, and
// a row's (2^26 at most) are one launch's.
static bool sizes_ok(int64_t rows, int64_t cols) {
    return rows >= 0 && rows < (1ll << 31) && cols > 0 && cols < (1ll << 31);
}

}  // namespace tkv

using namespace tkv;

extern "C" {

int32_t tkv_hip_dev_quantize_mxfp4(int64_t ctx, int32_t type, const void* x, int64_t stride, int64_t rows,
                                   int64_t cols, uint8_t* codes, uint8_t* scales) {
    if (!float_type(type)) return set_error(TKV_HIP_BAD_ARG, "quantize_mxfp4: types are F32, F16 or BF16");
    if (!sizes_ok(rows, cols) || (rows > 1 && stride < cols))
        return set_error(TKV_HIP_BAD_ARG, "quantize_mxfp4: sizes out of range, or a stride below cols");
    if (rows == 0) return TKV_HIP_OK;
    if (!x || !codes || !scales || !aligned(codes, 16) || !aligned(x, type_bytes(type)))
        return set_error(TKV_HIP_BAD_ARG, "quantize_mxfp4: NULL or unaligned buffers (codes: 16 bytes)");
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    return launch_mx_quantize(c, type, x, rows > 1 ? stride : cols, rows, cols, codes, scales, false);
}

int32_t tkv_hip_dev_dequantize_mxfp4(int64_t ctx, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                     int64_t cols, int32_t type, void* y, int64_t stride) {
    if (!float_type(type)) return set_error(TKV_HIP_BAD_ARG, "dequantize_mxfp4: types are F32, F16 or BF16");
    if (!sizes_ok(rows, cols) || (rows > 1 && stride < cols))
        return set_error(TKV_HIP_BAD_ARG, "dequantize_mxfp4: sizes out of range, or a stride below cols");
    if (rows == 0) return TKV_HIP_OK;
    if (!y || !codes || !scales || !aligned(codes, 16) || !aligned(y, type_bytes(type)))
        return set_error(TKV_HIP_BAD_ARG, "dequantize_mxfp4: NULL or unaligned buffers (codes: 16 bytes)");
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    return launch_mx_dequantize(c, codes, scales, rows, cols, type, y, rows > 1 ? stride : cols);
}

int32_t tkv_hip_dev_matmul_mxfp4(int64_t ctx, const uint8_t* a, const uint8_t* a_scales, const uint8_t* w,
                                 const uint8_t* w_scales, int64_t m, int64_t n, int64_t k, const float* bias,
                                 int32_t type_out, void* y, int64_t stride) {
    if (!float_type(type_out)) return set_error(TKV_HIP_BAD_ARG, "matmul_mxfp4: types are F32, F16 or BF16");
    if (m < 0 || n < 0 || k <= 0 || (m > 1 && stride < n))
        return set_error(TKV_HIP_BAD_ARG, "matmul_mxfp4: sizes out of range, or a stride below N");
    if (m >= (1ll << 31) || n >= (1ll << 28) || k >= (1ll << 17))
        return set_error(TKV_HIP_UNSUPPORTED, "matmul_mxfp4: K must be below 2^17, M below 2^31 and N below 2^28");
    if (m == 0 || n == 0) return TKV_HIP_OK;
    if (!a || !a_scales || !w || !w_scales || !y || !aligned(a, 16) || !aligned(w, 16) ||
        !aligned(y, type_bytes(type_out)) || !aligned(bias, 4))
        return set_error(TKV_HIP_BAD_ARG, "matmul_mxfp4: NULL or unaligned buffers (codes: 16 bytes)");
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    mx::Product p = {};
    p.a = a;
    p.as = a_scales;
    p.w = w;
    p.ws = w_scales;
    p.m = m;
    p.n = n;
    p.blocks = (int32_t)blocks_of(k);
    p.bias = bias;
    p.y = y;
    p.ldy = m > 1 ? stride : n;
    p.y_type = type_out;
    if (!mx::takes_rows(mx::shape_of(c, p))) {
        void *as, *ws;
        TKV_RC_TRY(mx_room(c, 1, slab_bytes(m, k), &as));
        TKV_RC_TRY(mx_room(c, 2, slab_bytes(n, k), &ws));
        TKV_RC_TRY(launch_mx_slabs(c, k, a_scales, m, static_cast<uint8_t*>(as), w_scales, n, static_cast<uint8_t*>(ws)));
        p.as = static_cast<uint8_t*>(as);
        p.ws = static_cast<uint8_t*>(ws);
        p.a_rows = slab_rows(m);
        p.w_rows = slab_rows(n);
    }
    return launch_mx_product(c, p);
}

}  // extern "C"
