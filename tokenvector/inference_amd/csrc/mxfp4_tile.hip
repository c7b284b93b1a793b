// mxfp4_tile.hip -- the product of microscaled 4-bit operands,
//   y[m, n] = sum_k a[m, k] w[n, k] + bias[n],
// on v_mfma_scale_f32_32x32x64_f8f6f4.  A lane's operand is one block, 16 bytes
// of codes and its scale byte, so the block scales cost nothing in the product;
// products are exact and sums f32 (within 2^-20 of the largest term for each
// instruction).
//
// Tiles: 4 waves, each a quarter of the workgroup's BM x BN outputs.  K goes in
// slices of 256 elements, 128 bytes a row: copied HBM / L2 -> LDS by
// global_load_lds into one of two stages while the other is multiplied.  Rows
// lie in LDS in 16-byte chunks whose place is XORed with the row, so that the
// 32 rows that a fragment's read takes spread over the banks; the copies are
// linear in LDS, so each lane fetches the chunk that belongs there.
//
// Order within a slice, of four steps of 64 elements: the next step's fragments
// are read while this one's are multiplied.  Before the last step's products
// the wave waits for its part of the next slice (copied during the whole slice)
// and for its own reads; behind the barrier the stage just read is free for the
// copies of the slice after next, and the next slice's first fragments are
// read while the last step is multiplied.
#include <type_traits>

#include "mxfp4.h"

namespace tkv {
namespace mx {

typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ __forceinline__ int chunk_xor(int row) { return (row >> 1) & 7; }

// Workgroups go to the 8 XCDs in turn: each XCD takes a contiguous range of
// tiles, and within it bands of 8 tile rows column by column, so that the tiles
// that run together share rows and columns in its L2.
__device__ __forceinline__ void tile_of(int64_t block, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int total = tiles_m * tiles_n, per = total >> 3, rem = total & 7;
    const int x = (int)(block & 7), j = (int)(block >> 3);
    const int t = x < rem ? x * (per + 1) + j : rem * (per + 1) + (x - rem) * per + j;
    const int band = t / (8 * tiles_n), first = band * 8;
    const int high = tiles_m - first < 8 ? tiles_m - first : 8, in = t - first * tiles_n;
    tm = first + in % high;
    tn = in / high;
}

template <int TM, int TN>  // 32 x 32 blocks of a wave
struct Tile {
    static constexpr int BM = 64 * TM, BN = 64 * TN;
    static constexpr int CODES = (BM + BN) * 128, SCALES = (BM + BN) * 8;
    static constexpr int STAGE = CODES + SCALES;
    static constexpr int PER_CU = STAGE * 4 <= 163840 ? 2 : 1;
};

template <int TM, int TN, typename TO>
__global__ __launch_bounds__(256, (Tile<TM, TN>::PER_CU)) void k_mx_tile(Product p, int tiles_m, int tiles_n) {
    using T = Tile<TM, TN>;
    constexpr int BM = T::BM, BN = T::BN;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * T::STAGE];
    const int64_t block = wide_block();
    if (block >= (int64_t)tiles_m * tiles_n) return;
    int tm, tn;
    tile_of(block, tiles_m, tiles_n, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, half = lane >> 5, l32 = lane & 31;
    const uint32_t row_bytes = (uint32_t)p.blocks * 16u;

    // copies: 1 KB, 8 rows, each; (BM + BN) / 32 of them a wave.  Groups of rows
    // that the operand does not have read its first instead; what passes its last
    // row's end the buffer's bounds turn into zeros.  Past a row's end is the next
    // row, which the scales 2^-127 there leave out.
    constexpr int COPIES = (BM + BN) / 32;
    const int rows_a = p.m - m0 < BM ? (int)(p.m - m0) : BM, rows_w = p.n - n0 < BN ? (int)(p.n - n0) : BN;
    const auto buffer_of = [&](const uint8_t* base, int rows) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, rows * (int)row_bytes, 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t from_a = buffer_of(p.a + m0 * row_bytes, rows_a);
    const __amdgpu_buffer_rsrc_t from_w = buffer_of(p.w + n0 * row_bytes, rows_w);
    // (a copy's first row is a multiple of 8: its part of chunk_xor is the wave's)
    const uint32_t lane_at =
        (uint32_t)(lane >> 3) * row_bytes + (uint32_t)(((lane & 7) ^ chunk_xor(wave * 8 + (lane >> 3))) * 16);
    constexpr int SBYTES = T::SCALES / 4;  // of a wave
    constexpr int SWIDTH = SBYTES % 1024 == 0 ? 16 : 4, SCOPIES = SBYTES / (64 * SWIDTH);
    const auto copy = [&](int slice, uint8_t* stage) {
#pragma unroll
        for (int d = 0; d < COPIES; d++) {
            const int first = (d * 4 + wave) * 8, in = d * 32 < BM ? first : first - BM;
            const uint32_t at = (in < (d * 32 < BM ? rows_a : rows_w) ? (uint32_t)in * row_bytes : 0u) + (uint32_t)slice * 128u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(d * 32 < BM ? from_a : from_w, (lds_ptr)(stage + first * 128), 16,
                                                     (int)lane_at, (int)at, 0, 0);
        }
#pragma unroll
        for (int d = 0; d < SCOPIES; d++) {
            const int at = (d * 4 + wave) * 64 * SWIDTH;
            const uint8_t* src = at < BM * 8 ? p.as + ((int64_t)slice * p.a_rows + m0) * 8 + at
                                             : p.ws + ((int64_t)slice * p.w_rows + n0) * 8 + (at - BM * 8);
            const void* from = src + lane * SWIDTH;
            if constexpr (SWIDTH == 16)
                __builtin_amdgcn_global_load_lds(from, (lds_ptr)(stage + T::CODES + at), 16, 0, 0);
            else
                __builtin_amdgcn_global_load_lds(from, (lds_ptr)(stage + T::CODES + at), 4, 0, 0);
        }
    };

    v16f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;

    v4i fa[2][TM], fw[2][TN];
    v2i sa[TM], sw[TN];                      // a slice's scales as read,
    int la[TM], ha[TM], lw[TN], hw[TN];      // and shifted
    const int ra = wm * TM * 32 + l32, rw = BM + wn * TN * 32 + l32;
    const int x = chunk_xor(l32);
    const auto read = [&](const uint8_t* stage, int step, int set) {
        const int c = ((2 * step + half) ^ x) * 16;
#pragma unroll
        for (int i = 0; i < TM; i++)
            fa[set][i] = *reinterpret_cast<const v4i*>(stage + (ra + i * 32) * 128 + c);
#pragma unroll
        for (int j = 0; j < TN; j++)
            fw[set][j] = *reinterpret_cast<const v4i*>(stage + (rw + j * 32) * 128 + c);
    };
    // a lane's blocks are 2 step + half: shifted so, step's byte is 2 (step % 2)
    const auto read_scales = [&](const uint8_t* stage) {
#pragma unroll
        for (int i = 0; i < TM; i++) sa[i] = *reinterpret_cast<const v2i*>(stage + T::CODES + (ra + i * 32) * 8);
#pragma unroll
        for (int j = 0; j < TN; j++) sw[j] = *reinterpret_cast<const v2i*>(stage + T::CODES + (rw + j * 32) * 8);
    };
    const auto shift_scales = [&]() {
#pragma unroll
        for (int i = 0; i < TM; i++) {
            la[i] = (int)((unsigned)sa[i].x >> (8 * half));
            ha[i] = (int)((unsigned)sa[i].y >> (8 * half));
        }
#pragma unroll
        for (int j = 0; j < TN; j++) {
            lw[j] = (int)((unsigned)sw[j].x >> (8 * half));
            hw[j] = (int)((unsigned)sw[j].y >> (8 * half));
        }
    };
    // the products of one step, between them nothing else
    const auto multiply = [&](auto step) {
        constexpr int S = decltype(step)::value;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const v4i a4 = fa[S & 1][i], w4 = fw[S & 1][j];
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                    v8i{a4.x, a4.y, a4.z, a4.w, 0, 0, 0, 0}, v8i{w4.x, w4.y, w4.z, w4.w, 0, 0, 0, 0}, acc[i][j], 4, 4,
                    2 * (S & 1), S < 2 ? la[i] : ha[i], 2 * (S & 1), S < 2 ? lw[j] : hw[j]);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto sync = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    const int slices = (p.blocks + 7) >> 3;
    constexpr int VM = COPIES + SCOPIES;
    static_assert(VM < 64, "vmcnt range");
    copy(0, lds);
    if (slices > 1) {
        copy(1, lds + T::STAGE);
        __builtin_amdgcn_s_waitcnt(0x0F70 | (VM & 15) | ((VM >> 4) << 14));
    } else {
        __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    sync();
    read_scales(lds);
    read(lds, 0, 0);
    for (int s = 0; s < slices - 1; s++) {
        uint8_t* stage = lds + (s & 1) * T::STAGE;
        const uint8_t* next = lds + ((s + 1) & 1) * T::STAGE;
        shift_scales();
        read(stage, 1, 1);
        multiply(std::integral_constant<int, 0>{});
        read(stage, 2, 0);
        multiply(std::integral_constant<int, 1>{});
        read(stage, 3, 1);
        multiply(std::integral_constant<int, 2>{});
        __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's copies of slice s + 1
        sync();
        if (s + 2 < slices) copy(s + 2, stage);
        read_scales(next);
        read(next, 0, 0);
        multiply(std::integral_constant<int, 3>{});
    }
    const uint8_t* stage = lds + ((slices - 1) & 1) * T::STAGE;
    shift_scales();
    read(stage, 1, 1);
    multiply(std::integral_constant<int, 0>{});
    read(stage, 2, 0);
    multiply(std::integral_constant<int, 1>{});
    read(stage, 3, 1);
    multiply(std::integral_constant<int, 2>{});
    multiply(std::integral_constant<int, 3>{});

    // a lane holds column l32 of each block, register r its row 8 (r / 4) + 4 half + r % 4
    const int64_t mw = m0 + wm * TM * 32, nw = n0 + wn * TN * 32;
    float b[TN];
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int64_t col = nw + j * 32 + l32;
        b[j] = p.bias ? p.bias[col < p.n ? col : p.n - 1] : 0.0f;
    }
    const int64_t lane_y = 4 * half * p.ldy + l32;
    const auto store = [&](auto whole) {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int64_t row = mw + i * 32 + 8 * (r >> 2) + (r & 3);
                TO* at = static_cast<TO*>(p.y) + row * p.ldy + nw;
#pragma unroll
                for (int j = 0; j < TN; j++)
                    if (decltype(whole)::value || (row + 4 * half < p.m && nw + j * 32 + l32 < p.n))
                        at[lane_y + j * 32] = from_f32<TO>(acc[i][j][r] + b[j]);
            }
    };
    if (m0 + BM <= p.m && n0 + BN <= p.n) store(std::true_type{});
    else store(std::false_type{});
}

template <int TM, int TN>
static int launch_tile(Ctx* c, const Product& p) {
    const int64_t tm = ceil_div(p.m, 64 * TM), tn = ceil_div(p.n, 64 * TN);
    if (tm * tn >= (1ll << 31)) return set_error(TKV_HIP_UNSUPPORTED, "matmul_mxfp4: 2^31 tiles and more");
    const dim3 grid = wide_grid(tm * tn);
    if (p.y_type == TKV_HIP_F32) k_mx_tile<TM, TN, float><<<grid, 256, 0, c->stream>>>(p, (int)tm, (int)tn);
    else if (p.y_type == TKV_HIP_F16) k_mx_tile<TM, TN, _Float16><<<grid, 256, 0, c->stream>>>(p, (int)tm, (int)tn);
    else k_mx_tile<TM, TN, __bf16><<<grid, 256, 0, c->stream>>>(p, (int)tm, (int)tn);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

}  // namespace mx

int launch_mx_product(Ctx* c, const mx::Product& p) {
    const auto tiles = [&](int64_t bm, int64_t bn) { return ceil_div(p.m, bm) * ceil_div(p.n, bn); };
    if (tiles(256, 256) >= c->num_cus) return mx::launch_tile<4, 4>(c, p);
    if (tiles(128, 128) >= c->num_cus) return mx::launch_tile<2, 2>(c, p);
    return mx::launch_tile<1, 1>(c, p);
}

}  // namespace tkv
