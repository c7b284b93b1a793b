// mxfp4_tile.hip -- the product of microscaled 4-bit operands,
//   y[m, n] = sum_k a[m, k] w[n, k] + bias[n],
// on v_mfma_scale_f32_32x32x64_f8f6f4.  A lane's operand is one block, 16 bytes
// of codes and its scale byte, so the block scales cost nothing in the product;
// products are exact and sums f32 (within 2^-20 of the largest term for each
// instruction).
//
// Tiles: 4 waves, each a quarter of the workgroup's BM x BN outputs.  K goes in
// slices of 256 elements, 128 bytes a row: copied HBM / L2 -> LDS by buffer loads
// into one of two stages while the other is multiplied.  Rows lie in LDS in
// 16-byte chunks whose place is XORed with the row, so that the 32 rows that a
// fragment's read takes spread over the banks; the copies are linear in LDS, so
// each lane fetches the chunk that belongs there.
//
// Order within a slice, of four steps of 64 elements: the next step's fragments
// are read between this one's products.  Before the last step the wave waits for
// its part of the next slice and for its own reads; behind the barrier the stage
// just read is free for the slice after next: half of its copies go between the
// last step's products, half between the next slice's first ones.  The wave is
// alone on its SIMD (its sums take half the registers), so what does not stand
// between two products stops them: copies and reads in one run, or a branch, past
// which the compiler moves the products, cost 2.13 us a slice instead of 1.77.
//
// What bounds it: 8192 x 8192 x 8192 in bf16 247 to 257 us, 4.3 PFLOP/s.  A slice of
// a tile alone on the card takes 1.14 us (2048 of its 2700 cycles the matrix units'),
// 1.45 at the 1.87 GHz that power leaves with all CUs at work, and then 1.77: the other
// 0.3 us is the copies' (without them 1.44).  Of random codes the matrix units alone,
// all operands in registers, reach 6.2 PFLOP/s at 1.55 GHz (10 at 2.4 GHz of zeros),
// 177 us.  (The 16x16x128 form reaches 6.9, its sums moved half as often, but took the same time
// here, with twice the scales to read.)
#include <type_traits>

#include "mxfp4.h"
#include "tkv_reduce.h"

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

// TM, TN: a wave's blocks of 32 tokens and of 32 weight rows.  ROWS: the scales come
// as [rows][blocks] (of kRowSlices slices at most), and all of the tile's are laid
// out in LDS first.
template <int TM, int TN, int STAGES, bool ROWS>
struct Tile {
    static constexpr int BM = 64 * TM, BN = 64 * TN;
    static constexpr int CODES = (BM + BN) * 128, SCALES = (BM + BN) * 8;
    static constexpr int STAGE = CODES + (ROWS ? 0 : SCALES);
    static constexpr int LDS = STAGES * STAGE + (ROWS ? kRowSlices * SCALES : 0);
    static constexpr int PER_CU = LDS * 4 <= 163840 ? 4 : LDS * 2 <= 163840 ? 2 : 1;
};

// K split over workgroups (blockIdx.z): their slices, sums [tiles][splits][256 lanes] of
// 16 f32, and an arrival count a tile.
struct Split {
    int32_t slices, splits;
    unsigned long long* sums;
    unsigned* arrivals;
};

template <int TM, int TN, int STAGES, bool ROWS, bool SPLIT, typename TO>
__global__ __launch_bounds__(256, (Tile<TM, TN, STAGES, ROWS>::PER_CU)) void k_mx_tile(Product p, int tiles_m,
                                                                                      int tiles_n, int vec,
                                                                                      Split split) {
    using T = Tile<TM, TN, STAGES, ROWS>;
    constexpr int BM = T::BM, BN = T::BN;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::LDS];
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
    // row's end the buffer's bounds turn into zeros: they are checked against the
    // vector offset alone, so the whole offset is in it and the scalar one is 0.
    // Past a row's end is the next row, which the scales 2^-127 there leave out.
    constexpr int COPIES = (BM + BN) / 32;
    const int rows_a = p.m - m0 < BM ? (int)(p.m - m0) : BM, rows_w = p.n - n0 < BN ? (int)(p.n - n0) : BN;
    const uint32_t bytes_a = (uint32_t)rows_a * row_bytes, bytes_w = (uint32_t)rows_w * row_bytes;
    const uint8_t *base_a = p.a + m0 * row_bytes, *base_w = p.w + n0 * row_bytes;
    // (a copy's first row is a multiple of 8: its part of chunk_xor is the wave's)
    const uint32_t lane_at =
        (uint32_t)(lane >> 3) * row_bytes + (uint32_t)(((lane & 7) ^ chunk_xor(wave * 8 + (lane >> 3))) * 16);
    constexpr int SBYTES = T::SCALES / 4;  // of a wave
    constexpr int SWIDTH = SBYTES % 1024 == 0 ? 16 : 4, SCOPIES = ROWS ? 0 : (SBYTES + 64 * SWIDTH - 1) / (64 * SWIDTH);
    constexpr int ITEMS = COPIES + SCOPIES;
    const int all = (p.blocks + 7) >> 3, begin = SPLIT ? (int)blockIdx.z * split.slices : 0;
    const int slices = SPLIT ? min(all, begin + split.slices) : all;  // from begin to here
    // (copies more than there are scales for copy the last again)
    const auto scale_place = [&](int d) {
        const int at = (d * 4 + wave) * 64 * SWIDTH;
        return at < T::SCALES ? at : T::SCALES - 64 * SWIDTH;
    };
    const uint8_t* scale_at[SCOPIES + 1];
    int64_t scale_step[SCOPIES + 1];
#pragma unroll
    for (int d = 0; d < SCOPIES; d++) {
        const int at = scale_place(d);
        scale_at[d] = at < BM * 8 ? p.as + m0 * 8 + at : p.ws + n0 * 8 + (at - BM * 8);
        scale_step[d] = (at < BM * 8 ? p.a_rows : p.w_rows) * 8;
    }
    // one of a wave's copies of a slice.  Of a slice that is not there only the
    // scales of the last are copied: no branch keeps the products from the copies.
    const auto copy = [&](int slice, uint8_t* stage, int d) {
        if (d < COPIES) {
            const bool is_a = d * 32 < BM;
            const int first = (d * 4 + wave) * 8, in = is_a ? first : first - BM;
            const uint32_t at = (in < (is_a ? rows_a : rows_w) ? (uint32_t)in * row_bytes : 0u) + (uint32_t)slice * 128u;
            const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(is_a ? base_a : base_w), 0, slice < slices ? (int)(is_a ? bytes_a : bytes_w) : 0, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)(stage + first * 128), 16, (int)(lane_at + at), 0, 0, 0);
        } else if constexpr (!ROWS) {
            const int k = d - COPIES, have = slice < slices ? slice : slices - 1, at = scale_place(k);
            const void* from = scale_at[k] + (int64_t)have * scale_step[k] + lane * SWIDTH;
            if constexpr (SWIDTH == 16)
                __builtin_amdgcn_global_load_lds(from, (lds_ptr)(stage + T::CODES + at), 16, 0, 0);
            else
                __builtin_amdgcn_global_load_lds(from, (lds_ptr)(stage + T::CODES + at), 4, 0, 0);
        }
    };

    v16f acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[j][i][r] = 0.0f;

    v4i fa[2][TM], fw[2][TN];
    v2i sa[TM], sw[TN];                      // a slice's scales as read,
    int la[TM], ha[TM], lw[TN], hw[TN];      // and shifted
    const int ra = wm * TM * 32 + l32, rw = BM + wn * TN * 32 + l32;
    const int x = chunk_xor(l32);
    constexpr int F = TM + TN;  // fragments of a step
    const auto read = [&](const uint8_t* stage, int step, int k) {
        const int c = ((2 * step + half) ^ x) * 16, set = step & 1;
        if (k < TN) fw[set][k] = *reinterpret_cast<const v4i*>(stage + (rw + k * 32) * 128 + c);
        else fa[set][k - TN] = *reinterpret_cast<const v4i*>(stage + (ra + (k - TN) * 32) * 128 + c);
    };
    const auto stage_of = [&](int slice) { return lds + ((unsigned)slice % STAGES) * T::STAGE; };
    const auto read_scales = [&](int slice, int k) {
        const uint8_t* at = ROWS ? lds + STAGES * T::STAGE + (slice < slices ? slice - begin : 0) * T::SCALES
                                 : stage_of(slice) + T::CODES;
        if (k < TN) sw[k] = *reinterpret_cast<const v2i*>(at + (rw + k * 32) * 8);
        else sa[k - TN] = *reinterpret_cast<const v2i*>(at + (ra + (k - TN) * 32) * 8);
    };
    // a lane's blocks are 2 step + half: shifted so, step's byte is 2 (step % 2)
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
    // the products of one step, and `n` copies and reads spread between them
    const auto multiply = [&](auto step, auto n, auto&& other) {
        constexpr int S = decltype(step)::value, N = decltype(n)::value, P = TM * TN;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < P; t++) {
            const int i = t / TN, j = t % TN;
            const v4i a4 = fa[S & 1][i], w4 = fw[S & 1][j];
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                v8i{w4.x, w4.y, w4.z, w4.w, 0, 0, 0, 0}, v8i{a4.x, a4.y, a4.z, a4.w, 0, 0, 0, 0}, acc[j][i], 4, 4,
                2 * (S & 1), S < 2 ? lw[j] : hw[j], 2 * (S & 1), S < 2 ? la[i] : ha[i]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = t * N / P; k < (t + 1) * N / P; k++) other(k);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const auto sync = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    // (a third to two thirds early: the same; all of them 5% slower)
    constexpr int EARLY = (ITEMS + 1) / 2, LATE = ITEMS - EARLY;
    // s_waitcnt vmcnt(n), leaving the other counts alone
#define TKV_MX_COPIES_LEFT(n) __builtin_amdgcn_s_waitcnt(0x0F70 | ((n) & 15) | (((n) >> 4) << 14))
    static_assert((STAGES & (STAGES - 1)) == 0 && (STAGES - 2) * ITEMS + EARLY < 64, "ring, vmcnt range");
#pragma unroll
    for (int t = 0; t < STAGES - 1; t++)
#pragma unroll
        for (int d = 0; d < ITEMS; d++) copy(begin + t, stage_of(begin + t), d);
#pragma unroll
    for (int d = 0; d < EARLY; d++) copy(begin + STAGES - 1, stage_of(begin + STAGES - 1), d);
    if constexpr (ROWS) {
        // a thread loads a part of a row's, all of its loads in flight together
        constexpr int PARTS = 256 / (BM + BN) > 0 ? 256 / (BM + BN) : 1, OWN = kRowSlices / PARTS;
        static_assert(256 % (BM + BN) == 0, "a part of a row for each thread");
        const int r = (int)threadIdx.x % (BM + BN), first = (int)threadIdx.x / (BM + BN) * OWN;
        const int64_t row = r < BM ? m0 + r : n0 + r - BM, last = (r < BM ? p.m : p.n) - 1;
        const uint8_t* from = (r < BM ? p.as : p.ws) + (row < last ? row : last) * p.blocks;
        v2i part[OWN];
#pragma unroll
        for (int h = 0; h < OWN; h++)
            part[h] = row_scales(from, begin + first + h, p.blocks);
#pragma unroll
        for (int h = 0; h < OWN; h++)
            *reinterpret_cast<v2i*>(lds + STAGES * T::STAGE + (first + h) * T::SCALES + r * 8) = part[h];
    }
    TKV_MX_COPIES_LEFT(ROWS ? 0 : (STAGES - 2) * ITEMS + EARLY);
    sync();
#pragma unroll
    for (int k = 0; k < F; k++) read_scales(begin, k);
#pragma unroll
    for (int k = 0; k < F; k++) read(stage_of(begin), 0, k);
#pragma unroll 1
    for (int s = begin; s < slices; s++) {
        uint8_t *stage = stage_of(s), *next = stage_of(s + 1), *last = stage_of(s + STAGES - 1);
        shift_scales();
        multiply(I0{}, std::integral_constant<int, F + LATE>{}, [&](int k) {
            if (k < F) read(stage, 1, k);
            else copy(s + STAGES - 1, last, EARLY + k - F);
        });
        multiply(I1{}, std::integral_constant<int, F>{}, [&](int k) { read(stage, 2, k); });
        multiply(I2{}, std::integral_constant<int, F>{}, [&](int k) { read(stage, 3, k); });
        TKV_MX_COPIES_LEFT((STAGES - 2) * ITEMS);  // this wave's of slice s + 1 are there
        sync();
        multiply(I3{}, std::integral_constant<int, 2 * F + EARLY>{}, [&](int k) {
            if (k < F) read(next, 0, k);
            else if (k < F + EARLY) copy(s + STAGES, stage, k - F);
            else read_scales(s + 1, k - F - EARLY);
        });
    }
#undef TKV_MX_COPIES_LEFT
    __builtin_amdgcn_s_waitcnt(0x0F70);

    if constexpr (SPLIT) {  // the tile's last workgroup adds the splits' sums in their order
        static_assert(TM * TN == 1, "a lane's 16 sums");
        unsigned long long* const sums = split.sums + block * split.splits * 2048 + threadIdx.x;
        const auto put = [&](int e) { return sums + ((int)blockIdx.z * 8 + e) * 256; };
#pragma unroll
        for (int e = 0; e < 8; e++)
            __hip_atomic_store(put(e),
                               (unsigned long long)__float_as_uint(acc[0][0][2 * e]) |
                                   (unsigned long long)__float_as_uint(acc[0][0][2 * e + 1]) << 32,
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        unsigned* const count = split.arrivals + block;
        if (!arrive_last(count, (unsigned)split.splits, *reinterpret_cast<int*>(lds))) return;
        arrive_clear(count, (unsigned)split.splits);
#pragma unroll
        for (int r = 0; r < 16; r++) acc[0][0][r] = 0.0f;
        for (int z0 = 0; z0 < split.splits; z0 += 4) {  // (four splits' on their way at once)
            unsigned long long two[4][8];
#pragma unroll
            for (int z = 0; z < 4; z++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int from = z0 + z < split.splits ? z0 + z : z0;
                    two[z][e] = __hip_atomic_load(sums + (from * 8 + e) * 256, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
#pragma unroll
            for (int z = 0; z < 4; z++) {
                if (z0 + z >= split.splits) break;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    acc[0][0][2 * e] += __uint_as_float((unsigned)two[z][e]);
                    acc[0][0][2 * e + 1] += __uint_as_float((unsigned)(two[z][e] >> 32));
                }
            }
        }
    }

    // A lane holds token l32 of each block, registers 4 q .. 4 q + 3 its outputs
    // 8 q + 4 half .. of 32.  They go out through LDS, 32 tokens at a time, so that a
    // store takes whole lines, and the code is a short loop: unrolled over the
    // registers it was longer to fetch than to run (a tile of 256 x 256 with edges
    // 45 us, 1024 deep).
    constexpr int ROW = TN * 32 * (int)sizeof(TO) + 16;  // bytes of a token in LDS
    static_assert(4 * 32 * ROW <= T::LDS, "the waves' parts");
    sync();  // the others may still read the last slice
    uint8_t* own = lds + wave * (32 * ROW);
    const int64_t nw = n0 + wn * TN * 32, mw = m0 + wm * TM * 32;
    float b[TN][16];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int64_t c = nw + j * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
            b[j][r] = p.bias ? p.bias[c < p.n ? c : p.n - 1] : 0.0f;
        }
    constexpr int LANES = TN * 32 * (int)sizeof(TO) / 16, STEP = 64 / LANES, E = 16 / (int)sizeof(TO);
    const int64_t n = nw + (lane % LANES) * E;
    const int64_t left = p.n - n;  // outputs from n on
    const bool whole = vec && m0 + BM <= p.m && n0 + BN <= p.n;
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                struct alignas(4 * sizeof(TO)) { TO e[4]; } v;
#pragma unroll
                for (int e = 0; e < 4; e++) v.e[e] = from_f32<TO>(acc[j][i][4 * q + e] + b[j][4 * q + e]);
                __builtin_memcpy(own + l32 * ROW + (j * 32 + 8 * q + 4 * half) * sizeof(TO), &v, sizeof(v));
            }
        __builtin_amdgcn_wave_barrier();
        if (whole) {
            v4i v[32 / STEP];
#pragma unroll
            for (int t = 0; t < 32 / STEP; t++)
                v[t] = *reinterpret_cast<const v4i*>(own + (t * STEP + lane / LANES) * ROW + (lane % LANES) * 16);
            TO* at = static_cast<TO*>(p.y) + (mw + i * 32 + lane / LANES) * p.ldy + n;
#pragma unroll
            for (int t = 0; t < 32 / STEP; t++) {
                v4i* to = reinterpret_cast<v4i*>(at + t * STEP * p.ldy);
                // past the L2's reuse, which the operands need more (8192 x 2304 of 768
                // 33.6 -> 28.8 us, 8192 x 8192 of 8192 264 -> 247); small outputs and
                // parts of lines lose by it (1000 x 12001 of 1001 21.5 -> 27.8)
                if constexpr (TM * TN > 1) __builtin_nontemporal_store(v[t], to);
                else *to = v[t];
            }
        } else {
#pragma unroll 1
            for (int t = lane / LANES; t < 32; t += STEP) {
                const int64_t m = mw + i * 32 + t;
                const v4i v = *reinterpret_cast<const v4i*>(own + t * ROW + (lane % LANES) * 16);
                TO* at = static_cast<TO*>(p.y) + m * p.ldy + n;
                if (m >= p.m || left <= 0) continue;
                if (left >= E) {
                    __builtin_memcpy(at, &v, 16);  // (of any alignment)
                } else {
                    TO e[E];
                    __builtin_memcpy(e, &v, 16);
#pragma unroll
                    for (int k = 0; k < E; k++)
                        if (k < left) at[k] = e[k];
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int TM, int TN, int STAGES, bool ROWS, bool SPLIT = false>
static int launch_tile(Ctx* c, const Product& p, int splits = 1) {
    const int64_t tm = ceil_div(p.m, 64 * TM), tn = ceil_div(p.n, 64 * TN);
    if (tm * tn >= (1ll << 31)) return set_error(TKV_HIP_UNSUPPORTED, "matmul_mxfp4: 2^31 tiles and more");
    dim3 grid = wide_grid(tm * tn);
    Split split = {};
    if (SPLIT) {
        const int64_t slices = ceil_div(p.blocks, 8);
        split.slices = (int32_t)ceil_div(slices, splits);
        split.splits = (int32_t)ceil_div(slices, split.slices);
        grid.z = (unsigned)split.splits;
        void* ws;
        TKV_RC_TRY(mx_room(c, 16, (size_t)(tm * tn * split.splits) << 14, &ws));
        split.sums = static_cast<unsigned long long*>(ws);
        split.arrivals = c->attn_arrivals;
    }
    const int m = (int)tm, n = (int)tn, vec = aligned(p.y, 16) && p.ldy * type_bytes(p.y_type) % 16 == 0;
    const auto start = [&](auto k) { k<<<grid, 256, 0, c->stream>>>(p, m, n, vec, split); };
    if (p.y_type == TKV_HIP_F32) start(k_mx_tile<TM, TN, STAGES, ROWS, SPLIT, float>);
    else if (p.y_type == TKV_HIP_F16) start(k_mx_tile<TM, TN, STAGES, ROWS, SPLIT, _Float16>);
    else start(k_mx_tile<TM, TN, STAGES, ROWS, SPLIT, __bf16>);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

}  // namespace mx

int launch_mx_product(Ctx* c, const mx::Product& p) {
    if (p.m <= mx::kFewRows) return launch_mx_few(c, p);
    const mx::TilePlan plan = mx::tile_plan(mx::shape_of(c, p));
    if (plan.splits > 1)
        return p.a_rows == 0 ? mx::launch_tile<1, 1, 4, true, true>(c, p, plan.splits)
                             : mx::launch_tile<1, 1, 4, false, true>(c, p, plan.splits);
    if (p.a_rows == 0) return mx::launch_tile<1, 1, 4, true>(c, p);
    switch (plan.kind) {
        case mx::TILE_256: return mx::launch_tile<4, 4, 2, false>(c, p);
        case mx::TILE_128: return mx::launch_tile<2, 2, 2, false>(c, p);
        case mx::TILE_128_64: return mx::launch_tile<2, 1, 2, false>(c, p);
        case mx::TILE_64: return mx::launch_tile<1, 1, 2, false>(c, p);
        default: return mx::launch_tile<1, 1, 4, false>(c, p);
    }
}

}  // namespace tkv
