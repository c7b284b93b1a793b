// attn_tile.h -- attention of many query rows on the matrix units (MFMA).
//
// Softmax in one pass over the keys: per query row a running maximum m, a sum l
// and the unnormalised output O, all f32.  A workgroup of four waves takes 128
// rows of one key / value head; a row is a (token, query head of the group)
// pair, token-major, so grouped heads share every key tile and a causal tile's
// rows span few positions.  Each wave owns 32 rows, all waves share the key and
// value tiles in LDS, which global_load_lds copies a tile ahead (two buffers,
// one barrier per tile).
//
// Both products are computed transposed, so that a lane owns one query row
// (column lane & 31 of the 32 x 32 accumulators; lanes l and l + 32 share it):
//   S^T = K Q^T     A = key rows from LDS, B = the wave's queries in registers
//   O^T = V^T P^T   A = value columns, B = the weights in registers
// The maximum, the sum and the rescaling of O are then lane-local (one
// permlane32_swap joins the halves), and the accumulator layout of S^T (lane
// half h holds keys 8 i + 4 h .. + 3) is a B operand's layout up to the order
// of the keys in the contraction: the values are read in that order
// (ds_read_b64_tr_b16: four keys of one column per lane), and P never leaves
// its registers.  f32 uses the 32x32x2 product, whose two-key steps take the
// same registers as they are.
//
// Measured: 16384 f16 tokens of 16 / 4 heads of 128 in 1.20 ms, 919 TFLOP/s (a
// library product of 8192^3: 1160); 4 x 512 new tokens over 16384 cached ones, 32 /
// 8 heads, 0.63 ms, 885; f32, 4096 tokens of 12 heads of 64, 283 us, 91 (library:
// 154).  There the matrix units are busy in 50 % of the cycles and the vector units
// in 47 %, LDS in 25 % (no bank conflicts): the two waves of a SIMD rarely have one
// multiply while the other takes exponentials.  Short rows are bound by latency: a
// wave alone takes 0.9 us (heads of 64) to 1.6 us (128) for a tile of 64 keys, LDS
// reads, products and exponentials after each other, and 5 us to start and end: 8 x
// 1024 tokens of 12 heads of 64 31 us, 421 TFLOP/s.  What did not help: 64 rows
// per wave (half the LDS reads, half the waves: 16384 tokens of heads of 64 467 ->
// 515 us, 8 x 1024 30 -> 42), two teams of four waves with every other tile each (30
// -> 36), three buffers (no change: the copies are there in time), products of the
// next tile between the exponentials of this one (registers: 1.14 -> 2.36 ms).
#pragma once

#include "attn_mfma.h"

namespace tkv {
namespace attn {

// DP: head size, padded (64, 96, 128, 192, 256; f32 96 only as 128).  Keys of a
// tile: as many as two workgroups per CU have registers and LDS for, 64 where the
// maximum, the rescaling test and the barrier of a tile spread over more of them.
// NARROW: 32 keys, and three workgroups per CU (heads of 128), which pays where
// many short rows make starts and ends weigh (the rule is launch_attention's).  64
// keys -> 32, us, 32 / 8 heads:
//   prompts   64 of 64 25 -> 21, 64 of 256 116 -> 98, 300 of up to 200 102 -> 87, 12
//             of 1024 147 -> 142, 8 of 4096 1288 -> 1231; 6 of 1024 80 -> 83, one of
//             16384 1090 -> 1110
//   chunks    13 x 350 under a window of 256 57 -> 47, of 1024 121 -> 110, of 2048 213
//             -> 196; 64 x 64 over 512 68 -> 60; 64 x 100 over 1000 177 -> 179
// It loses where two workgroups per CU come out even and three do not: chunks of 16 x
// 256 over 1024 82 -> 95, over 4096 323 -> 410; 32 x 128 over 2048 179 -> 218.
template <typename T, int DP, bool NARROW>
struct TileShape {
    static constexpr int E = sizeof(T);
    static constexpr int BN = (NARROW || E == 4 || DP >= 192) ? 32 : 64;
    static constexpr int CPR = DP * E / 16;
    static constexpr int CE = 16 / E;                           // elements of a chunk
    static constexpr int TILE = BN * DP * E;                    // bytes
    static constexpr int NT = 256;
    static constexpr int N = BN * CPR / NT;                     // chunks a thread copies
    static_assert(BN * CPR % NT == 0, "chunks per thread");
    static constexpr int LDS = 4 * TILE + 4 * BN * 4;           // two buffers of K and V, scales
};

template <typename T, int DP, int KV, bool NARROW>
__global__ __launch_bounds__(256, NARROW ? 3 : (DP == 256 || (sizeof(T) == 4 && DP > 128)) ? 1 : 2)
void k_attn_tile(AttnArgs a) {
    using S = TileShape<T, DP, NARROW>;
    using V8 = typename Vec<T>::type;
    constexpr bool PAGED = KV != KV_PACKED, I8 = KV == KV_I8, F32 = sizeof(T) == 4;
    constexpr int BN = S::BN, NKB = BN / 32, NDB = DP / 32, CPR = S::CPR, N = S::N;
    constexpr float kInf = __builtin_inff();
    using C = typename std::conditional<I8, int8_t, T>::type;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* lds_ks = reinterpret_cast<float*>(lds + 4 * S::TILE);  // [2][BN] keys' and values' scales
    float* lds_vs = lds_ks + 2 * BN;

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int l31 = lane & 31, half = lane >> 5;
    // heads vary fastest: one head's tiles stay on few XCDs, whose L2 then holds
    // its keys; later tiles, the longest ones where causal, start first
    const int kvh = blockIdx.x % a.hkv;
    const int unit = a.units - 1 - (int)(blockIdx.x / a.hkv);
    int first;
    const int seq = tile_seq<PAGED, kTileRows>(a, unit, &first);
    if (seq < 0) return;
    Seq s = seq_of<PAGED>(a, seq);
    s.q0 = uniform(s.q0), s.n = uniform(s.n), s.len = uniform(s.len);
    const int rows = s.n * a.g;
    const int row0 = (unit - first) * kTileRows;
    if (row0 >= rows) return;
    const int32_t* table = PAGED ? a.pages + seq * a.pages_st : nullptr;

    // positions of the workgroup's and the wave's rows, and what they see
    const int shift = s.len - s.n;
    const int last_row = min(row0 + kTileRows, rows) - 1;
    int kb = seen_begin(a, shift + (int)div_by(a.gdiv, row0));
    int ke = seen_end(a, shift + (int)div_by(a.gdiv, last_row), s.len);
    const int wrow = row0 + 32 * wave, wlast = min(wrow + 31, rows - 1);
    const bool live = wrow < rows;
    const int pos_lo = shift + (int)div_by(a.gdiv, live ? wrow : 0);
    const int pos_hi = shift + (int)div_by(a.gdiv, live ? wlast : 0);
    const int w_begin = uniform(seen_begin(a, pos_lo)), w_end = uniform(live ? seen_end(a, pos_hi, s.len) : 0);
    const int f_begin = uniform(seen_begin(a, pos_hi)), f_end = uniform(seen_end(a, pos_lo, s.len));
    // this lane's row
    const int row = wrow + l31;
    const bool mine = row < rows;
    const int tok = (int)div_by(a.gdiv, mine ? row : 0), head = kvh * a.g + (mine ? row : 0) - tok * a.g;
    const int my_begin = seen_begin(a, shift + tok), my_end = mine ? seen_end(a, shift + tok, s.len) : 0;

    // tiles of this split
    int t0 = kb / BN, t1 = ke > kb ? (ke + BN - 1) / BN : t0;
    int splits = 1;  // that have tiles
    if (a.splits > 1 && t1 > t0) {
        const int per = (t1 - t0 + a.splits - 1) / a.splits;
        splits = (t1 - t0 + per - 1) / per;
        t0 += (int)blockIdx.y * per;
        t1 = min(t0 + per, t1);
    }
    if ((int)blockIdx.y >= splits) return;
    t0 = uniform(t0), t1 = uniform(t1);
    const bool split = splits > 1;

    // queries: element order of a B operand, chunk 2 i + half of the row
    V8 q[CPR / 2];
    {
        const T* qr = static_cast<const T*>(a.q) + (int64_t)(s.q0 + tok) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
        for (int i = 0; i < CPR / 2; i++) {
            const int e = (2 * i + half) * S::CE;
            q[i] = V8{};
            if (mine && e < a.d) q[i] = *reinterpret_cast<const V8*>(qr + e);
        }
    }
    if (a.d < DP) {
        // the chunks past the head's end are never copied: zeros, as the queries there
        for (int i = tid; i < 4 * S::TILE / 16; i += 256)
            reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
        barrier();
    }

    // ---- copies: thread's chunk i is position i * 256 + tid of the tile ----
    // Addresses are a wave-uniform base per 1 KB copy and an offset per lane that
    // stays the same from tile to tile (only the sequence's last tile clamps rows
    // past its end to the last key, masked later).  Paged, a copy's rows lie in one
    // page where the page size is a multiple of them; else each lane looks one
    // key's row up and the lanes that copy its chunks get it by shuffle.
    constexpr int RPC = CPR <= 64 && 64 % CPR == 0 ? 64 / CPR : 0;  // rows of a copy, 0: not whole
    constexpr bool ALIKE = RPC > 0 && 4 * RPC % 16 == 0;  // all of a thread's chunks are swizzled alike
    constexpr int NO = ALIKE ? 1 : N;
    const bool whole = !PAGED || (!I8 && RPC > 0 && a.page.d % (RPC > 0 ? RPC : 1) == 0);
    const uint32_t row_bytes = (uint32_t)a.d * S::E;  // of a cached row
    const uint32_t k_step = PAGED ? row_bytes : (uint32_t)a.k_st * S::E;
    const uint32_t v_step = PAGED ? row_bytes : (uint32_t)a.v_st * S::E;
    uint32_t k_off[NO], v_off[NO];  // of a thread's chunks (from the copy's first row where paged)
    bool k_in[NO], v_in[NO];
#pragma unroll
    for (int i = 0; i < NO; i++) {
        const int pos = (i * 256 + tid) % CPR, r = (i * 256 + tid) / CPR;
        const int ck = pos ^ swz_k<CPR>(r), cv = pos ^ swz_v<CPR, S::E>(r);
        const int from = PAGED ? (RPC > 0 ? r % (RPC > 0 ? RPC : 1) : 0) : r;
        k_off[i] = from * k_step + ck * 16;
        v_off[i] = from * v_step + cv * 16;
        k_in[i] = ck * S::CE < a.d;
        v_in[i] = cv * S::CE < a.d;
    }
    const char* const k_head = static_cast<const char*>(a.k) + (PAGED ? 0 : (s.k0 * a.k_st + kvh * a.k_sh) * S::E);
    const char* const v_head = static_cast<const char*>(a.v) + (PAGED ? 0 : (s.k0 * a.v_st + kvh * a.v_sh) * S::E);
    int ids[PAGED ? N : 1], lane_id = 0;  // pages of the next tile's copies, or of the lane's key
    const auto copy_first = [&](int t, int i) { return min(t * BN + (i * 4 + wave) * RPC, s.len - 1); };
    const auto find_pages = [&](int t) {
        if constexpr (PAGED) {
            if (whole) {
#pragma unroll
                for (int i = 0; i < N; i++) ids[i] = load_uniform(table + div_by(a.page, copy_first(t, i)));
            } else {
                lane_id = table[div_by(a.page, min(t * BN + (lane & (BN - 1)), s.len - 1))];
            }
        }
    };
    // pool row of the lane's key of tile t, whose page find_pages(t) has looked up
    const auto lane_row = [&](int t) {
        const uint32_t j = min(t * BN + (lane & (BN - 1)), s.len - 1), pg = div_by(a.page, j);
        const uint32_t id = lane_id < a.pool_pages && lane_id >= 0 ? lane_id : 0;
        return (id * (uint32_t)a.hkv + kvh) * a.page.d + (j - pg * a.page.d);
    };
    constexpr int NR = I8 ? BN * (DP / 8) / 256 : 1;  // 8 codes per thread and trip
    uint2 kc[NR], vc[NR];
    float sc = 0.0f;
    const auto copy_tile = [&](int t, int buf) {
        if constexpr (!I8) {
            const unsigned dst0 = lds_at(lds) + buf * 2 * S::TILE + wave * 1024;
            const bool last = (t + 1) * BN > s.len;
            if (PAGED && !whole) {
                const uint32_t my_row = lane_row(t);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int pos = (i * 256 + tid) % CPR, r = (i * 256 + tid) / CPR;
                    const int ck = pos ^ swz_k<CPR>(r), cv = pos ^ swz_v<CPR, S::E>(r);
                    const int64_t at = (int64_t)(uint32_t)__shfl((int)my_row, r) * row_bytes;
                    const unsigned dst = uniform(dst0 + i * 4096);
                    if (ck * S::CE < a.d) copy16_to_lds(k_head + at + ck * 16, dst);
                    if (cv * S::CE < a.d) copy16_to_lds(v_head + at + cv * 16, dst + S::TILE);
                }
                return;
            }
            const char *kt = k_head, *vt = v_head;
            if constexpr (!PAGED) {
                kt += (int64_t)t * BN * k_step;
                vt += (int64_t)t * BN * v_step;
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int o = ALIKE ? 0 : i;
                const char *kr = kt, *vr = vt;
                int rows_in;  // rows of the copy (or tile) that the sequence has
                if constexpr (PAGED) {
                    const int j = copy_first(t, i);
                    const uint32_t slot = j - div_by(a.page, j) * a.page.d;
                    const uint32_t id = ids[i] < a.pool_pages && ids[i] >= 0 ? ids[i] : 0;
                    const int64_t at = (int64_t)((id * (uint32_t)a.hkv + kvh) * a.page.d + slot) * row_bytes;
                    kr += at;
                    vr += at;
                    rows_in = s.len - j;
                } else {
                    if (ALIKE) {
                        kr += (int64_t)(i * 4 * RPC) * k_step;
                        vr += (int64_t)(i * 4 * RPC) * v_step;
                    }
                    rows_in = s.len - t * BN - (ALIKE ? i * 4 * RPC : 0);
                }
                uint32_t ko = k_off[o], vo = v_off[o];
                if (last) {
                    // rows past the end: back to the last one, wherever it lies
                    const int r = PAGED ? (RPC > 0 ? lane / CPR : 0)
                                        : ((ALIKE ? 0 : i * 256) + tid) / CPR;
                    const int past = max(r - (rows_in - 1), 0);
                    if constexpr (PAGED) {
                        ko -= past * k_step;
                        vo -= past * v_step;
                    } else {
                        const int64_t back_k = (int64_t)past * k_step, back_v = (int64_t)past * v_step;
                        if (k_in[o]) copy16_to_lds(kr + ko - back_k, uniform(dst0 + i * 4096));
                        if (v_in[o]) copy16_to_lds(vr + vo - back_v, uniform(dst0 + i * 4096) + S::TILE);
                        continue;
                    }
                }
                const unsigned dst = uniform(dst0 + i * 4096);
                if (k_in[o]) copy16_to_lds(uniform(kr), ko, dst);
                if (v_in[o]) copy16_to_lds(uniform(vr), vo, dst + S::TILE);
            }
        } else {
            // codes through registers: converted on their way to LDS, below
            const uint32_t my_row = lane_row(t);
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const int x = i * 256 + tid, e = 8 * (x % (DP / 8));
                const int64_t at = (int64_t)(uint32_t)__shfl((int)my_row, x / (DP / 8)) * a.d + e;
                kc[i] = vc[i] = uint2{0, 0};
                if (e < a.d) {
                    kc[i] = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.k) + at);
                    vc[i] = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.v) + at);
                }
            }
            if (tid < 2 * BN) sc = (tid < BN ? a.ks : a.vs)[my_row];
        }
    };
    const auto put_codes = [&](int buf) {
        if constexpr (I8) {
            char* base = lds + buf * 2 * S::TILE;
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const int x = i * 256 + tid, r = x / (DP / 8), e = 8 * (x % (DP / 8));
                const auto put = [&](char* to, uint2 w, int swz) {
#pragma unroll
                    for (int h = 0; h < 8 / S::CE; h++) {
                        V8 y;
#pragma unroll
                        for (int j = 0; j < S::CE; j++) {
                            const int at = h * S::CE + j;
                            y[j] = (T)(float)(int8_t)((at < 4 ? w.x : w.y) >> (8 * (at & 3)));
                        }
                        *reinterpret_cast<V8*>(to + r * (CPR * 16) + (((e / S::CE + h) ^ swz) << 4)) = y;
                    }
                };
                put(base, kc[i], swz_k<CPR>(r));
                put(base + S::TILE, vc[i], swz_v<CPR, S::E>(r));
            }
            if (tid < 2 * BN) (tid < BN ? lds_ks : lds_vs)[buf * BN + (tid & (BN - 1))] = sc;
        }
    };

    f32x16 o[NDB];
#pragma unroll
    for (int b = 0; b < NDB; b++) o[b] = f32x16{};
    float m = -kInf, l = 0.0f;
    constexpr bool SCALED = I8 && std::is_same<T, _Float16>::value;
    constexpr float LIFT = kLift<T, SCALED>;
    float vexp = SCALED ? 0.0f : 1.0f, wtop = 0.0f;  // SCALED: O is in units of vexp (product_unit)

    // LDS offsets of this lane's reads
    const int k_row = l31 * (CPR * 16), k_swz = swz_k<CPR>(l31);
    const int vr = half * 4 + ((lane & 15) >> 2);
    const int v_swz = swz_v<CPR, S::E>(vr);
    const int v_col = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);  // chunk of the lane's column block

    if (t0 < t1) {
        find_pages(t0);
        copy_tile(t0, 0);
        put_codes(0);
        if (t0 + 1 < t1) find_pages(t0 + 1);
    }
    for (int t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1;
        if constexpr (!I8) wait_vm();
        barrier();  // tile t is in LDS, and nobody reads the other buffer any more
        if (t + 1 < t1) {
            copy_tile(t + 1, buf ^ 1);
            if (t + 2 < t1) find_pages(t + 2);
        }
        const int j0 = t * BN;
        if (j0 < w_end && j0 + BN > w_begin) {
            const char* kt = lds + buf * 2 * S::TILE;
            const char* vt = kt + S::TILE;
            f32x16 x[NKB];
#pragma unroll
            for (int b = 0; b < NKB; b++) {
                x[b] = f32x16{};
#pragma unroll
                for (int i = 0; i < CPR / 2; i++) {
                    const V8 k = *reinterpret_cast<const V8*>(kt + b * 32 * (CPR * 16) + k_row +
                                                              (((2 * i + half) ^ k_swz) << 4));
                    if constexpr (F32) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            x[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[j], q[i][j], x[b], 0, 0, 0);
                    } else {
                        x[b] = mfma32(k, q[i], x[b]);
                    }
                }
            }
            const bool full = j0 >= f_begin && j0 + BN <= f_end;
            float vs[I8 ? NKB * 16 : 1];
            if constexpr (I8) {
#pragma unroll
                for (int b = 0; b < NKB; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int key = b * 32 + 8 * i + 4 * half;
                        const f32x4 ks4 = *reinterpret_cast<const f32x4*>(lds_ks + buf * BN + key);
                        const f32x4 vs4 = *reinterpret_cast<const f32x4*>(lds_vs + buf * BN + key);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            x[b][4 * i + j] *= ks4[j];
                            vs[b * 16 + 4 * i + j] = vs4[j];
                        }
                    }
            }
            if (!full) {
                // what this lane's row sees: keys [lo, hi) counted from the lane's first
                const int lo = my_begin - j0 - 4 * half, hi = my_end - j0 - 4 * half;
#pragma unroll
                for (int b = 0; b < NKB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int j = b * 32 + (e & 3) + 8 * (e >> 2);
                        const bool seen = j >= lo && j < hi;
                        x[b][e] = seen ? x[b][e] : -kInf;
                        if constexpr (I8) vs[b * 16 + e] = seen ? vs[b * 16 + e] : 0.0f;
                    }
            }
            float mx = -kInf;
#pragma unroll
            for (int b = 0; b < NKB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, x[b][e]);
            mx = fmaxf(mx, other_half(mx)) * a.scale_log2;
            // O and l are rescaled only once the maximum has grown by 2^8: the
            // weights stay below that (f16: times 2^kLift), inside every type's range, and most
            // tiles skip 4 * DP multiplications per row
            if (__any(mx > m + 8.0f || (m == -kInf && mx > -kInf))) {
                const float mn = fmaxf(m, mx);
                const float fix = mn == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= fix;
                if constexpr (SCALED) wtop *= fix;
#pragma unroll
                for (int b = 0; b < NDB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[b][e] *= fix;
            }
            const float base = m == -kInf ? 0.0f : m - LIFT;
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < NKB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    x[b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b][e], a.scale_log2, -base));
                    sum += x[b][e];
                }
            l += sum;
            if constexpr (I8) {
#pragma unroll
                for (int b = 0; b < NKB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) x[b][e] *= vs[b * 16 + e];
                if constexpr (SCALED) {
                    float top = 0.0f;
#pragma unroll
                    for (int b = 0; b < NKB; b++)
#pragma unroll
                        for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(x[b][e]));
                    wtop = fmaxf(wtop, fmaxf(top, other_half(top)));
                    const float unit = product_unit(vexp, wtop);
                    if (__any(unit != vexp)) {
                        const float fix = vexp * inverse_unit(unit);
#pragma unroll
                        for (int b = 0; b < NDB; b++)
#pragma unroll
                            for (int e = 0; e < 16; e++) o[b][e] *= fix;
                    }
                    // (of unit: taken from vexp, the compiler multiplied in both branches,
                    // and tiles of heads of 128 spilled 45 registers)
                    vexp = unit;
                    const float inv = inverse_unit(unit);
#pragma unroll
                    for (int b = 0; b < NKB; b++)
#pragma unroll
                        for (int e = 0; e < 16; e++) x[b][e] *= inv;
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int key = (e & 3) + 8 * (e >> 2) + 4 * half;
                    const char* row_at = vt + key * (CPR * 16);
                    const int swz = swz_v<CPR, 4>(key);
#pragma unroll
                    for (int b = 0; b < NDB; b++) {
                        const int col = b * 32 + l31;
                        const float v = *reinterpret_cast<const float*>(
                            row_at + (((col >> 2) ^ swz) << 4) + ((col & 3) << 2));
                        o[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, x[0][e], o[b], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int st = 0; st < BN / 16; st++) {
                    V8 p;
#pragma unroll
                    for (int j = 0; j < 8; j++) p[j] = (T)x[st >> 1][(st & 1) * 8 + j];
#pragma unroll
                    for (int b = 0; b < NDB; b++) {
                        const char* at = vt + (st * 16 + vr) * (CPR * 16) + (((b * 4 + v_col) ^ v_swz) << 4) +
                                         ((lane & 1) << 3);
                        typedef __attribute__((address_space(3))) s16x4* lds4;
                        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
                        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * (CPR * 16)));
                        typedef short s16x8 __attribute__((ext_vector_type(8)));
                        const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                        o[b] = mfma32(__builtin_bit_cast(V8, v), p, o[b]);
                    }
                }
            }
        }
        if (t + 1 < t1) put_codes(buf ^ 1);
    }
    l += other_half(l);
    m -= LIFT;

    // A value that no row of a wave's tile may see still meets a weight of zero
    // in the product; where that left something that is not finite, those rows
    // are computed again, key by key.  Rows that see such values end up the same.
    bool bad = !(fabsf(l) < kInf);
#pragma unroll
    for (int b = 0; b < NDB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) bad |= !(fabsf(o[b][e] * vexp) < kInf);
    const unsigned long long ball = __ballot(bad && mine);
    unsigned again = uniform((unsigned)ball | (unsigned)(ball >> 32));

    // a split's sums, in this kernel's register layout
    const auto sum_of = [&](int i) {
        return reinterpret_cast<u64*>(a.sums + ((int64_t)i * gridDim.x + blockIdx.x) * a.sum_bytes);
    };
    const auto put_sums = [&](u64* sum) __attribute__((always_inline)) {
        if (half == 0) put_sum(sum + wave * 32 + l31, m, l);
#pragma unroll
        for (int b = 0; b < NDB; b++)
#pragma unroll
            for (int e = 0; e < 16; e += 2)
                put_sum(sum + kTileRows + (b * 8 + e / 2) * 256 + tid, o[b][e] * vexp, o[b][e + 1] * vexp);
    };
    u64* const mine_sum = split ? sum_of(blockIdx.y) : nullptr;
    if (split && !((again >> l31) & 1)) put_sums(mine_sum);
    for (unsigned todo = again; todo; todo &= todo - 1) {
        const int i = __builtin_ctz(todo);
        const int r = wrow + i, tk = (int)div_by(a.gdiv, (uint32_t)r), h = kvh * a.g + r - tk * a.g;
        const int64_t t_at = s.q0 + tk;
        const T* qr = static_cast<const T*>(a.q) + t_at * a.q_st + (int64_t)h * a.q_sh;
        float mm, ll, acc[4];
        attend_row<T, C, PAGED>(a, s, table, kvh, qr, max(seen_begin(a, shift + tk), t0 * BN),
                                min(seen_end(a, shift + tk, s.len), t1 * BN), &mm, &ll, acc);
        if (!split) {
            put_row<T>(a, t_at, h, ll, acc);
            continue;
        }
        if (lane == 0) put_sum(mine_sum + wave * 32 + i, mm, ll);
        for (int x4 = 0; x4 < 4; x4++) {
            const int x = lane + 64 * x4, y = x & 31;  // register 4 (y / 8) + y % 4 of lane half y / 4 % 2
            if (x >= DP) continue;
            const float v = x < a.d ? acc[x4] : 0.0f, next = __shfl_down(v, 1);
            if (!(x & 1))
                put_sum(mine_sum + kTileRows + ((x >> 5) * 8 + 2 * (y >> 3) + ((y & 3) >> 1)) * 256 + wave * 64 +
                            32 * ((y >> 2) & 1) + i,
                        v, next);
        }
    }
    if (split) {
        // the unit's last workgroup joins its splits, in their order:
        //   O = sum_s 2^(m_s - m) O_s,  l = sum_s 2^(m_s - m) l_s
        // Above kJoin of them the last workgroup of each kJoin joins those first.
        unsigned* const counter = a.arrivals + blockIdx.x * (1 + kJoin);
        const int group = blockIdx.y / kJoin;
        bool top = splits <= kJoin;
        int from = top ? 0 : group * kJoin, n = top ? splits : min(kJoin, splits - from);
        for (;;) {
            unsigned* const count = counter + (top ? 0 : 1 + group);
            if (!arrive_last(count, n)) return;
            arrive_clear(count, n);
            m = -kInf, l = 0.0f, vexp = 1.0f;
            for (int k = 0; k < n; k++) {
                const u64* sum = sum_of(from + k);
                const float2 ml = get_sum(sum + wave * 32 + l31);
                float2 y[NDB * 8];
#pragma unroll
                for (int e = 0; e < NDB * 8; e++) y[e] = get_sum(sum + kTileRows + e * 256 + tid);
                const float mn = fmaxf(m, ml.x), base = mn == -kInf ? 0.0f : mn;
                const float fix = __builtin_amdgcn_exp2f(m - base), w = __builtin_amdgcn_exp2f(ml.x - base);
                m = mn;
                l = l * fix + ml.y * w;
#pragma unroll
                for (int b = 0; b < NDB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float v = e & 1 ? y[b * 8 + e / 2].y : y[b * 8 + e / 2].x;
                        // a sum that nothing was added to may follow one that is not finite
                        o[b][e] = (k == 0 ? 0.0f : o[b][e] * fix) + (w == 0.0f ? 0.0f : v * w);
                    }
            }
            if (top) break;
            put_sums(sum_of(a.splits + group));
            top = true;
            from = a.splits;
            n = (splits + kJoin - 1) / kJoin;
        }
        again = 0;
    }

    if (!mine || ((again >> l31) & 1)) return;
    const int64_t t_at = s.q0 + tok;
    const float scale = (l == 0.0f ? 1.0f : 1.0f / l) * vexp;
#pragma unroll
    for (int b = 0; b < NDB; b++) {
        if (F32 || a.out_f32) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = b * 32 + 8 * i + 4 * half;
                const f32x4 y = {o[b][4 * i] * scale, o[b][4 * i + 1] * scale, o[b][4 * i + 2] * scale,
                                 o[b][4 * i + 3] * scale};
                if (e < a.d) put_out4<float>(a, t_at, head, e, y);
            }
        } else if constexpr (!F32) {
            // halves exchange groups of four: 8 elements, 16 bytes, per store
            T* out = static_cast<T*>(a.out) + t_at * a.o_st + (int64_t)head * a.o_sh;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                T y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = (T)(o[b][8 * i + j] * scale);
                uint2 lo, hi;
                __builtin_memcpy(&lo, y, 8);
                __builtin_memcpy(&hi, y + 4, 8);
                const auto sx = __builtin_amdgcn_permlane32_swap(lo.x, hi.x, false, false);
                const auto sy = __builtin_amdgcn_permlane32_swap(lo.y, hi.y, false, false);
                const int e = b * 32 + 16 * i + 8 * half;
                if (e < a.d) *reinterpret_cast<u32x4*>(out + e) = u32x4{sx[0], sy[0], sx[1], sy[1]};
            }
        }
    }
}

template <typename T, int DP, int KV, bool NARROW = false>
int launch_tile_dp(Ctx* c, const AttnArgs& a) {
    using S = TileShape<T, DP, NARROW>;
    static_assert(S::LDS <= 163840, "LDS of a workgroup");
    if ((size_t)S::LDS > c->max_lds) return set_error(TKV_HIP_UNSUPPORTED, "attention: not enough LDS");
    const int64_t blocks = (int64_t)a.units * a.hkv;
    k_attn_tile<T, DP, KV, NARROW>
        <<<dim3((unsigned)blocks, (unsigned)a.splits), 256, S::LDS, c->stream>>>(a);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

template <typename T, int KV>
int launch_tile_kv(Ctx* c, const AttnArgs& a) {
    if (a.d <= 64) return launch_tile_dp<T, 64, KV>(c, a);
    if constexpr (sizeof(T) == 2)
        if (a.d <= 96) return launch_tile_dp<T, 96, KV>(c, a);
    if constexpr (sizeof(T) == 2 && KV != KV_I8)
        if (a.d <= 128 && a.narrow) return launch_tile_dp<T, 128, KV, true>(c, a);
    if (a.d <= 128) return launch_tile_dp<T, 128, KV>(c, a);
    if (a.d <= 192) return launch_tile_dp<T, 192, KV>(c, a);
    return launch_tile_dp<T, 256, KV>(c, a);
}

template <typename T>
int launch_tile(Ctx* c, const AttnArgs& a, bool i8) {
    if (!a.pages) return launch_tile_kv<T, KV_PACKED>(c, a);
    return i8 ? launch_tile_kv<T, KV_I8>(c, a) : launch_tile_kv<T, KV_PAGED>(c, a);
}

}  // namespace attn
}  // namespace tkv
