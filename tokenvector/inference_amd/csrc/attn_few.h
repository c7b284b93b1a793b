// attn_few.h -- attention of few query rows over a paged cache: decoding, and
// chunks of up to 32 (token, query head of the group) rows.  HBM bound: the
// cache's bytes, read once for all heads of a group.
//
// Each wave streams tiles of its own, without barriers: K and V rows are copied
// to the wave's part of LDS (global_load_lds, two buffers), page ids two tiles
// further ahead (four small buffers), so that between one and two tiles per
// wave, 64 to 128 KB per CU, are always on their way.  Tiles are small, so that
// two workgroups fit a CU and one's start and end run beside the other's stream.
// Every vector memory operation of the loop is such a copy, so the waits count
// them exactly.
//
// The products are transposed as in the 128-row kernel, with 16 x 16
// accumulators: a lane owns query row lane & 15 of each block of 16 rows, and
// its group g = lane >> 4 holds keys 16 b + 4 g .. + 3 of key block b, which is
// again the weights' layout as a B operand.
//
// int8 caches are copied as codes, and converting them would take more of the
// vector unit than everything else (64 sequences of 8000 keys at most: 153 us).
// So the keys' codes are multiplied as they are, on the INT8 matrix units, with
// the queries split into digits of base 256: q = u (d0 + 256 d1 + 65536 d2), u the
// power of two that gives the row's largest element 22 bits and a sign (f32 rows:
// four digits, 30 bits).  bf16 and f16 elements down to 2^-14 and 2^-11 of the
// largest are exact; smaller ones are off by 2^-23 of it at most, as a sum in f32
// would be.  The digits' sums are exact in INT32, and three roundings join them.
// The values' codes are converted after a byte transpose read; the keys' scales
// multiply the logits, the values' scales the weights.
//
// At the end the workgroup's waves are joined through LDS, in order, and the
// splits of the keys over workgroups by the unit's last workgroup, in order.
//
// Measured: 32 sequences of up to 32768 keys, 8 heads of 128, bf16: 355 us, 5.45
// TB/s; 64 of up to 8000, int8: 133 us, 4.4 TB/s; one token over 1000 keys of 12
// heads of 64: 7.1 us, most of it launch, first loads and join.
#pragma once

#include "attn_mfma.h"

namespace tkv {
namespace attn {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Value rows of one transposed read: 16-bit, 8 rows x 32 bytes per half wave;
// f32, rows 4 apart x 64 bytes; int8, 16 rows x 16 bytes per half wave.
template <int CPR, int E>
__device__ __forceinline__ int swz_few_v(int row) {
    if constexpr (E == 4) return ((row >> 2) & 3) << 2;
    else if constexpr (E == 2) {
        if constexpr (CPR % 16 == 0) return (row & 7) << 1;
        else if constexpr (CPR % 8 == 0) return ((row >> 1) & 3) << 1;
        else return ((row >> 2) & 1) << 1;
    } else {
        if constexpr (CPR % 16 == 0) return (row & 7) | ((row >> 4) & 1) << 3;
        else if constexpr (CPR % 8 == 0) return ((row >> 1) & 3) | ((row >> 4) & 1) << 2;
        else if constexpr (CPR % 4 == 0) return ((row >> 2) & 1) | ((row >> 4) & 1) << 1;
        else return (row >> 2) & 1;
    }
}

template <typename T, int DP, bool I8>
struct FewShape {
    static constexpr int E = I8 ? 1 : sizeof(T);             // bytes of a cached element
    // keys of a tile: 4 to 8 KB of K and of V (f32 to 16 KB)
    static constexpr int BN = E == 4 ? 16 : (DP <= 96 ? 64 : 32) / E;
    static constexpr int TILE = BN * DP * E;                 // bytes, K or V
    static constexpr int CPR = DP * E / 16;
    static constexpr int IDS = 4 * 256;
    static constexpr int WAVE = 4 * TILE + IDS + (I8 ? 2 * 512 : 0);
    // as many waves, up to four, as let two workgroups share a CU's LDS.  (Three and
    // four waves also need 256 registers at most: with 32 rows over int8, heads of 96
    // and 192, and f32 queries of heads of 64, are 10 to 92 above, one workgroup per CU.)
    static constexpr int FIT = 80 * 1024 / WAVE;
    static constexpr int NW = FIT < 1 ? 1 : FIT > 4 ? 4 : FIT;
    static constexpr int COPIES = 2 * TILE / 1024 + (I8 ? 2 : 0);  // memory operations of a tile
};

template <typename T, int DP, bool I8, int NB>
__global__ __launch_bounds__((64 * FewShape<T, DP, I8>::NW)) void k_attn_few(AttnArgs a) {
    using S = FewShape<T, DP, I8>;
    using V8 = typename Vec<T>::type;
    using C = typename std::conditional<I8, int8_t, T>::type;
    constexpr bool F32 = sizeof(T) == 4, SCALED = I8 && std::is_same<T, _Float16>::value;
    constexpr float LIFT = kLift<T, SCALED>;
    constexpr int BN = S::BN, CPR = S::CPR, NW = S::NW, ROWS = 16 * NB;
    constexpr int CE = Vec<T>::N, QC = DP / (4 * CE);  // 16-byte chunks of a lane's query
    constexpr int NKB = BN / 16, NDB = DP / 16;
    // int8: the queries in digits, 24 bits from a row's largest element on (f32: 32)
    constexpr int STEPS = (DP + 63) / 64, DIGITS = F32 ? 4 : 3;
    constexpr float kInf = __builtin_inff();
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float2 row_ml[NW][ROWS];
    __shared__ int row_bad[ROWS];

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int l15 = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.hkv, seq = blockIdx.x / a.hkv;
    Seq s = seq_of<true>(a, seq);
    s.q0 = uniform(s.q0), s.n = uniform(s.n), s.len = uniform(s.len);
    const int rows = s.n * a.g;
    const int32_t* table = a.pages + seq * a.pages_st;
    const int shift = s.len - s.n;
    char* mem = lds + wave * S::WAVE;
    int* ids = reinterpret_cast<int*>(mem + 4 * S::TILE);
    float* scales = reinterpret_cast<float*>(mem + 4 * S::TILE + S::IDS);  // [2][K, V][64]

    if (rows == 0) return;
    // A sequence of more rows than the caller's max_q said is still right, if
    // slow: its first split's workgroup takes those past the block key by key.
    if (rows > ROWS && blockIdx.y == 0) {
        for (int row = ROWS + wave; row < rows; row += NW) {
            const int tok = (int)div_by(a.gdiv, (uint32_t)row), h = kvh * a.g + row - tok * a.g;
            const T* qr = static_cast<const T*>(a.q) + (int64_t)(s.q0 + tok) * a.q_st + (int64_t)h * a.q_sh;
            float mm, ll, acc[4];
            attend_row<T, C, true>(a, s, table, kvh, qr, seen_begin(a, shift + tok),
                                   seen_end(a, shift + tok, s.len), &mm, &ll, acc);
            put_row<T>(a, s.q0 + tok, h, ll, acc);
        }
    }
    const int pos_lo = shift;
    const int pos_hi = shift + (int)div_by(a.gdiv, min(ROWS, rows) - 1);
    const int kb = seen_begin(a, pos_lo), ke = seen_end(a, pos_hi, s.len);
    const int f_begin = uniform(seen_begin(a, pos_hi)), f_end = uniform(seen_end(a, pos_lo, s.len));
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

    if (tid < ROWS) row_bad[tid] = 0;
    if (a.d < DP) {
        // the chunks past the head's end are never copied: zeros, as the queries there
        for (int i = lane; i < 4 * S::TILE / 16; i += 64)
            reinterpret_cast<u32x4*>(mem)[i] = u32x4{0, 0, 0, 0};
        wait_lds();
    }

    const int count = t1 - t0 > wave ? (t1 - t0 - wave + NW - 1) / NW : 0;
    const auto tile = [&](int k) { return t0 + wave + k * NW; };
    const auto key_of = [&](int k) {  // this lane's key of the k-th tile; past the end the last one, masked
        return min(min(tile(k), t1 - 1) * BN + (lane & (BN - 1)), s.len - 1);
    };
    const auto copy_ids = [&](int k) {
        copy4_to_lds(table + div_by(a.page, (uint32_t)key_of(k)), uniform(lds_at(ids + 64 * (k & 3))));
    };
    const auto copy_tile = [&](int k) {
        // pool row of this lane's key, handed to the lanes that copy its chunks
        const uint32_t j = (uint32_t)key_of(k), pg = div_by(a.page, j);
        uint32_t id = (uint32_t)ids[64 * (k & 3) + lane];
        id = (int64_t)id < a.pool_pages ? id : 0;
        const uint32_t my_row = (id * (uint32_t)a.hkv + kvh) * a.page.d + (j - pg * a.page.d);
        const unsigned dst = uniform(lds_at(mem) + (k & 1) * 2 * S::TILE);
        const int64_t row_bytes = (int64_t)a.d * S::E;
#pragma unroll
        for (int i = 0; i < S::TILE / 1024; i++) {
            const int r = (i * 64 + lane) / CPR, c = (i * 64 + lane) % CPR;
            const int64_t at = (int64_t)(uint32_t)__shfl((int)my_row, r) * row_bytes;
            const int ck = c ^ swz_k<CPR>(r), cv = c ^ swz_few_v<CPR, S::E>(r);
            if (ck * 16 < row_bytes) copy16_to_lds(static_cast<const char*>(a.k) + at + ck * 16, dst + i * 1024);
            if (cv * 16 < row_bytes)
                copy16_to_lds(static_cast<const char*>(a.v) + at + cv * 16, dst + S::TILE + i * 1024);
        }
        if constexpr (I8) {
            const unsigned to = uniform(lds_at(scales + 128 * (k & 1)));
            copy4_to_lds(a.ks + my_row, to);
            copy4_to_lds(a.vs + my_row, to + 256);
        }
    };

    if (count > 0) {
        copy_ids(0);
        copy_ids(1);
    }
    const auto join_max = [](float x) {  // over the four key groups of a row
        x = fmaxf(x, other_row(x));
        return fmaxf(x, other_half(x));
    };
    // queries, B operand: row l15, chunk 4 i + g (int8: 16 elements from 64 i + 16 g on)
    constexpr int QN = I8 ? STEPS * (16 / CE) : QC;
    V8 q[NB][QN];
    int my_begin[NB], my_end[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int row = 16 * b + l15;
        const bool mine = row < rows;
        const int tok = (int)div_by(a.gdiv, mine ? row : 0), h = kvh * a.g + (mine ? row : 0) - tok * a.g;
        const T* qr = static_cast<const T*>(a.q) + (int64_t)(s.q0 + tok) * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int e = I8 ? 64 * (i / (16 / CE)) + 16 * g + i % (16 / CE) * CE : (4 * i + g) * CE;
            q[b][i] = V8{};
            if (mine && e < a.d) q[b][i] = *reinterpret_cast<const V8*>(qr + e);
        }
        my_begin[b] = seen_begin(a, shift + tok);
        my_end[b] = mine ? seen_end(a, shift + tok, s.len) : 0;
    }
    if (count > 0) {
        wait_vm();
        copy_tile(0);
        copy_ids(2);
        if (count > 1) copy_tile(1);
        copy_ids(3);
    }
    // int8: the elements in units of the row's largest power of two /
    // 2^(8 DIGITS - 2), in digits of base 256 from -128 to 127
    i32x4 qd[I8 ? NB : 1][I8 ? STEPS : 1][DIGITS];
    float qunit[NB];  // of the lowest digit
    if constexpr (I8) {
#pragma unroll
        for (int b = 0; b < NB; b++) {
            // NaN where the row is not finite: so are then its logits
            float top = 0.0f, sick = 0.0f;
#pragma unroll
            for (int i = 0; i < QN; i++)
#pragma unroll
                for (int k = 0; k < CE; k++) {
                    const float x = fabsf(to_f32(q[b][i][k]));
                    top = fmaxf(top, x);
                    sick = x < kInf ? sick : 1.0f;
                }
            top = join_max(top);
            const bool finite = join_max(sick) == 0.0f;
            const int e2 = finite && top > 0.0f ? ilogbf(top) + 1 : 0;  // |x| < 2^e2
            qunit[b] = finite ? __builtin_ldexpf(1.0f, e2 - (8 * DIGITS - 2)) : __builtin_nanf("");
#pragma unroll
            for (int i = 0; i < STEPS; i++)
#pragma unroll
                for (int j4 = 0; j4 < 4; j4++) {
                    // v + 0x80 in every byte: its bytes are the digits + 128
                    unsigned v[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int at = 4 * j4 + k;
                        const float x = to_f32(q[b][i * (16 / CE) + at / CE][at % CE]);
                        const float y = __builtin_rintf(__builtin_ldexpf(x, 8 * DIGITS - 2 - e2));
                        v[k] = (unsigned)(finite ? (int)y : 0) + 0x80808080u;
                    }
#pragma unroll
                    for (int n = 0; n < DIGITS; n++) {
                        const unsigned at = n | (4 + n) << 8;  // bytes n of two words
                        const unsigned lo = __builtin_amdgcn_perm(v[1], v[0], at | 0x0c0c0000u);
                        const unsigned hi = __builtin_amdgcn_perm(v[3], v[2], at << 16 | 0x0c0cu);
                        qd[b][i][n][j4] = (int)((lo | hi) ^ 0x80808080u);
                    }
                }
        }
    }

    f32x4 o[NB][NDB];
    float m[NB], l[NB], vexp[NB], wtop[NB];  // SCALED: O is in units of vexp (product_unit)
#pragma unroll
    for (int b = 0; b < NB; b++) {
        m[b] = -kInf, l[b] = 0.0f, vexp[b] = SCALED ? 0.0f : 1.0f, wtop[b] = 0.0f;
#pragma unroll
        for (int n = 0; n < NDB; n++) o[b][n] = f32x4{};
    }
    const int k_swz = swz_k<CPR>(l15);  // rows 16 apart are swizzled alike
    // value rows of a transposed read: 4 g + i of a block (and + 16)
    const int v_row16 = 4 * g + (l15 >> 2), v_row8 = (l15 >> 1) < 4 ? 4 * g + (l15 >> 1) : 12 + 4 * g + (l15 >> 1);

    for (int k = 0; k < count; k++) {
        if (k + 1 < count) wait_vm_but<S::COPIES + 1>();  // all but the next tile and its ids' successor
        else wait_vm();
        const int j0 = tile(k) * BN;
        const char* kt = mem + (k & 1) * 2 * S::TILE;
        const char* vt = kt + S::TILE;
        const float* sk = scales + 128 * (k & 1);
        f32x4 x[NB][NKB];
#pragma unroll
        for (int b = 0; b < NKB; b++) {
            const char* kr = kt + (b * 16 + l15) * (CPR * 16);
            if constexpr (I8) {
                // the codes as they are against the queries' digits: exact sums, one
                // rounding when they are joined (a chunk past the row's end meets
                // digits of zero)
                i32x4 sum[NB][DIGITS];
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int k = 0; k < DIGITS; k++) sum[n][k] = i32x4{};
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    const i32x4 kf = *reinterpret_cast<const i32x4*>(kr + (((4 * i + g) ^ k_swz) << 4));
#pragma unroll
                    for (int n = 0; n < NB; n++)
#pragma unroll
                        for (int k = 0; k < DIGITS; k++)
                            sum[n][k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qd[n][i][k], sum[n][k], 0, 0, 0);
                }
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float y = (float)sum[n][DIGITS - 1][j];
#pragma unroll
                        for (int k = DIGITS - 2; k >= 0; k--) y = __builtin_fmaf(y, 256.0f, (float)sum[n][k][j]);
                        x[n][b][j] = y;
                    }
            } else {
#pragma unroll
                for (int n = 0; n < NB; n++) x[n][b] = f32x4{};
#pragma unroll
                for (int i = 0; i < QC; i++) {
                    const V8 kf = *reinterpret_cast<const V8*>(kr + (((4 * i + g) ^ k_swz) << 4));
#pragma unroll
                    for (int n = 0; n < NB; n++) {
                        if constexpr (F32) {
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                x[n][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], q[n][i][j], x[n][b], 0, 0, 0);
                        } else {
                            x[n][b] = mfma16(kf, q[n][i], x[n][b]);
                        }
                    }
                }
            }
        }
        const bool full = j0 >= f_begin && j0 + BN <= f_end;
#pragma unroll
        for (int n = 0; n < NB; n++) {
            float vs[I8 ? BN / 4 : 1];
            float mx = -kInf;
#pragma unroll
            for (int b = 0; b < NKB; b++) {
                if constexpr (I8) {
                    const f32x4 ks4 = *reinterpret_cast<const f32x4*>(sk + b * 16 + 4 * g);
                    const f32x4 vs4 = *reinterpret_cast<const f32x4*>(sk + 64 + b * 16 + 4 * g);
                    x[n][b] *= ks4 * qunit[n];
#pragma unroll
                    for (int j = 0; j < 4; j++) vs[b * 4 + j] = vs4[j];
                }
                if (!full) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int key = j0 + b * 16 + 4 * g + j;
                        const bool seen = key >= my_begin[n] && key < my_end[n];
                        x[n][b][j] = seen ? x[n][b][j] : -kInf;
                        if constexpr (I8) vs[b * 4 + j] = seen ? vs[b * 4 + j] : 0.0f;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) mx = fmaxf(mx, x[n][b][j]);
            }
            mx = join_max(mx) * a.scale_log2;
            // rescaled only once the maximum has grown by 2^8, as in the 128-row kernel
            if (__any(mx > m[n] + 8.0f || (m[n] == -kInf && mx > -kInf))) {
                const float mn = fmaxf(m[n], mx);
                const float fix = mn == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m[n] - mn);
                m[n] = mn;
                l[n] *= fix;
                if constexpr (SCALED) wtop[n] *= fix;
#pragma unroll
                for (int d = 0; d < NDB; d++) o[n][d] *= fix;
            }
            const float base = m[n] == -kInf ? 0.0f : m[n] - LIFT;
#pragma unroll
            for (int b = 0; b < NKB; b++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[n][b][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[n][b][j], a.scale_log2, -base));
                    l[n] += x[n][b][j];
                }
            if constexpr (I8) {
#pragma unroll
                for (int b = 0; b < NKB; b++)
#pragma unroll
                    for (int j = 0; j < 4; j++) x[n][b][j] *= vs[b * 4 + j];
                if constexpr (SCALED) {
                    float top = 0.0f;
#pragma unroll
                    for (int b = 0; b < NKB; b++)
#pragma unroll
                        for (int j = 0; j < 4; j++) top = fmaxf(top, fabsf(x[n][b][j]));
                    wtop[n] = fmaxf(wtop[n], join_max(top));
                    const float unit = product_unit(vexp[n], wtop[n]);
                    if (__any(unit != vexp[n])) {
                        const float fix = vexp[n] * inverse_unit(unit);
#pragma unroll
                        for (int d = 0; d < NDB; d++) o[n][d] *= fix;
                    }
                    vexp[n] = unit;
                    const float inv = inverse_unit(unit);
#pragma unroll
                    for (int b = 0; b < NKB; b++)
#pragma unroll
                        for (int j = 0; j < 4; j++) x[n][b][j] *= inv;
                }
            }
        }
        // values: steps of 32 keys (blocks 2 st and 2 st + 1) or of 16
        constexpr int STEP = NKB == 1 ? 1 : 2;
#pragma unroll
        for (int st = 0; st < NKB / STEP; st++) {
            typedef T P __attribute__((ext_vector_type(4 * STEP)));
            P p[NB];
            if constexpr (!F32) {
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int j = 0; j < 4 * STEP; j++) p[n][j] = (T)x[n][STEP * st + (j >> 2)][j & 3];
            }
#pragma unroll
            for (int d = 0; d < NDB; d++) {
                if constexpr (I8) {
                    const int r = st * 32 + v_row8;
                    const char* at = vt + r * (CPR * 16) + ((d ^ swz_few_v<CPR, 1>(v_row8)) << 4) + ((lane & 1) << 3);
                    typedef __attribute__((address_space(3))) i32x2* lds2;
                    const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds2)at);
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) y[j] = (float)(int8_t)(w[j >> 2] >> (8 * (j & 3)));
                    if constexpr (F32) {
#pragma unroll
                        for (int n = 0; n < NB; n++)
#pragma unroll
                            for (int j = 0; j < 8; j++)
                                o[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    y[j], x[n][2 * st + (j >> 2)][j & 3], o[n][d], 0, 0, 0);
                    } else {
                        V8 v;
#pragma unroll
                        for (int j = 0; j < 8; j++) v[j] = (T)y[j];
#pragma unroll
                        for (int n = 0; n < NB; n++) o[n][d] = mfma16(v, p[n], o[n][d]);
                    }
                } else if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        static_assert(STEP == 1 || !F32 || I8, "f32 tiles are one block");
                        const int r = st * 16 + 4 * g + j, col = d * 16 + l15;
                        const float v = *reinterpret_cast<const float*>(
                            vt + r * (CPR * 16) + (((col >> 2) ^ swz_few_v<CPR, 4>(4 * g)) << 4) + ((col & 3) << 2));
#pragma unroll
                        for (int n = 0; n < NB; n++)
                            o[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[n][st][j], o[n][d], 0, 0, 0);
                    }
                } else {
                    const int c = d * 2 + ((l15 & 3) >> 1);
                    const char* at = vt + (st * 16 * STEP + v_row16) * (CPR * 16) +
                                     ((c ^ swz_few_v<CPR, 2>(v_row16)) << 4) + ((lane & 1) << 3);
                    typedef __attribute__((address_space(3))) s16x4* lds4;
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
                    if constexpr (STEP == 1) {
#pragma unroll
                        for (int n = 0; n < NB; n++) o[n][d] = mfma16(__builtin_bit_cast(P, lo), p[n], o[n][d]);
                        continue;
                    }
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 16 * (CPR * 16)));
                    typedef short s16x8 __attribute__((ext_vector_type(8)));
                    const V8 v = __builtin_bit_cast(V8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                    if constexpr (STEP == 2) {
#pragma unroll
                        for (int n = 0; n < NB; n++) o[n][d] = mfma16(v, p[n], o[n][d]);
                    }
                }
            }
        }
        wait_lds();  // this tile is read: its buffer is free
        if (k + 2 < count) copy_tile(k + 2);
        copy_ids(k + 4);
    }
    wait_vm();

    // the waves' sums, joined in their order: rows of DP f32 per wave in LDS
    barrier();
    float* sums = reinterpret_cast<float*>(lds) + wave * ROWS * DP;
#pragma unroll
    for (int n = 0; n < NB; n++) {
        l[n] += other_row(l[n]);
        l[n] += other_half(l[n]);
        // what a masked key's values left behind: such rows are computed again,
        // as in the 128-row kernel
        bool bad = !(fabsf(l[n]) < kInf);
#pragma unroll
        for (int d = 0; d < NDB; d++) {
#pragma unroll
            for (int j = 0; j < 4; j++) bad |= !(fabsf(o[n][d][j] * vexp[n]) < kInf);
            *reinterpret_cast<f32x4*>(sums + (n * 16 + l15) * DP + d * 16 + 4 * g) = o[n][d] * vexp[n];
        }
        if (bad) row_bad[n * 16 + l15] = 1;
        if (g == 0) row_ml[wave][n * 16 + l15] = make_float2(m[n] - LIFT, l[n]);
    }
    barrier();
    const bool split = splits > 1;
    // sums of a split: (m, l) of the rows, then two planes of 8 bytes per four elements
    constexpr int QUADS = ROWS * (DP / 4);
    const auto sum_of = [&](int i) {
        return reinterpret_cast<u64*>(a.sums + ((int64_t)i * gridDim.x + blockIdx.x) * a.sum_bytes);
    };
    const auto put_quad = [&](u64* sum, int i, f32x4 y) {
        put_sum(sum + ROWS + i, y[0], y[1]);
        put_sum(sum + ROWS + QUADS + i, y[2], y[3]);
    };
    for (int i = tid; i < QUADS; i += 64 * NW) {
        const int r = i / (DP / 4), e = 4 * (i % (DP / 4));
        if (r >= rows || e >= a.d || row_bad[r]) continue;
        float mm = -kInf;
#pragma unroll
        for (int w = 0; w < NW; w++) mm = fmaxf(mm, row_ml[w][r].x);
        const float base = mm == -kInf ? 0.0f : mm;
        float ll = 0.0f;
        f32x4 y = {};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(row_ml[w][r].x - base);
            ll = __builtin_fmaf(f, row_ml[w][r].y, ll);
            y += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds) + (w * ROWS + r) * DP + e);
        }
        if (split) {
            u64* sum = sum_of(blockIdx.y);
            if (e == 0) put_sum(sum + r, mm, ll);
            put_quad(sum, i, y);
        } else {
            const int tok = (int)div_by(a.gdiv, (uint32_t)r), h = kvh * a.g + r - tok * a.g;
            put_out4<T>(a, s.q0 + tok, h, e, y * (ll == 0.0f ? 1.0f : 1.0f / ll));
        }
    }
    for (int r = wave; r < ROWS; r += NW) {
        if (r >= rows || !uniform(row_bad[r])) continue;
        const int tok = (int)div_by(a.gdiv, (uint32_t)r), h = kvh * a.g + r - tok * a.g;
        const int64_t t_at = s.q0 + tok;
        const T* qr = static_cast<const T*>(a.q) + t_at * a.q_st + (int64_t)h * a.q_sh;
        float mm, ll, acc[4];
        attend_row<T, C, true>(a, s, table, kvh, qr, max(seen_begin(a, shift + tok), t0 * BN),
                               min(seen_end(a, shift + tok, s.len), t1 * BN), &mm, &ll, acc);
        if (!split) {
            put_row<T>(a, t_at, h, ll, acc);
            continue;
        }
        u64* sum = sum_of(blockIdx.y);
        if (lane == 0) put_sum(sum + r, mm, ll);
        for (int x4 = 0; x4 < 4; x4++) {
            const int x = lane + 64 * x4;
            const float v = acc[x4], next = __shfl_down(v, 1);
            if (x < a.d && !(x & 1)) put_sum(sum + ROWS + (x & 2 ? QUADS : 0) + r * (DP / 4) + x / 4, v, next);
        }
    }
    if (!split) return;

    // The unit's last workgroup joins its splits, in their order,
    //   O = sum_s 2^(m_s - m) O_s,  l = sum_s 2^(m_s - m) l_s;
    // above kJoin of them the last workgroup of each kJoin joins those first, so
    // that none reads more than kJoin sums per level, all of them in flight
    // together.
    const auto join = [&](auto most, int from, int n, int to) __attribute__((always_inline)) {
        constexpr int MOST = decltype(most)::value;
        for (int i = tid; i < QUADS; i += 64 * NW) {
            const int r = i / (DP / 4), e = 4 * (i % (DP / 4));
            if (r >= rows || e >= a.d) continue;
            float2 ml[MOST], lo[MOST], hi[MOST];
#pragma unroll
            for (int k = 0; k < MOST; k++) {
                const u64* sum = sum_of(from + min(k, n - 1));
                ml[k] = get_sum(sum + r);
                lo[k] = get_sum(sum + ROWS + i);
                hi[k] = get_sum(sum + ROWS + QUADS + i);
            }
            float mm = -kInf, ll = 0.0f;
#pragma unroll
            for (int k = 0; k < MOST; k++) mm = fmaxf(mm, ml[k].x);
            const float base = mm == -kInf ? 0.0f : mm;
            f32x4 y = {};
#pragma unroll
            for (int k = 0; k < MOST; k++) {
                const float w = k < n ? __builtin_amdgcn_exp2f(ml[k].x - base) : 0.0f;
                ll = __builtin_fmaf(w, ml[k].y, ll);
                if (w != 0.0f) y += w * f32x4{lo[k].x, lo[k].y, hi[k].x, hi[k].y};
            }
            if (to >= 0) {
                if (e == 0) put_sum(sum_of(to) + r, mm, ll);
                put_quad(sum_of(to), i, y);
            } else {
                const int tok = (int)div_by(a.gdiv, (uint32_t)r), h = kvh * a.g + r - tok * a.g;
                put_out4<T>(a, s.q0 + tok, h, e, y * (ll == 0.0f ? 1.0f : 1.0f / ll));
            }
        }
    };
    const auto join_all = [&](int from, int n, int to) __attribute__((always_inline)) {
        if (n <= 4) join(std::integral_constant<int, 4>{}, from, n, to);
        else if (n <= 8) join(std::integral_constant<int, 8>{}, from, n, to);
        else join(std::integral_constant<int, kJoin>{}, from, n, to);
    };
    unsigned* counter = a.arrivals + blockIdx.x * (1 + kJoin);
    int from = 0, n = splits;
    if (splits > kJoin) {
        const int group = blockIdx.y / kJoin, members = min(kJoin, splits - group * kJoin);
        if (!arrive_last(counter + 1 + group, members)) return;
        arrive_clear(counter + 1 + group, members);
        join_all(group * kJoin, members, a.splits + group);
        from = a.splits;
        n = (splits + kJoin - 1) / kJoin;
    }
    if (!arrive_last(counter, n)) return;
    arrive_clear(counter, n);
    join_all(from, n, -1);
}

template <typename T, int DP, bool I8>
int launch_few_dp(Ctx* c, const AttnArgs& a, int blocks_of_16) {
    using S = FewShape<T, DP, I8>;
    constexpr int LDS = S::NW * S::WAVE;
    static_assert(LDS <= 163840 - 4096 && S::NW * 32 * DP * 4 <= LDS, "LDS of a workgroup");
    if ((size_t)LDS + 4096 > c->max_lds) return set_error(TKV_HIP_UNSUPPORTED, "attention: not enough LDS");
    const int64_t blocks = (int64_t)a.units * a.hkv;
    const dim3 grid((unsigned)blocks, (unsigned)a.splits);
    if (blocks_of_16 == 1) k_attn_few<T, DP, I8, 1><<<grid, 64 * S::NW, LDS, c->stream>>>(a);
    else k_attn_few<T, DP, I8, 2><<<grid, 64 * S::NW, LDS, c->stream>>>(a);
    TKV_LAUNCH_CHECK();
    return TKV_HIP_OK;
}

template <typename T, bool I8>
int launch_few_kv(Ctx* c, const AttnArgs& a, int blocks_of_16) {
    if (a.d <= 64) return launch_few_dp<T, 64, I8>(c, a, blocks_of_16);
    if constexpr (sizeof(T) == 2)
        if (a.d <= 96) return launch_few_dp<T, 96, I8>(c, a, blocks_of_16);
    if (a.d <= 128) return launch_few_dp<T, 128, I8>(c, a, blocks_of_16);
    if (a.d <= 192) return launch_few_dp<T, 192, I8>(c, a, blocks_of_16);
    return launch_few_dp<T, 256, I8>(c, a, blocks_of_16);
}

template <typename T>
int launch_few(Ctx* c, const AttnArgs& a, bool i8, int blocks_of_16) {
    return i8 ? launch_few_kv<T, true>(c, a, blocks_of_16) : launch_few_kv<T, false>(c, a, blocks_of_16);
}

}  // namespace attn
}  // namespace tkv
