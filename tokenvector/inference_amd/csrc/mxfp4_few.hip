// mxfp4_few.hip -- products and linears of few rows with a 4-bit weight: the
// weight is streamed once, and its bytes are what bounds them.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 with the weight's rows as its rows and the
// tokens as its columns.  A lane's operand is a block of a row, 16 bytes and a
// scale byte, straight from memory: a row's four lanes take the chunks of a
// 128-byte line with two instructions, 256 elements.  The waves of a workgroup take
// 256-element slabs of K in turn, each for all of the workgroup's 16 NR rows, and
// their sums are added in LDS in the waves' order.  Where the row blocks leave CUs idle
// K is split over workgroups too, whose sums the last of them adds in their order.
//
// The linear's form codes the tokens on the way, every workgroup all of them (of its
// part of K), into LDS, while the first of its weights are on their way.
#include <type_traits>

#include "mxfp4.h"
#include "tkv_reduce.h"

namespace tkv {
namespace mx {

struct FewArgs {
    Product p;
    const void* x;  // the linear's rows
    int64_t stride, k;
    int32_t slabs;     // of a workgroup, at most
    FastDiv quarters;  // of those
    // split over K: the sums [row blocks][splits][tokens / 16][64 lanes] of v4f, and
    // an arrival count a row block
    int32_t splits;
    unsigned long long* sums;
    unsigned* arrivals;
};

// Bytes of a coded token in LDS, and of its scales.
__host__ __device__ __forceinline__ uint32_t coded_bytes(uint32_t blocks) { return blocks * 16u + 16u; }
__host__ __device__ __forceinline__ uint32_t scale_bytes(uint32_t blocks) { return ((blocks + 7) >> 3) * 8u; }

struct Coded {};      // the tokens come as codes and slabs,
struct CodedRows {};  // or the scales of both as [rows][blocks]

template <typename TI, int NR, int MT, int WAVES, bool SPLIT>
__global__ __launch_bounds__(WAVES * 64) void k_mx_few(FewArgs a) {
    constexpr bool ROWS = std::is_same<TI, CodedRows>::value, CODED = ROWS || std::is_same<TI, Coded>::value;
    typedef typename std::conditional<CODED, float, TI>::type TX;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Product& p = a.p;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int64_t n0 = wide_block() * (16 * NR);
    if (n0 >= p.n) return;
    const uint32_t row_bytes = (uint32_t)p.blocks * 16u;
    const int all = (p.blocks + 7) >> 3;
    const int begin = SPLIT ? (int)blockIdx.z * a.slabs : 0, slabs = SPLIT ? min(all, begin + a.slabs) : all;
    const uint32_t blocks = (uint32_t)(SPLIT ? min(p.blocks, slabs * 8) - begin * 8 : p.blocks);  // of this workgroup

    // rows past the weight's, and tokens past m, read the last one
    const uint8_t* w_row[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const int64_t row = n0 + r * 16 + l16;
        w_row[r] = p.w + (row < p.n ? row : p.n - 1) * row_bytes;
    }
    int token[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) token[t] = t * 16 + l16 < (int)p.m ? t * 16 + l16 : (int)p.m - 1;

    struct Weights {
        v4i w[NR][2];
        v2i s[NR];
    };
    struct Tokens {
        v4i t[MT][2];
        v2i s[MT];
    };
    // chunks past the row: its last, whose scales are 2^-127
    const auto place = [&](int s, int h, uint32_t bytes) {
        const uint32_t at = (uint32_t)s * 128u + (uint32_t)(h * 64 + g * 16);
        return at < bytes ? at : bytes - 16;
    };
    const auto load_weight = [&](int s, Weights& b) {
#pragma unroll
        for (int r = 0; r < NR; r++) {
#pragma unroll
            for (int h = 0; h < 2; h++) b.w[r][h] = *reinterpret_cast<const v4i*>(w_row[r] + place(s, h, row_bytes));
            if constexpr (ROWS) {
                const int64_t row = n0 + r * 16 + l16;
                b.s[r] = row_scales(p.ws + (row < p.n ? row : p.n - 1) * p.blocks, s, p.blocks);
            } else {
                b.s[r] = *reinterpret_cast<const v2i*>(p.ws + ((int64_t)s * p.w_rows + n0 + r * 16 + l16) * 8);
            }
        }
    };
    uint8_t* const scales = lds + (uint32_t)p.m * coded_bytes(blocks);  // of the tokens coded here
    const auto load_tokens = [&](int s, Tokens& b) {
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const uint8_t* row = CODED ? p.a + (uint64_t)token[t] * row_bytes : lds + (uint32_t)token[t] * coded_bytes(blocks);
#pragma unroll
            for (int h = 0; h < 2; h++)
                b.t[t][h] = *reinterpret_cast<const v4i*>(row + (CODED ? place(s, h, row_bytes) : place(s - begin, h, blocks * 16)));
            if constexpr (!CODED)
                b.s[t] = *reinterpret_cast<const v2i*>(scales + (uint32_t)token[t] * scale_bytes(blocks) + (s - begin) * 8);
            else if constexpr (ROWS)
                b.s[t] = row_scales(p.as + (int64_t)token[t] * p.blocks, s, p.blocks);
            else
                b.s[t] = *reinterpret_cast<const v2i*>(p.as + ((int64_t)s * p.a_rows + t * 16 + l16) * 8);
        }
    };

    v4f acc[NR][MT];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int t = 0; t < MT; t++) acc[r][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // a wave's next slabs on their way (four instead of two were no faster)
    constexpr int DEPTH = 2;
    Weights weights[DEPTH];
    Tokens tokens[DEPTH];
#pragma unroll
    for (int u = 0; u < DEPTH; u++)
        if (begin + wave + u * WAVES < slabs) {
            load_weight(begin + wave + u * WAVES, weights[u]);
            if constexpr (CODED) load_tokens(begin + wave + u * WAVES, tokens[u]);
        }
    if constexpr (!CODED) {
        // a thread takes one quarter of a block of every token, or of every `apart`-th
        // where the rows are short
        constexpr int THREADS = WAVES * 64;
        const int per = (int)a.quarters.d, apart = per < THREADS ? THREADS / per : 1;
        const int first = per < THREADS ? (int)div_by(a.quarters, threadIdx.x) : 0;
        const int many = first < apart ? (int)p.m : 0, quarters = (slabs - begin) * 32;
        const auto code_tokens = [&](auto ragged, auto batch) {
            constexpr bool RAGGED = decltype(ragged)::value;
            constexpr int B = decltype(batch)::value;  // tokens in flight
            for (int c = (int)threadIdx.x - first * per; c < quarters; c += THREADS) {  // (whole blocks: four lanes stay together)
                const TX* from = static_cast<const TX*>(a.x) + (int64_t)first * a.stride;
                uint8_t* to = lds + (uint32_t)first * coded_bytes(blocks) + c * 4;
                uint8_t* scale = scales + (uint32_t)first * scale_bytes(blocks) + (c >> 2);
                const int64_t step = (int64_t)apart * a.stride, at = ((int64_t)begin * 32 + c) * 8;
                const uint32_t to_step = (uint32_t)apart * coded_bytes(blocks);
                const uint32_t scale_step = (uint32_t)apart * scale_bytes(blocks);
                for (int t = first; t < many; t += B * apart) {
                    Quarter<TX> x[B];  // (of tokens past the last: the first again)
#pragma unroll
                    for (int u = 0; u < B; u++) {
                        const int v = t + u * apart < many ? u : 0;
                        x[u] = load_quarter<TX>(from + v * step, at, a.k);
                    }
                    from += B * step;
#pragma unroll
                    for (int u = 0; u < B; u++) {
                        if (t + u * apart >= many) break;
                        end_quarter<TX, RAGGED>(x[u], at, a.k);
                        unsigned byte;
                        const unsigned code = code_quarter<TX>(x[u], byte);
                        if (c < (int)blocks * 4) *reinterpret_cast<unsigned*>(to) = code;
                        if ((c & 3) == 0) *scale = (uint8_t)byte;
                        to += to_step;
                        scale += scale_step;
                    }
                }
            }
        };
        using One = std::integral_constant<int, 1>;
        using Four = std::integral_constant<int, 4>;
        if (a.k & 7) code_tokens(std::true_type{}, Four{});
        else if (p.m == 1) code_tokens(std::false_type{}, One{});
        else code_tokens(std::false_type{}, Four{});
        __syncthreads();
    }
    for (int s0 = begin + wave; s0 < slabs; s0 += DEPTH * WAVES) {
#pragma unroll
        for (int u = 0; u < DEPTH; u++) {
            const int s = s0 + u * WAVES, then = s + DEPTH * WAVES;
            if (s >= slabs) break;
            if constexpr (!CODED) load_tokens(s, tokens[u]);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const v4i w = weights[u].w[r][h];
                    const unsigned wb = (unsigned)weights[u].s[r][h] >> (8 * g);
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        const v4i x = tokens[u].t[t][h];
                        const unsigned tb = (unsigned)tokens[u].s[t][h] >> (8 * g);
                        acc[r][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                            v8i{w.x, w.y, w.z, w.w, 0, 0, 0, 0}, v8i{x.x, x.y, x.z, x.w, 0, 0, 0, 0}, acc[r][t], 4, 4,
                            0, (int)wb, 0, (int)tb);
                    }
                }
            if (then < slabs) {
                load_weight(then, weights[u]);
                if constexpr (CODED) load_tokens(then, tokens[u]);
            }
        }
    }
    if constexpr (!CODED) __syncthreads();  // the codes' place is the sums'

    // a lane holds rows 4 g .. 4 g + 3 of 16 for token l16
    v4f* part = reinterpret_cast<v4f*>(lds);  // [WAVES][NR * MT][64]
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
        for (int t = 0; t < MT; t++) part[(wave * NR * MT + r * MT + t) * 64 + lane] = acc[r][t];
    __syncthreads();
    const auto join = [&](int i) {
        v4f sum = part[i * 64 + lane];
#pragma unroll
        for (int w = 1; w < WAVES; w++) sum += part[(w * NR * MT + i) * 64 + lane];
        return sum;
    };
    // the row block's last workgroup adds the splits' sums in their order
    unsigned long long* const sums = SPLIT ? a.sums + (n0 / 16 * a.splits * MT * 64 + lane) * 2 : nullptr;
    if constexpr (SPLIT) {
        for (int i = wave; i < MT; i += WAVES) {
            const v4f sum = join(i);
            unsigned long long two[2];
            __builtin_memcpy(two, &sum, 16);
            for (int e = 0; e < 2; e++)
                __hip_atomic_store(sums + ((int)blockIdx.z * MT + i) * 128 + e, two[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        unsigned* const count = a.arrivals + n0 / 16;
        if (!arrive_last(count, (unsigned)a.splits)) return;
        arrive_clear(count, (unsigned)a.splits);
    }
    for (int i = wave; i < NR * MT; i += WAVES) {
        v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (SPLIT) {
            v4f v[kFewSplits];  // (all on their way at once)
#pragma unroll
            for (int z = 0; z < kFewSplits; z++) {
                const int have = z < a.splits ? z : 0;
                unsigned long long two[2];
#pragma unroll
                for (int e = 0; e < 2; e++)
                    two[e] = __hip_atomic_load(sums + (have * MT + i) * 128 + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __builtin_memcpy(&v[z], two, 16);
            }
#pragma unroll
            for (int z = 0; z < kFewSplits; z++)
                if (z < a.splits) sum += v[z];
        } else {
            sum = join(i);
        }
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

template <typename TI, int NR, int MT, int WAVES = 8, bool SPLIT = false>
static void start_few(Ctx* c, FewArgs& a, int64_t rows) {
    constexpr bool CODED = std::is_same<TI, Coded>::value || std::is_same<TI, CodedRows>::value;
    const int64_t slabs = ceil_div(a.p.blocks, 8);
    a.slabs = (int32_t)ceil_div(slabs, a.splits);
    a.splits = (int32_t)ceil_div(slabs, a.slabs);
    a.quarters = fast_div((uint32_t)a.slabs * 32);
    const uint32_t sums = WAVES * NR * MT * 1024;
    const uint32_t blocks = (uint32_t)(a.p.blocks < a.slabs * 8 ? a.p.blocks : a.slabs * 8);
    const uint32_t codes = CODED ? 0 : (uint32_t)a.p.m * (coded_bytes(blocks) + scale_bytes(blocks));
    dim3 grid = wide_grid(ceil_div(rows, NR));
    grid.z = (unsigned)a.splits;
    k_mx_few<TI, NR, MT, WAVES, SPLIT><<<grid, WAVES * 64, sums > codes ? sums : codes, c->stream>>>(a);
}

template <typename TI, int MT>
static int launch_few(Ctx* c, FewArgs& a) {
    constexpr bool CODED = std::is_same<TI, Coded>::value || std::is_same<TI, CodedRows>::value;
    constexpr bool WIDE = CODED || MT == 1;
    // (at most 1536 blocks a split are coded on the way, and 64 make one: 25 tokens)
    constexpr bool JOINS = CODED || MT < 4;
    const FewPlan plan = few_plan(shape_of(c, a.p), CODED);
    const int64_t rows = ceil_div(a.p.n, 16);
    a.splits = JOINS ? plan.splits : 1;
    if (a.splits > 1) {
        void* ws;
        TKV_RC_TRY(mx_room(c, 16, (size_t)(rows * a.splits * MT * 1024), &ws));
        a.sums = static_cast<unsigned long long*>(ws);
        a.arrivals = c->attn_arrivals;
        start_few<TI, 1, MT, 8, JOINS>(c, a, rows);
    } else if (plan.row_blocks == 4) {
        start_few<TI, WIDE && MT < 4 ? 4 : 1, MT>(c, a, rows);
    } else if (plan.row_blocks == 2) {
        start_few<TI, WIDE ? 2 : 1, MT>(c, a, rows);
    } else if (plan.waves == 16) {
        start_few<TI, 1, MT, WIDE && !CODED ? 16 : 8>(c, a, rows);
    } else {
        start_few<TI, 1, MT>(c, a, rows);
    }
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

template <typename T>
static int launch_few_linear(Ctx* c, FewArgs& a) {
    if (a.p.m <= 16) return launch_few<T, 1>(c, a);
    if (a.p.m <= 32) return launch_few<T, 2>(c, a);
    return launch_few<T, 4>(c, a);
}

int launch_mx_few_linear(Ctx* c, int type, const void* x, int64_t stride, int64_t k, const Product& p) {
    FewArgs a = {};
    a.p = p;
    a.x = x;
    a.stride = stride;
    a.k = k;
    if (type == TKV_HIP_F32) return launch_few_linear<float>(c, a);
    if (type == TKV_HIP_F16) return launch_few_linear<_Float16>(c, a);
    return launch_few_linear<__bf16>(c, a);
}

}  // namespace tkv
