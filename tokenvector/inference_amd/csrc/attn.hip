// attn.hip -- entry points of the attention operators: argument checks and the
// choice of kernel.
#include <algorithm>
#include <cmath>
#include <string>

#include "attn.h"

namespace tkv {

static int check_attention(const char* who, int32_t type, int32_t type_out, int64_t tokens,
                           int64_t heads_q, int64_t heads_kv, int64_t head_dim, int64_t sequences,
                           const tkv_hip_rows* q, const tkv_hip_rows* out, float scale,
                           int64_t window) {
    const std::string w(who);
    if (!float_type(type) || (type_out != type && type_out != TKV_HIP_F32))
        return set_error(TKV_HIP_BAD_ARG, w + ": type is F32, F16 or BF16, type_out the same or F32");
    if (tokens < 0 || tokens >= (1ll << 31) || sequences < 0 || sequences >= (1ll << 31) ||
        heads_q <= 0 || heads_kv <= 0 || heads_q > 65535 || head_dim <= 0 || head_dim > 256)
        return set_error(TKV_HIP_BAD_ARG, w + ": sizes out of range (head_dim 1 .. 256)");
    if (heads_q % heads_kv)
        return set_error(TKV_HIP_BAD_ARG, w + ": heads_q is not a multiple of heads_kv");
    if (window < 0) return set_error(TKV_HIP_BAD_ARG, w + ": negative window");
    if (!(scale >= 0.0f) || !std::isfinite(scale))
        return set_error(TKV_HIP_BAD_ARG, w + ": scale is negative or not finite");
    if (!q || !out || (tokens > 0 && (!q->data || !out->data)))
        return set_error(TKV_HIP_BAD_ARG, w + ": NULL rows");
    return TKV_HIP_OK;
}

static void common_args(AttnArgs* a, int32_t type, int32_t type_out, int64_t tokens, int64_t heads_q,
                        int64_t heads_kv, int64_t head_dim, int64_t sequences,
                        const tkv_hip_rows* q, const tkv_hip_rows* out, float scale,
                        int32_t causal, int64_t window) {
    a->q = q->data;
    a->q_st = q->stride_token;
    a->q_sh = q->stride_head;
    a->out = out->data;
    a->o_st = out->stride_token;
    a->o_sh = out->stride_head;
    a->tokens = tokens;
    a->seqs = (int32_t)sequences;
    a->hq = (int32_t)heads_q;
    a->hkv = (int32_t)heads_kv;
    a->g = (int32_t)(heads_q / heads_kv);
    a->d = (int32_t)head_dim;
    a->causal = causal != 0;
    a->window = window;
    // a scale of zero (equal weights) as f32's least, 2^-149, so that hidden logits of
    // -inf stay -inf: it makes less than 2^-21 of the largest f32 product.  And
    // finite, so that logits of zero stay zero
    a->scale_log2 = (float)std::min(std::max((double)scale * 1.4426950408889634, 0x1p-149), 3.4028234e38);
    a->out_f32 = type_out == TKV_HIP_F32;
}

static bool rows_of_16(const void* p, int64_t st, int64_t sh, int64_t bytes) {
    return aligned(p, 16) && st * bytes % 16 == 0 && sh * bytes % 16 == 0;
}

// keys: the most that a sequence can have, as far as the host knows.
static int launch_attention(Ctx* c, AttnArgs a, int type, int kv_type, int64_t max_q, int64_t keys) {
    const bool i8 = kv_type == TKV_HIP_I8;
    const int64_t b = type_bytes(type), kb = type_bytes(kv_type), ob = a.out_f32 ? 4 : b;
    const int64_t chunk = i8 ? 8 : 16 / b;
    if (a.d % chunk || !rows_of_16(a.q, a.q_st, a.q_sh, b) || !rows_of_16(a.out, a.o_st, a.o_sh, ob) ||
        !rows_of_16(a.k, a.k_st, a.k_sh, kb) || !rows_of_16(a.v, a.v_st, a.v_sh, kb) ||
        std::min(a.k_st, a.v_st) < 0 || std::max(a.k_st, a.v_st) >= (1ll << 22))
        return launch_attn_any(c, a, type, kv_type);
    a.gdiv = fast_div((uint32_t)a.g);
    // row numbers, rounded up to units of 128 and to the 64 sequences that are looked at
    // together, in 32 bits
    if (a.tokens * a.g > (1ll << 31) - (1 << 14))
        return set_error(TKV_HIP_UNSUPPORTED, "attention: too many rows");
    // Up to 32 rows per sequence take the streaming kernel, blocks of 16 rows, a
    // unit per sequence; else units of 128 rows (see tile_seq).  Both at 4, 16 and 32
    // rows of each of 8 heads of 128, streaming / tiles, us:
    //                 32 x 4096 keys               1 x 8192
    //   bf16          99/111  102/113  113/113     13/45  21/45  34/45
    //   f32           237/369 249/441  379/480     25/75  35/76  59/75
    //   bf16 on int8  52/92   54/93    63/94       15/45  22/45  35/45
    //   f32 on int8   73/331  76/424   121/456     17/74  23/74  40/74
    // (8 x 1024, and 12 heads of 64, between them.)  The choice is the call's: one
    // sequence of more rows takes all of them to the tiles.
    const int64_t longest = a.pages ? (a.cu_q ? max_q : 1) * a.g : 0;
    const bool few = longest > 0 && longest <= 32 && !(i8 && a.d % 16);
    const int blocks16 = longest <= 16 ? 1 : 2;
    const int64_t block = few ? 16 * blocks16 : kTileRows;
    const int64_t units = few ? a.seqs : a.tokens * a.g / block + a.seqs;
    if (units * a.hkv * 256 > kGridItems) return launch_attn_any(c, a, type, kv_type);
    a.units = (int32_t)units;
    const int64_t tiles = (few ? a.seqs : std::max<int64_t>(ceil_div(a.tokens * a.g, block), a.seqs)) * a.hkv;
    // Splits over the keys: as many as fill the chip once, 128 keys (streaming) or
    // 256 (tiles) at least to each; a split of fewer costs more in the join than it
    // saves (200 tokens of 12 heads over 2200 keys in 8 splits 19.1 us, in 17 25.7).
    // f32 products take eight times as long: there 64 keys are enough as long as no
    // CU gets a second workgroup (12 heads of 64, 256 tokens 24.1 -> 14.5 us, 512
    // 28.9 -> 20.7; 768 tokens in 4 splits, 288 workgroups, 39 us, in 3 30).
    // Workgroups that fill the chip: two per CU; three with heads of 64 (2048 tokens
    // of 12 heads 26.6 -> 23.7 us, f32 127 -> 86; in four 95); four f32 ones with
    // larger heads, which even out (2048 tokens of 32 heads of 128: 376 -> 331 us).
    // Streaming, up to eight times as many splits where each still has 512 KB to
    // read, so that caches of different lengths even out: a workgroup's start and
    // end take as long as reading about 100 KB.
    const int64_t slots = (few ? 2 : a.d <= 64 ? 3 : type == TKV_HIP_F32 ? 4 : 2) * c->num_cus;
    int64_t want = keys / (few ? 128 : 256);
    if (!few && type == TKV_HIP_F32) want = std::max(want, std::min<int64_t>(keys / 64, c->num_cus / tiles));
    want = std::min(want, slots / tiles);
    if (few)
        want = std::max(want, std::min<int64_t>(8 * slots / tiles, keys * 2 * a.d * kb / (512 << 10)));
    a.splits = (int32_t)std::min<int64_t>(std::max<int64_t>(want, 1), kMaxSplits);
    // many short rows (measured at TileShape): clearly over two workgroups per CU, up
    // to 4096 keys each as far as the host knows
    int64_t per_row = a.pages ? keys : a.tokens_k / a.seqs;
    if (a.window > 0) per_row = std::min(per_row, a.window + kTileRows);
    a.narrow = 10 * tiles > 23 * c->num_cus && per_row <= 4096;
    if (units * a.hkv * (1 + kJoin) > kAttnCounters) a.splits = 1;
    a.arrivals = c->attn_arrivals;
    if (a.splits > 1) {
        const int64_t groups = a.splits > kJoin ? ceil_div(a.splits, kJoin) : 0;
        // (m, l) and O of a workgroup's rows
        a.sum_bytes = block * (8 + 4 * padded_head(a.d, type == TKV_HIP_F32));
        void* ws;
        const int rc = ctx_workspace(c, 16, (size_t)(units * a.hkv * (a.splits + groups) * a.sum_bytes), &ws);
        if (no_room(rc)) {
            a.splits = 1;
        } else {
            TKV_RC_TRY(rc);
            a.sums = static_cast<char*>(ws);
        }
    }
    if (few)
        TKV_RC_TRY(type == TKV_HIP_F32   ? launch_attn_few_f32(c, a, i8, blocks16)
                   : type == TKV_HIP_F16 ? launch_attn_few_f16(c, a, i8, blocks16)
                                         : launch_attn_few_bf16(c, a, i8, blocks16));
    else
        TKV_RC_TRY(type == TKV_HIP_F32   ? launch_attn_tile_f32(c, a, i8)
                   : type == TKV_HIP_F16 ? launch_attn_tile_f16(c, a, i8)
                                         : launch_attn_tile_bf16(c, a, i8));
    return TKV_HIP_OK;
}

}  // namespace tkv

using namespace tkv;

extern "C" {

int32_t tkv_hip_dev_attention_prompt(int64_t ctx, int32_t type, int64_t tokens, int64_t tokens_k,
                                     int64_t heads_q, int64_t heads_kv, int64_t head_dim,
                                     int64_t sequences, const tkv_hip_rows* q,
                                     const tkv_hip_rows* k, const tkv_hip_rows* v,
                                     const tkv_hip_rows* out, int32_t type_out,
                                     const int32_t* cu_q, const int32_t* cu_k, float scale,
                                     int32_t causal, int64_t window) {
    TKV_RC_TRY(check_attention("attention_prompt", type, type_out, tokens, heads_q, heads_kv,
                               head_dim, sequences, q, out, scale, window));
    if (tokens_k < 0 || tokens_k > kMaxKeys || !k || !v || (tokens_k > 0 && (!k->data || !v->data)) ||
        (sequences > 0 && !cu_q))
        return set_error(TKV_HIP_BAD_ARG, "attention_prompt: bad keys, values or cu_q");
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    if (tokens == 0 || sequences == 0) return TKV_HIP_OK;
    AttnArgs a = {};
    common_args(&a, type, type_out, tokens, heads_q, heads_kv, head_dim, sequences, q, out, scale,
                causal, window);
    a.k = k->data;
    a.k_st = k->stride_token;
    a.k_sh = k->stride_head;
    a.v = v->data;
    a.v_st = v->stride_token;
    a.v_sh = v->stride_head;
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.tokens_k = tokens_k;
    a.page = fast_div(1);
    return launch_attention(c, a, type, type, tokens, tokens_k);
}

int32_t tkv_hip_dev_attention_paged(int64_t ctx, int32_t type, int64_t tokens, int64_t heads_q,
                                    int64_t cache, int64_t sequences, const tkv_hip_rows* q,
                                    const tkv_hip_rows* out, int32_t type_out,
                                    const int32_t* page_table, int64_t table_stride,
                                    const int32_t* cu_q, const int32_t* kv_lens, int64_t max_q,
                                    int64_t max_kv, float scale, int32_t causal, int64_t window) {
    const KvCache* kv = reinterpret_cast<const KvCache*>(cache);
    if (!kv) return set_error(TKV_HIP_BAD_ARG, "attention_paged: NULL cache");
    TKV_RC_TRY(check_attention("attention_paged", type, type_out, tokens, heads_q, kv->heads, kv->d,
                               sequences, q, out, scale, window));
    if (kv->type != type && kv->type != TKV_HIP_I8)
        return set_error(TKV_HIP_BAD_ARG, "attention_paged: the cache's type is neither type nor I8");
    if (table_stride < 0 || table_stride >= (1ll << 31) || max_q < 0 || max_kv < 0 ||
        (sequences > 0 && (!kv_lens || (table_stride > 0 && !page_table))))
        return set_error(TKV_HIP_BAD_ARG, "attention_paged: bad page table, lengths or bounds");
    if (!cu_q && tokens != sequences)
        return set_error(TKV_HIP_BAD_ARG, "attention_paged: without cu_q each sequence has one token");
    Ctx* c;
    TKV_RC_TRY(ctx_get(ctx, &c));
    if (kv->device != c->device)
        return set_error(TKV_HIP_BAD_ARG, "attention_paged: the cache is on another device");
    if (tokens == 0 || sequences == 0) return TKV_HIP_OK;
    AttnArgs a = {};
    common_args(&a, type, type_out, tokens, heads_q, kv->heads, kv->d, sequences, q, out, scale,
                causal, window);
    a.k = kv->k;
    a.v = kv->v;
    a.ks = kv->ks;
    a.vs = kv->vs;
    // a table without entries still tells the kernels that keys are paged; it
    // is not read, since it leaves no lengths
    a.pages = page_table ? page_table : kv_lens;
    a.pages_st = table_stride;
    a.pool_pages = kv->pages;
    a.page = fast_div((uint32_t)kv->page);
    a.cu_q = cu_q;
    a.kv_lens = kv_lens;
    const int64_t held = table_stride * kv->page;
    return launch_attention(c, a, type, kv->type, std::min(max_q, tokens), max_kv ? std::min(max_kv, held) : held);
}

}  // extern "C"
