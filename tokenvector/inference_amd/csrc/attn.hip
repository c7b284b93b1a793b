// attn.hip -- entry points of the attention operators: argument checks and the
// choice of kernel.
#include <string>

#include "attn.h"

namespace tkv {

static int check_attention(const char* who, int32_t type, int32_t type_out, int64_t tokens,
                           int64_t heads_q, int64_t heads_kv, int64_t head_dim, int64_t sequences,
                           const tkv_hip_rows* q, const tkv_hip_rows* out, int64_t window) {
    const std::string w(who);
    if (!float_type(type) || (type_out != type && type_out != TKV_HIP_F32))
        return set_error(TKV_HIP_BAD_ARG, w + ": type is F32, F16 or BF16, type_out the same or F32");
    if (tokens < 0 || tokens >= (1ll << 31) || sequences < 0 || sequences >= (1ll << 31) ||
        heads_q <= 0 || heads_kv <= 0 || heads_q > 65535 || head_dim <= 0 || head_dim > 256)
        return set_error(TKV_HIP_BAD_ARG, w + ": sizes out of range (head_dim 1 .. 256)");
    if (heads_q % heads_kv)
        return set_error(TKV_HIP_BAD_ARG, w + ": heads_q is not a multiple of heads_kv");
    if (window < 0) return set_error(TKV_HIP_BAD_ARG, w + ": negative window");
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
    a->scale_log2 = (float)((double)scale * 1.4426950408889634);
    a->out_f32 = type_out == TKV_HIP_F32;
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
                               head_dim, sequences, q, out, window));
    if (tokens_k < 0 || tokens_k >= (1ll << 31) || !k || !v || (tokens_k > 0 && (!k->data || !v->data)) ||
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
    return launch_attn_any(c, a, type, type);
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
                               sequences, q, out, window));
    if (kv->type != type && kv->type != TKV_HIP_I8)
        return set_error(TKV_HIP_BAD_ARG, "attention_paged: the cache's type is neither type nor I8");
    if (table_stride < 0 || max_q < 0 || max_kv < 0 ||
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
    return launch_attn_any(c, a, type, kv->type);
}

}  // extern "C"
