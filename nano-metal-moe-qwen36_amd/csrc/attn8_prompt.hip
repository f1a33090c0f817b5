/*
 * attn8_prompt.hip -- attention of prompts, or pieces of them, over a paged
 * cache in 8 bits (nmoe_attn8_prompt).
 */
#include "nmoe_attn8.h"

extern "C" size_t nmoe_attn8_prompt_workspace(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, int q_heads, int nseq,
                                              int ntok, int max_q, int max_len) {
    return 0;
}

extern "C" int nmoe_attn8_prompt(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const void *q, int q_dtype, int q_heads,
                                 int nseq, const int32_t *cu_q, int ntok, const int32_t *seq_lens, const int32_t *page_table,
                                 int max_pages, int max_q, int max_len, int causal, float scale, void *out, float *lse,
                                 void *ws, size_t ws_bytes, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_attn8_check(ctx, cache, "prompt", q, q_dtype, q_heads, nseq, seq_lens, page_table, max_pages, scale, out, lse);
    if (rc != NMOE_HIP_OK) return rc;
    if (cu_q == NULL || !nmoe_aligned(cu_q, 4) || ntok < 0 || ntok > NMOE_MAX_ROWS || max_q < 0 || max_len < 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: cu_q, 0 <= ntok <= 2^22, max_q >= 0 and max_len >= 0 are required");
    if (nseq == 0 || ntok == 0) return NMOE_HIP_OK;
    nmoe_on_device here(ctx);
    nmoe_attn8_rows(nmoe_stream_of(ctx, stream), *cache, q, q_dtype, q_heads, nseq, cu_q, ntok, seq_lens, page_table, max_pages,
                    causal, scale, out, lse);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
