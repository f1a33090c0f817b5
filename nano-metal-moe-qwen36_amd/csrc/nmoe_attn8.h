/*
 * nmoe_attn8.h -- what decode and prompt attention over a cache in 8 bits
 * (attn8_decode.hip, attn8_prompt.hip) share: the checks of their arguments.
 */
#ifndef NMOE_ATTN8_H
#define NMOE_ATTN8_H

#include "nmoe_kv8.h"

/* attn8_decode.hip; `what` opens the message. */
int nmoe_attn8_check_heads(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const char *what, int q_heads, int nseq);
int nmoe_attn8_check(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const char *what, const void *q, int q_dtype,
                     int q_heads, int nseq, const int32_t *seq_lens, const int32_t *page_table, int max_pages, float scale,
                     const void *out, const float *lse);

#endif
