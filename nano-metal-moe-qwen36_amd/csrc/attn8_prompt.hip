/*
 * attn8_prompt.hip -- attention of prompts, or pieces of them, over a paged
 * cache in 8 bits (nmoe_attn8_prompt).
 */
#include "nmoe_attn8.h"

template <typename T, int D>
__global__ void __launch_bounds__(256)
    nmoe_attn8_rows_kernel(nmoe_hip_kv8_cache cache, const T *q, int q_heads, int nseq, const int32_t *cu_q, int ntok,
                           const int32_t *seq_lens, const int32_t *page_table, int max_pages, int causal, float scale, T *out,
                           float *lse) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x % 64;
    const int64_t unit = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const int t = (int)(unit / q_heads), h = (int)(unit % q_heads);
    if (t >= ntok) return;
    int b = t, first = t, nq = 1;
    if (cu_q != NULL) {
        for (b = 0; b < nseq; b++) {
            first = min(max(cu_q[b], 0), ntok);
            nq = min(max(cu_q[b + 1], first), ntok) - first;
            if (t >= first && t < first + nq) break;
        }
        if (b == nseq) return;
    }
    const int len = nmoe_kv8_len(seq_lens[b], max_pages, cache.page_size);
    const int see = causal ? min(max(t - first + 1 + max(len, 0) - nq, 0), max(len, 0)) : max(len, 0);
    const int64_t row = (int64_t)t * q_heads + h;
    const int kh = h / (q_heads / cache.kv_heads);
    float x[E], o[E], m = -3.402823466e38f, l = 0.0f;
    bool bad = len < 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        x[e] = nmoe_elem<T>::get(q[row * D + lane * E + e]);
        o[e] = 0.0f;
    }
    for (int j = 0; j < see; j++) {
        int page = page_table[(int64_t)b * max_pages + j / cache.page_size];
        if ((uint32_t)page >= (uint32_t)cache.num_pages) {
            bad = true;
            page = 0;
        }
        const int place = j % cache.page_size;
        const int64_t at = page * cache.page_stride + place * cache.token_stride + kh * cache.head_stride + lane * E;
        const int64_t sc = nmoe_kv8_scale_at(cache, page, place, kh);
        const float ks = cache.k_scale[sc], vs = cache.v_scale[sc];
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) s += x[e] * (ks * __builtin_amdgcn_cvt_f32_fp8(((const uint8_t *)cache.k)[at + e], 0));
        s = nmoe_wave_sum_tree(s) * scale;
        const float mn = fmaxf(m, s), a = nmoe_exp2(m - mn), p = nmoe_exp2(s - mn);
        m = mn;
        l = l * a + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * a + p * (vs * __builtin_amdgcn_cvt_f32_fp8(((const uint8_t *)cache.v)[at + e], 0));
    }
    if (bad) l = NAN;
#pragma unroll
    for (int e = 0; e < E; e++)
        out[row * D + lane * E + e] = nmoe_elem<T>::put(see == 0 && !bad ? 0.0f : o[e] / l);
    if (lse != NULL && lane == 0) lse[row] = see == 0 && !bad ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
}

template <typename T>
static void nmoe_attn8_rows_as(hipStream_t s, const nmoe_hip_kv8_cache &c, const void *q, int q_heads, int nseq, const int32_t *cu,
                               int ntok, const int32_t *lens, const int32_t *table, int max_pages, int causal, float scale,
                               void *out, float *lse) {
    const dim3 g((uint32_t)(((int64_t)ntok * q_heads + 3) / 4));
    scale *= 1.44269504088896341f;
    if (c.head_dim == 64)
        hipLaunchKernelGGL((nmoe_attn8_rows_kernel<T, 64>), g, dim3(256), 0, s, c, (const T *)q, q_heads, nseq, cu, ntok, lens,
                           table, max_pages, causal, scale, (T *)out, lse);
    else if (c.head_dim == 128)
        hipLaunchKernelGGL((nmoe_attn8_rows_kernel<T, 128>), g, dim3(256), 0, s, c, (const T *)q, q_heads, nseq, cu, ntok, lens,
                           table, max_pages, causal, scale, (T *)out, lse);
    else
        hipLaunchKernelGGL((nmoe_attn8_rows_kernel<T, 256>), g, dim3(256), 0, s, c, (const T *)q, q_heads, nseq, cu, ntok, lens,
                           table, max_pages, causal, scale, (T *)out, lse);
}

static void nmoe_attn8_rows(hipStream_t s, const nmoe_hip_kv8_cache &c, const void *q, int q_dtype, int q_heads, int nseq,
                     const int32_t *cu, int ntok, const int32_t *lens, const int32_t *table, int max_pages, int causal,
                     float scale, void *out, float *lse) {
    if (q_dtype == NMOE_HIP_BF16)
        nmoe_attn8_rows_as<nmoe_bf16>(s, c, q, q_heads, nseq, cu, ntok, lens, table, max_pages, causal, scale, out, lse);
    else
        nmoe_attn8_rows_as<_Float16>(s, c, q, q_heads, nseq, cu, ntok, lens, table, max_pages, causal, scale, out, lse);
}

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
