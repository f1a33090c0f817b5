/*
 * attn_prompt.hip -- attention over whole prompts packed one behind the
 * other, causal or full, with grouped heads (nmoe_attn_prompt).
 */
#include "nmoe_context.h"

#define NMOE_PR_WAVES 4

/* A wavefront a query row and head, keys one after the other. */
template <typename T, int D>
__global__ void __launch_bounds__(64 * NMOE_PR_WAVES)
    nmoe_attn_prompt_kernel(nmoe_hip_qkv rows, int nseq, const int32_t *cu_q, const int32_t *cu_k, int ntok_q,
                            int ntok_k, int causal, float scale, T *out, float *lse) {
    constexpr int E = D / 64;
    const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x % 64, w = threadIdx.x / 64;
    const int q0 = min(max(cu_q[b], 0), ntok_q), q1 = min(max(cu_q[b + 1], q0), ntok_q);
    const int k0 = min(max(cu_k[b], 0), ntok_k), k1 = min(max(cu_k[b + 1], k0), ntok_k);
    const int nq = q1 - q0, nk = k1 - k0, kh = h / (rows.q_heads / rows.kv_heads);
    for (int64_t at = (int64_t)blockIdx.x * NMOE_PR_WAVES + w; at < nq; at += (int64_t)gridDim.x * NMOE_PR_WAVES) {
        const int i = (int)at;
        const T *q = (const T *)rows.q + (q0 + i) * rows.q_stride + h * rows.q_head_stride + E * lane;
        float x[E], o[E], m = -INFINITY, l = 0.0f;
        for (int e = 0; e < E; e++) {
            x[e] = nmoe_elem<T>::get(q[e]);
            o[e] = 0.0f;
        }
        const int see = causal ? min(i + nk - nq + 1, nk) : nk;
        for (int j = 0; j < see; j++) {
            const T *k = (const T *)rows.k + (k0 + j) * rows.k_stride + kh * rows.k_head_stride + E * lane;
            const T *v = (const T *)rows.v + (k0 + j) * rows.v_stride + kh * rows.v_head_stride + E * lane;
            float s = 0.0f;
            for (int e = 0; e < E; e++) s += x[e] * nmoe_elem<T>::get(k[e]);
            s = nmoe_wave_sum_tree(s) * scale;
            const float mn = fmaxf(m, s), a = __expf(m - mn), p = __expf(s - mn);
            m = mn;
            l = l * a + p;
            for (int e = 0; e < E; e++) o[e] = o[e] * a + p * nmoe_elem<T>::get(v[e]);
        }
        T *dst = out + ((int64_t)(q0 + i) * rows.q_heads + h) * D + E * lane;
        for (int e = 0; e < E; e++) dst[e] = nmoe_elem<T>::put(see <= 0 ? 0.0f : o[e] / l);
        if (lse != NULL && lane == 0) lse[(int64_t)(q0 + i) * rows.q_heads + h] = see <= 0 ? -INFINITY : m + logf(l);
    }
}

template <typename T>
static void nmoe_pr_launch(hipStream_t s, const nmoe_hip_qkv &r, int nseq, const int32_t *cu_q, const int32_t *cu_k,
                           int ntok_q, int ntok_k, int max_q, int causal, float scale, void *out, float *lse) {
    const dim3 g((max_q + NMOE_PR_WAVES - 1) / NMOE_PR_WAVES, r.q_heads, nseq), b(64 * NMOE_PR_WAVES);
    T *o = (T *)out;
    if (r.head_dim == 64)
        hipLaunchKernelGGL((nmoe_attn_prompt_kernel<T, 64>), g, b, 0, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k, causal, scale, o, lse);
    else if (r.head_dim == 128)
        hipLaunchKernelGGL((nmoe_attn_prompt_kernel<T, 128>), g, b, 0, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k, causal, scale, o, lse);
    else
        hipLaunchKernelGGL((nmoe_attn_prompt_kernel<T, 256>), g, b, 0, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k, causal, scale, o, lse);
}

extern "C" int nmoe_attn_prompt(nmoe_hip_ctx *ctx, const nmoe_hip_qkv *rows, int nseq, const int32_t *cu_q,
                                const int32_t *cu_k, int ntok_q, int ntok_k, int max_q, int max_k, int causal,
                                float scale, void *out, float *lse, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_check_rows(ctx, rows, 1);
    if (rc != NMOE_HIP_OK) return rc;
    if (!nmoe_is_half(rows->dtype)) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: dtype %d is neither bf16 nor f16", rows->dtype);
    if (cu_q == NULL || out == NULL || !nmoe_aligned(out, 16) || !nmoe_aligned(cu_q, 4) || !nmoe_aligned(cu_k, 4) ||
        !nmoe_aligned(lse, 4))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: cu_q and out (16-byte aligned) are required");
    if (nseq < 0 || nseq > 65535 || ntok_q < 0 || ntok_k < 0 || max_q < 0 || max_k < 0 || !isfinite(scale))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: nseq %d outside 0..65535, a negative size or a scale that is not finite", nseq);
    if (nseq == 0 || ntok_q == 0) return NMOE_HIP_OK;
    if (max_q < 1) max_q = 1;
    if (max_q > ntok_q) max_q = ntok_q;
    if (cu_k == NULL) cu_k = cu_q;
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (rows->dtype == NMOE_HIP_BF16)
        nmoe_pr_launch<nmoe_bf16>(s, *rows, nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, causal, scale, out, lse);
    else
        nmoe_pr_launch<_Float16>(s, *rows, nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, causal, scale, out, lse);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
