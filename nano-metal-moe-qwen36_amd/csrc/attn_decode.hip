/*
 * attn_decode.hip -- attention of one new token a sequence over a paged
 * key-value cache (nmoe_attn_decode).
 */
#include "nmoe_context.h"

#define NMOE_DEC_WAVES 4

/* One block a sequence and query head; wavefront w takes keys w, w + 4, ...
 * with a running maximum and sum, and the four are joined in LDS. */
template <typename T, int D>
__global__ void __launch_bounds__(64 * NMOE_DEC_WAVES)
    nmoe_attn_decode_kernel(nmoe_hip_kv_cache cache, const T *q, int q_heads, const int32_t *seq_lens,
                            const int32_t *page_table, int max_pages, float scale, T *out, float *lse) {
    constexpr int E = D / 64;
    __shared__ float s_m[NMOE_DEC_WAVES], s_l[NMOE_DEC_WAVES], s_o[NMOE_DEC_WAVES][D];
    __shared__ int s_bad;
    const int b = blockIdx.x / q_heads, h = blockIdx.x % q_heads, tid = threadIdx.x, w = tid / 64, lane = tid % 64;
    const int kh = h / (q_heads / cache.kv_heads), len = seq_lens[b];
    if (tid == 0) s_bad = len > 0 && (int64_t)len > (int64_t)max_pages * cache.page_size;
    __syncthreads();
    const int pages = s_bad || len <= 0 ? 0 : (int)(((int64_t)len + cache.page_size - 1) / cache.page_size);
    for (int i = tid; i < pages; i += 64 * NMOE_DEC_WAVES)
        if ((uint32_t)page_table[(int64_t)b * max_pages + i] >= (uint32_t)cache.num_pages) s_bad = 1;
    __syncthreads();
    const bool bad = s_bad != 0;
    float x[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) {
        x[i] = nmoe_elem<T>::get(q[(int64_t)blockIdx.x * D + E * lane + i]);
        o[i] = 0.0f;
    }
    if (!bad)
        for (int j = w; j < len; j += NMOE_DEC_WAVES) {
            const int page = page_table[(int64_t)b * max_pages + j / cache.page_size];
            const int64_t row = page * cache.page_stride + (j % cache.page_size) * cache.token_stride +
                                kh * cache.head_stride + E * lane;
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < E; i++) s += x[i] * nmoe_elem<T>::get(((const T *)cache.k)[row + i]);
            s = nmoe_wave_sum_tree(s) * scale;
            const float mn = fmaxf(m, s), a = __expf(m - mn), p = __expf(s - mn);
            m = mn;
            l = l * a + p;
#pragma unroll
            for (int i = 0; i < E; i++) o[i] = o[i] * a + p * nmoe_elem<T>::get(((const T *)cache.v)[row + i]);
        }
#pragma unroll
    for (int i = 0; i < E; i++) s_o[w][E * lane + i] = o[i];
    if (lane == 0) {
        s_m[w] = m;
        s_l[w] = l;
    }
    __syncthreads();
    float mt = -INFINITY, lt = 0.0f;
    for (int i = 0; i < NMOE_DEC_WAVES; i++) mt = fmaxf(mt, s_m[i]);
    for (int i = 0; i < NMOE_DEC_WAVES; i++) lt += s_m[i] == -INFINITY ? 0.0f : s_l[i] * __expf(s_m[i] - mt);
    for (int e = tid; e < D; e += 64 * NMOE_DEC_WAVES) {
        float v = 0.0f;
        for (int i = 0; i < NMOE_DEC_WAVES; i++) v += s_m[i] == -INFINITY ? 0.0f : s_o[i][e] * __expf(s_m[i] - mt);
        out[(int64_t)blockIdx.x * D + e] = nmoe_elem<T>::put(bad ? NAN : len <= 0 ? 0.0f : v / lt);
    }
    if (tid == 0 && lse != NULL) lse[blockIdx.x] = bad ? NAN : len <= 0 ? -INFINITY : mt + logf(lt);
}

template <typename T>
static void nmoe_dec_launch(hipStream_t s, const nmoe_hip_kv_cache &c, const void *q, int q_heads, int nseq,
                            const int32_t *lens, const int32_t *table, int max_pages, float scale, void *out,
                            float *lse) {
    const dim3 g((uint32_t)nseq * q_heads), b(64 * NMOE_DEC_WAVES);
    const T *tq = (const T *)q;
    T *to = (T *)out;
    if (c.head_dim == 64)
        hipLaunchKernelGGL((nmoe_attn_decode_kernel<T, 64>), g, b, 0, s, c, tq, q_heads, lens, table, max_pages, scale, to, lse);
    else if (c.head_dim == 128)
        hipLaunchKernelGGL((nmoe_attn_decode_kernel<T, 128>), g, b, 0, s, c, tq, q_heads, lens, table, max_pages, scale, to, lse);
    else
        hipLaunchKernelGGL((nmoe_attn_decode_kernel<T, 256>), g, b, 0, s, c, tq, q_heads, lens, table, max_pages, scale, to, lse);
}

static int nmoe_dec_check(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *cache, int q_heads, int nseq, int max_len) {
    int rc = nmoe_check_cache(ctx, cache);
    if (rc != NMOE_HIP_OK) return rc;
    if (q_heads < 1 || q_heads > NMOE_MAX_HEADS || q_heads % cache->kv_heads != 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: %d query heads on %d key heads (1..%d, a multiple)", q_heads,
                         cache->kv_heads, NMOE_MAX_HEADS);
    if (nseq < 0 || nseq > (1 << 20) || max_len < 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: nseq %d outside 0..2^20 or max_len %d < 0", nseq, max_len);
    return NMOE_HIP_OK;
}

extern "C" size_t nmoe_attn_decode_workspace(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *cache, int q_heads, int nseq,
                                             int max_len) {
    if (ctx == NULL || nmoe_dec_check(ctx, cache, q_heads, nseq, max_len) != NMOE_HIP_OK) return 0;
    return 0;
}

extern "C" int nmoe_attn_decode(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *cache, const void *q, int q_heads, int nseq,
                                const int32_t *seq_lens, const int32_t *page_table, int max_pages, int max_len,
                                float scale, void *out, float *lse, void *ws, size_t ws_bytes, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_dec_check(ctx, cache, q_heads, nseq, max_len);
    if (rc != NMOE_HIP_OK) return rc;
    if (q == NULL || out == NULL || seq_lens == NULL || page_table == NULL || !nmoe_aligned(q, 16) ||
        !nmoe_aligned(out, 16) || !nmoe_aligned(lse, 4) || !nmoe_aligned(seq_lens, 4) || !nmoe_aligned(page_table, 4))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: q and out (16-byte aligned), seq_lens and page_table are required");
    if (max_pages < 1 || !isfinite(scale))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: max_pages >= 1 and a finite scale are required");
    (void)ws;
    (void)ws_bytes;
    if (nseq == 0) return NMOE_HIP_OK;
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (cache->dtype == NMOE_HIP_BF16)
        nmoe_dec_launch<nmoe_bf16>(s, *cache, q, q_heads, nseq, seq_lens, page_table, max_pages, scale, out, lse);
    else
        nmoe_dec_launch<_Float16>(s, *cache, q, q_heads, nseq, seq_lens, page_table, max_pages, scale, out, lse);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
