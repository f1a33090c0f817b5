/*
 * kv8.hip -- appending keys and values to a paged cache in 8 bits, with the
 * norm and the rotation of q and k on the way (nmoe_kv8_append).
 *
 * 16 tokens of a head share a scale 2^e, the least with which none of their
 * magnitudes is above the largest code, 448.  A power of two costs a code of 4
 * significant bits nothing, makes quotient and product exact, and lets a block
 * grow: with a larger scale an older code is the old one with another
 * exponent, so it is rounded again only below 2^-6.
 */
#include "nmoe_kv8.h"

#define NMOE_KV8_THREADS 256
#define NMOE_KV8_WAVES (NMOE_KV8_THREADS / 64)
#define NMOE_KV8_SEQS (1 << 20)
#define NMOE_KV8_UNITS (1 << 20) /* most blocks of a launch; they go on to further ones */

int nmoe_check_cache8(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *c) {
    if (c == NULL || c->k == NULL || c->v == NULL || !nmoe_aligned(c->k, 16) || !nmoe_aligned(c->v, 16))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: k and v (16-byte aligned) are required");
    if (c->k_scale == NULL || c->v_scale == NULL || !nmoe_aligned(c->k_scale, 4) || !nmoe_aligned(c->v_scale, 4))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: k_scale and v_scale (4-byte aligned) are required");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: head_dim %d is not 64, 128 or 256", c->head_dim);
    if (c->kv_heads < 1 || c->kv_heads > NMOE_MAX_HEADS)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: kv_heads %d outside 1..%d", c->kv_heads, NMOE_MAX_HEADS);
    if (c->page_size < 16 || c->page_size % 16 != 0 || c->num_pages < 1 ||
        (int64_t)c->page_size * c->num_pages > 0x7fffffff)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: page_size %d (a multiple of 16) times num_pages %d outside 1..2^31-1",
                         c->page_size, c->num_pages);
    const int64_t st[3] = {c->page_stride, c->token_stride, c->head_stride};
    for (int i = 0; i < 3; i++)
        if (st[i] < 0 || st[i] % 16 != 0 || st[i] >= (int64_t)1 << (i == 0 ? NMOE_PAGE_STRIDE : NMOE_ROW_STRIDE))
            return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: strides are multiples of 16 bytes, not negative, below 2^%d "
                                                   "(page_stride 2^%d)", NMOE_ROW_STRIDE, NMOE_PAGE_STRIDE);
    return NMOE_HIP_OK;
}

/* Units are numbered (sequence, block of 16 tokens, part of the heads).  How
 * many blocks a sequence has is known on the device alone: sequence b's begin
 * at cu[b] / 16 + 2 b, which leaves it n / 16 + 2 or more, and n tokens from
 * any place on touch no more than (n + 30) / 16 of them. */
__device__ __forceinline__ int64_t nmoe_kv8_first(const int32_t *cu, int b, int ntok) {
    return min(max(cu[b], 0), ntok) / 16 + 2 * (int64_t)b;
}

/* The sequence that unit `slot` belongs to: 64 places at a time. */
__device__ __forceinline__ int nmoe_kv8_find(const int32_t *cu, int nseq, int ntok, int64_t slot) {
    const int lane = threadIdx.x % 64;
    int lo = 0, n = nseq;
    while (n > 1) {
        const int step = (n + 63) / 64, at = lane * step;
        const uint64_t below = __ballot(at < n && nmoe_kv8_first(cu, lo + min(at, n - 1), ntok) <= slot);
        const int last = max((int)__popcll(below) - 1, 0) * step;
        lo += last;
        n = min(step, n - last);
    }
    return lo;
}

/* A block of 4 wavefronts: 16 tokens, a wavefront a head of q, k or v.  A
 * row is held by D / 8 lanes, 8 neighbouring elements each, so a wavefront has
 * all of a head's 16 rows in registers when it has their largest magnitude. */
template <typename T, typename C, int D>
__global__ void __launch_bounds__(NMOE_KV8_THREADS)
    nmoe_kv8_append_kernel(nmoe_hip_qkv rows, nmoe_hip_kv8_cache cache, nmoe_hip_qk_prep prep, int nseq,
                           const int32_t *cu, int ntok, const int32_t *seq_lens, const int32_t *page_table, int max_pages,
                           const int32_t *positions, C *q_out, int64_t slots, int parts) {
    constexpr int LANES = D / 8, R = 64 / LANES, STEPS = 16 / R;
    __shared__ float s_cos[16][D / 2], s_sin[16][D / 2];
    const int tid = threadIdx.x, lane = tid % 64, e0 = 8 * (lane % LANES), half = prep.rotary_dim / 2;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int qh = q_out != NULL ? rows.q_heads : 0, all = qh + 2 * rows.kv_heads;
    const bool turns = e0 < prep.rotary_dim, upper = e0 >= half;
    for (int64_t unit = blockIdx.x; unit < slots * parts; unit += gridDim.x) {
        const int64_t slot = unit / parts;
        const int b = nmoe_kv8_find(cu, nseq, ntok, slot);
        const int t0 = min(max(cu[b], 0), ntok), n = min(max(cu[b + 1], t0), ntok) - t0, len = seq_lens[b];
        const bool bad = len < n || nmoe_kv8_len(len, max_pages, cache.page_size) < 0;
        const int begin = bad ? 0 : len - n; /* tokens before these */
        const int64_t first = nmoe_kv8_first(cu, b, ntok), block = slot - first + begin / 16;
        if (n == 0 || slot < first || block * 16 >= (int64_t)begin + n) continue; /* the whole workgroup */
        const int at = (int)block * 16, lo = max(begin - at, 0), hi = min(begin + n - at, 16); /* places of new tokens */
        const int tile = (int)(unit % parts) * NMOE_KV8_WAVES + wave;
        const int token = t0 + at - begin; /* row of place 0 */
        if (half != 0) {
            for (int i = tid; i < 16 * half; i += NMOE_KV8_THREADS) {
                const int p = i / half, f = i % half;
                if (p >= lo && p < hi)
                    nmoe_turn(positions != NULL ? positions[token + p] : at + p, prep.inv_freq[f], s_cos[p][f], s_sin[p][f]);
            }
            __syncthreads();
        }
        if (tile < all) {
            const int kind = tile < qh ? 0 : tile < qh + rows.kv_heads ? 1 : 2;
            const int head = kind == 0 ? tile : kind == 1 ? tile - qh : tile - qh - rows.kv_heads;
            const T *src = (const T *)(kind == 0 ? rows.q : kind == 1 ? rows.k : rows.v) + e0 +
                           head * (kind == 0 ? rows.q_head_stride : kind == 1 ? rows.k_head_stride : rows.v_head_stride);
            const int64_t stride = kind == 0 ? rows.q_stride : kind == 1 ? rows.k_stride : rows.v_stride;
            float x[STEPS][8];
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int p = min(max(s * R + lane / LANES, lo), hi - 1); /* rows there are */
                nmoe_load<T, 8>(src + (token + p) * stride, x[s]);
            }
            const uint16_t *norm = kind == 0 ? prep.q_norm : prep.k_norm;
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = 1.0f;
            if (prep.qk_norm && kind != 2 && norm != NULL) {
                nmoe_load<nmoe_bf16, 8>((const nmoe_bf16 *)norm + e0, w);
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] += prep.add_one ? 1.0f : 0.0f;
            }
            const int page = bad ? -1 : page_table[(int64_t)b * max_pages + at / cache.page_size];
            const bool keep = kind != 0 && page >= 0 && page < cache.num_pages;
            float amax = 0.0f;
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int p = s * R + lane / LANES;
                if (prep.qk_norm && kind != 2) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; i++) ss += x[s][i] * x[s][i];
                    ss = nmoe_dpp_group_sum<LANES == 8 ? 8 : 16>(ss);
                    if (LANES == 32) ss += __shfl_xor(ss, 16, 64);
                    const float inv = rsqrtf(ss / (float)D + prep.eps);
#pragma unroll
                    for (int i = 0; i < 8; i++) x[s][i] *= inv * w[i];
                }
                if (half != 0 && kind != 2) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        y[i] = prep.interleaved ? x[s][i ^ 1] : __shfl(x[s][i], (lane + (upper ? -half / 8 : half / 8)) & 63, 64);
                    if (turns) {
                        const int f0 = prep.interleaved ? e0 / 2 : upper ? e0 - half : e0;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int f = f0 + (prep.interleaved ? i / 2 : i);
                            const bool minus = prep.interleaved ? i % 2 == 0 : !upper;
                            x[s][i] = fmaf(x[s][i], s_cos[p][f], y[i] * (minus ? -s_sin[p][f] : s_sin[p][f]));
                        }
                    }
                }
                if (kind == 0) {
                    if (p >= lo && p < hi) {
                        if (bad) {
#pragma unroll
                            for (int i = 0; i < 8; i++) x[s][i] = NAN;
                        }
                        nmoe_store<C, 8>(q_out + ((int64_t)(token + p) * rows.q_heads + head) * D + e0, x[s]);
                    }
                } else if (p >= lo && p < hi) {
#pragma unroll
                    for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[s][i]) < INFINITY ? fabsf(x[s][i]) : 0.0f);
                }
            }
            if (keep) {
                amax = nmoe_wave_max_f(amax);
                const int place = at % cache.page_size;
                uint8_t *dst = (uint8_t *)(kind == 1 ? cache.k : cache.v) + page * cache.page_stride +
                               place * cache.token_stride + head * cache.head_stride + e0;
                float *const scale = (kind == 1 ? cache.k_scale : cache.v_scale) + nmoe_kv8_scale_at(cache, page, place, head);
                int e = nmoe_kv8_power(amax);
                if (lo > 0) { /* older tokens in the block */
                    const int was = min(max((int)(__float_as_uint(*scale) >> 23 & 255u) - 127, NMOE_KV8_LOW), NMOE_KV8_HIGH);
                    if (was < e) {
                        const float f = nmoe_kv8_two_to(max(was - e, -126));
#pragma unroll
                        for (int s = 0; s < STEPS; s++) {
                            const int p = s * R + lane / LANES;
                            if (p < lo) {
                                uint2 c = *(const uint2 *)(dst + p * cache.token_stride);
                                c.x = nmoe_kv8_again(c.x, f);
                                c.y = nmoe_kv8_again(c.y, f);
                                *(uint2 *)(dst + p * cache.token_stride) = c;
                            }
                        }
                    }
                    e = max(e, was);
                }
                const float inv = nmoe_kv8_two_to(-e);
#pragma unroll
                for (int s = 0; s < STEPS; s++) {
                    const int p = s * R + lane / LANES;
                    if (p >= lo && p < hi) {
                        const uint2 c = {nmoe_kv8_codes(&x[s][0], inv), nmoe_kv8_codes(&x[s][4], inv)};
                        *(uint2 *)(dst + p * cache.token_stride) = c;
                    }
                }
                if (lane == 0) *scale = nmoe_kv8_two_to(e);
            }
        }
        if (half != 0) __syncthreads(); /* the angles are read */
    }
}

template <typename T, typename C>
static void nmoe_kv8_launch(hipStream_t s, const nmoe_hip_qkv &r, const nmoe_hip_kv8_cache &c, const nmoe_hip_qk_prep &p,
                            int nseq, const int32_t *cu, int ntok, const int32_t *lens, const int32_t *table, int max_pages,
                            const int32_t *positions, void *q_out) {
    const int all = (q_out != NULL ? r.q_heads : 0) + 2 * r.kv_heads, parts = (all + NMOE_KV8_WAVES - 1) / NMOE_KV8_WAVES;
    const int64_t slots = ntok / 16 + 2 * (int64_t)nseq, units = slots * parts;
    const dim3 g((uint32_t)(units < NMOE_KV8_UNITS ? units : NMOE_KV8_UNITS)), b(NMOE_KV8_THREADS);
    if (c.head_dim == 64)
        hipLaunchKernelGGL((nmoe_kv8_append_kernel<T, C, 64>), g, b, 0, s, r, c, p, nseq, cu, ntok, lens, table, max_pages,
                           positions, (C *)q_out, slots, parts);
    else if (c.head_dim == 128)
        hipLaunchKernelGGL((nmoe_kv8_append_kernel<T, C, 128>), g, b, 0, s, r, c, p, nseq, cu, ntok, lens, table, max_pages,
                           positions, (C *)q_out, slots, parts);
    else
        hipLaunchKernelGGL((nmoe_kv8_append_kernel<T, C, 256>), g, b, 0, s, r, c, p, nseq, cu, ntok, lens, table, max_pages,
                           positions, (C *)q_out, slots, parts);
}

template <typename T>
static void nmoe_kv8_launch_from(hipStream_t s, const nmoe_hip_qkv &r, const nmoe_hip_kv8_cache &c, const nmoe_hip_qk_prep &p,
                                 int nseq, const int32_t *cu, int ntok, const int32_t *lens, const int32_t *table,
                                 int max_pages, const int32_t *positions, void *q_out, int q_dtype) {
    if (q_dtype == NMOE_HIP_BF16)
        nmoe_kv8_launch<T, nmoe_bf16>(s, r, c, p, nseq, cu, ntok, lens, table, max_pages, positions, q_out);
    else
        nmoe_kv8_launch<T, _Float16>(s, r, c, p, nseq, cu, ntok, lens, table, max_pages, positions, q_out);
}

extern "C" int nmoe_kv8_append(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const nmoe_hip_qkv *rows,
                               const nmoe_hip_qk_prep *prep, int nseq, const int32_t *cu, int ntok, const int32_t *seq_lens,
                               const int32_t *page_table, int max_pages, const int32_t *positions, void *q_out, int q_dtype,
                               void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_check_cache8(ctx, cache);
    if (rc == NMOE_HIP_OK) rc = nmoe_check_rows(ctx, rows, q_out != NULL || (rows != NULL && rows->q != NULL));
    if (rc != NMOE_HIP_OK) return rc;
    if ((rows->q != NULL) != (q_out != NULL) || !nmoe_aligned(q_out, 16))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: q rows and q_out (16-byte aligned) come together");
    if (!nmoe_is_half(q_dtype)) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: q_dtype %d is neither bf16 nor f16", q_dtype);
    if (rows->kv_heads != cache->kv_heads || rows->head_dim != cache->head_dim)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: rows of %d heads of %d, a cache of %d of %d", rows->kv_heads,
                         rows->head_dim, cache->kv_heads, cache->head_dim);
    if (nseq < 0 || nseq > NMOE_KV8_SEQS || ntok < 0 || ntok > NMOE_MAX_ROWS || max_pages < 1)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: 0 <= nseq <= 2^20, 0 <= ntok <= 2^22, max_pages >= 1 are required");
    if (cu == NULL || seq_lens == NULL || page_table == NULL || !nmoe_aligned(cu, 4) || !nmoe_aligned(seq_lens, 4) ||
        !nmoe_aligned(page_table, 4) || !nmoe_aligned(positions, 4))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: cu, seq_lens and page_table are required, 4-byte aligned");
    nmoe_hip_qk_prep p;
    rc = nmoe_check_prep(ctx, prep, cache->head_dim, &p);
    if (rc != NMOE_HIP_OK) return rc;
    if (ntok == 0 || nseq == 0) return NMOE_HIP_OK;
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (rows->dtype == NMOE_HIP_F32)
        nmoe_kv8_launch_from<float>(s, *rows, *cache, p, nseq, cu, ntok, seq_lens, page_table, max_pages, positions, q_out, q_dtype);
    else if (rows->dtype == NMOE_HIP_BF16)
        nmoe_kv8_launch_from<nmoe_bf16>(s, *rows, *cache, p, nseq, cu, ntok, seq_lens, page_table, max_pages, positions, q_out, q_dtype);
    else
        nmoe_kv8_launch_from<_Float16>(s, *rows, *cache, p, nseq, cu, ntok, seq_lens, page_table, max_pages, positions, q_out, q_dtype);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
