/*
 * kv.hip -- appending keys and values to a paged cache, with the norm and
 * the rotation of q and k on the way (nmoe_kv_append).
 */
#include "nmoe_context.h"

int nmoe_check_cache(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *c) {
    if (c == NULL || c->k == NULL || c->v == NULL || !nmoe_aligned(c->k, 16) || !nmoe_aligned(c->v, 16))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: k and v (16-byte aligned) are required");
    if (!nmoe_is_half(c->dtype)) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: dtype %d is neither bf16 nor f16", c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: head_dim %d is not 64, 128 or 256", c->head_dim);
    if (c->kv_heads < 1 || c->kv_heads > NMOE_MAX_HEADS)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: kv_heads %d outside 1..%d", c->kv_heads, NMOE_MAX_HEADS);
    if (c->page_size < 16 || c->page_size % 16 != 0 || c->num_pages < 1 ||
        (int64_t)c->page_size * c->num_pages > 0x7fffffff)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: page_size %d (a multiple of 16) times num_pages %d outside 1..2^31-1",
                         c->page_size, c->num_pages);
    if (!nmoe_stride_ok(c->page_stride, c->dtype, NMOE_PAGE_STRIDE) ||
        !nmoe_stride_ok(c->token_stride, c->dtype, NMOE_ROW_STRIDE) ||
        !nmoe_stride_ok(c->head_stride, c->dtype, NMOE_ROW_STRIDE))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "cache: strides are multiples of 8 elements, not negative, below 2^%d "
                                               "(page_stride 2^%d)", NMOE_ROW_STRIDE, NMOE_PAGE_STRIDE);
    return NMOE_HIP_OK;
}

int nmoe_check_rows(nmoe_hip_ctx *ctx, const nmoe_hip_qkv *r, int with_q) {
    if (r == NULL) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "rows are required");
    if (r->dtype != NMOE_HIP_F32 && !nmoe_is_half(r->dtype))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "rows: unknown dtype %d", r->dtype);
    if (r->head_dim != 64 && r->head_dim != 128 && r->head_dim != 256)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "rows: head_dim %d is not 64, 128 or 256", r->head_dim);
    if (r->kv_heads < 1 || r->kv_heads > NMOE_MAX_HEADS ||
        (with_q && (r->q_heads < 1 || r->q_heads > NMOE_MAX_HEADS || r->q_heads % r->kv_heads != 0)))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "rows: %d query heads on %d key heads (1..%d, a multiple)", r->q_heads,
                         r->kv_heads, NMOE_MAX_HEADS);
    if (!nmoe_rows_ok(r->k, r->k_stride, r->k_head_stride, r->dtype) ||
        !nmoe_rows_ok(r->v, r->v_stride, r->v_head_stride, r->dtype) ||
        (with_q && !nmoe_rows_ok(r->q, r->q_stride, r->q_head_stride, r->dtype)))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "rows: q, k and v are 16-byte aligned, their strides multiples of 16 "
                                               "bytes, not negative, below 2^%d", NMOE_ROW_STRIDE);
    return NMOE_HIP_OK;
}

#define NMOE_KV_THREADS 256
#define NMOE_KV_AHEAD 3
#define NMOE_KV_BLOCKS 4 /* a CU */
#define NMOE_KV_PAIRS 128 /* rotated pairs of the widest head */

/* cos and sin of position * inv_freq, reduced to a turn in 64 bits: a
 * position of 2^31 times a frequency of 24 bits has 55, so the product is
 * off by at most 2^-22 turns there and exact below 2^29. */
__device__ __forceinline__ void nmoe_turn(int position, float inv_freq, float &c, float &s) {
    const double turns = (double)position * (double)inv_freq * 0.15915494309189533577;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
}

/* One block a token, or several in turn.  A row of D elements is held by D / 8
 * lanes, 8 neighbouring elements each, so a pair of the half-split rotation is
 * lane +- rotary_dim / 16 with the same element, and an interleaved pair is in
 * one lane.
 * It is bound by its bytes, and those by how many are under way: a thread asks
 * for NMOE_KV_AHEAD rows at once, and for the next, which may be the next
 * token's, before it works on them.  4097 tokens of 16 query and 2 key heads
 * of 256, bf16: 84 MB in 20 us, 4.2 TB/s (a plain copy of as many: 17.7 us);
 * a block a token took 23.6.  2000 of 32 and 8 heads of 128: 13.1 us instead
 * of 17.3.  One token: 4.6 us, the launch. */
template <typename T, typename C, int D>
__global__ void __launch_bounds__(NMOE_KV_THREADS)
    nmoe_kv_append_kernel(nmoe_hip_qkv rows, nmoe_hip_kv_cache cache, nmoe_hip_qk_prep prep, const int32_t *positions,
                          const int64_t *slots, int ntok, C *q_out) {
    constexpr int LANES = D / 8, PER = NMOE_KV_THREADS / LANES, STEP = NMOE_KV_AHEAD * PER;
    __shared__ float s_cos[2][NMOE_KV_PAIRS], s_sin[2][NMOE_KV_PAIRS];
    const int tid = threadIdx.x, half = prep.rotary_dim / 2;
    const int qh = q_out != NULL ? rows.q_heads : 0, all = qh + 2 * rows.kv_heads;
    const int lane = tid % LANES, e0 = 8 * lane;
    const T *qr = (const T *)rows.q + e0, *kr = (const T *)rows.k + e0, *vr = (const T *)rows.v + e0;
    auto load = [&](int t, int r0, nmoe_pack<T, 8> (&raw)[NMOE_KV_AHEAD]) {
#pragma unroll
        for (int i = 0; i < NMOE_KV_AHEAD; i++) {
            const int r = min(r0 + i * PER + tid / LANES, all - 1); /* behind the last: that one again, not stored */
            const T *p = r < qh                   ? qr + t * rows.q_stride + r * rows.q_head_stride
                         : r < qh + rows.kv_heads ? kr + t * rows.k_stride + (r - qh) * rows.k_head_stride
                                                  : vr + t * rows.v_stride + (r - qh - rows.kv_heads) * rows.v_head_stride;
            raw[i] = *(const nmoe_pack<T, 8> *)p;
        }
    };
    static_assert(NMOE_KV_PAIRS <= NMOE_KV_THREADS, "a thread a pair");
    const float freq = tid < half ? prep.inv_freq[tid] : 0.0f;
    auto angles = [&](int position, int buf) {
        if (tid < half) nmoe_turn(position, freq, s_cos[buf][tid], s_sin[buf][tid]);
    };
    const bool turns = e0 < prep.rotary_dim, upper = e0 >= half;
    uint4 qw = {0, 0, 0, 0}, kw = {0, 0, 0, 0};
    if (prep.qk_norm && prep.q_norm != NULL) qw = *(const uint4 *)(prep.q_norm + e0);
    if (prep.qk_norm && prep.k_norm != NULL) kw = *(const uint4 *)(prep.k_norm + e0);
    const float q1 = prep.q_norm == NULL || prep.add_one ? 1.0f : 0.0f, k1 = prep.k_norm == NULL || prep.add_one ? 1.0f : 0.0f;
    int t = blockIdx.x, r0 = 0, buf = 0;
    nmoe_pack<T, 8> xa[NMOE_KV_AHEAD], xb[NMOE_KV_AHEAD];
    /* of this token and the next: asked for before the rows, so that the wait for them is none for those (without a
     * rotation no position is read, but a place that is there: a load on some paths only would be waited for on all) */
    int64_t slot = slots[t], slot_next = slots[min(t + (int)gridDim.x, ntok - 1)];
    const int32_t *const at_position = half != 0 ? positions : (const int32_t *)slots;
    int position = at_position[t], position_next = at_position[min(t + (int)gridDim.x, ntok - 1)];
    load(t, 0, xa);
    if (half != 0) {
        angles(position, 0);
        nmoe_lds_sync();
    }
    /* the lane's angles, the same for every row: sin with the sign that its partner takes */
    float c[8], sn[8];
    /* one set of rows, with the next, which may be the next token's, under way */
    auto work = [&](nmoe_pack<T, 8> (&raw)[NMOE_KV_AHEAD], nmoe_pack<T, 8> (&ahead)[NMOE_KV_AHEAD]) {
        const bool last = r0 + STEP >= all;
        const int tn = last ? t + gridDim.x : t, rn = last ? 0 : r0 + STEP;
        const bool more = tn < ntok;
        if (r0 == 0 && turns) {
            const int p0 = prep.interleaved ? e0 / 2 : upper ? e0 - half : e0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                c[i] = s_cos[buf][p0 + (prep.interleaved ? i / 2 : i)];
                sn[i] = s_sin[buf][p0 + (prep.interleaved ? i / 2 : i)];
                if (prep.interleaved ? i % 2 == 0 : !upper) sn[i] = -sn[i];
            }
        }
        const int64_t slot_now = slot;
        if (more) {
            if (last) {
                slot = slot_next;
                position = position_next;
                slot_next = slots[min(tn + (int)gridDim.x, ntok - 1)];
                position_next = at_position[min(tn + (int)gridDim.x, ntok - 1)];
            }
            load(tn, rn, ahead);
            if (last && half != 0) angles(position, 1 - buf);
        }
        const bool keep = slot_now >= 0 && slot_now < (int64_t)cache.page_size * cache.num_pages;
        const uint32_t page = keep ? (uint32_t)slot_now / (uint32_t)cache.page_size : 0u;
        const uint32_t at = keep ? (uint32_t)slot_now % (uint32_t)cache.page_size : 0u;
        const int64_t row = (int64_t)page * cache.page_stride + (int64_t)at * cache.token_stride;
#pragma unroll
        for (int n = 0; n < NMOE_KV_AHEAD; n++) {
            const int r = r0 + n * PER + tid / LANES;
            if (r0 + n * PER >= all) break;
            const int kind = r < qh ? 0 : r < qh + rows.kv_heads ? 1 : 2;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = nmoe_elem<T>::get(raw[n].v[i]);
            if (prep.qk_norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss += x[i] * x[i];
                ss = nmoe_dpp_group_sum<LANES == 8 ? 8 : 16>(ss);
                if (LANES == 32) ss += __shfl_xor(ss, 16, 64);
                if (kind != 2) {
                    const float inv = rsqrtf(ss / (float)D + prep.eps), one = kind == 0 ? q1 : k1;
                    const uint4 w = kind == 0 ? qw : kw;
                    const uint32_t wb[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] *= inv * (one + nmoe_bf16f(i % 2 ? wb[i / 2] >> 16 : wb[i / 2] & 0xffffu));
                }
            }
            if (turns && kind != 2) { /* whole rows or none, and of a row both of a pair */
                float y[8];
                if (prep.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = x[i ^ 1];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = __shfl(x[i], (tid & 63) + (upper ? -half / 8 : half / 8), 64);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = fmaf(x[i], c[i], y[i] * sn[i]);
            }
            if (r >= all) continue;
            if (kind == 0)
                nmoe_store<C, 8>(q_out + ((int64_t)t * rows.q_heads + r) * D + e0, x);
            else if (keep)
                nmoe_store<C, 8>((C *)(kind == 1 ? cache.k : cache.v) + row +
                                     (kind == 1 ? r - qh : r - qh - rows.kv_heads) * cache.head_stride + e0, x);
        }
        if (last && more && half != 0) nmoe_lds_sync();
        if (last) buf = 1 - buf;
        t = tn;
        r0 = rn;
        return more;
    };
    while (work(xa, xb) && work(xb, xa)) {}
}

template <typename T, typename C>
static void nmoe_kv_launch(hipStream_t s, const nmoe_hip_qkv &rows, const nmoe_hip_kv_cache &cache,
                           const nmoe_hip_qk_prep &prep, int ntok, const int32_t *positions, const int64_t *slots,
                           int num_cus, void *q_out) {
    const int most = NMOE_KV_BLOCKS * (num_cus > 0 ? num_cus : 256);
    const dim3 g(ntok < most ? ntok : most), b(NMOE_KV_THREADS);
    if (cache.head_dim == 64)
        hipLaunchKernelGGL((nmoe_kv_append_kernel<T, C, 64>), g, b, 0, s, rows, cache, prep, positions, slots, ntok, (C *)q_out);
    else if (cache.head_dim == 128)
        hipLaunchKernelGGL((nmoe_kv_append_kernel<T, C, 128>), g, b, 0, s, rows, cache, prep, positions, slots, ntok, (C *)q_out);
    else
        hipLaunchKernelGGL((nmoe_kv_append_kernel<T, C, 256>), g, b, 0, s, rows, cache, prep, positions, slots, ntok, (C *)q_out);
}

template <typename T>
static void nmoe_kv_launch_from(hipStream_t s, const nmoe_hip_qkv &rows, const nmoe_hip_kv_cache &cache,
                                const nmoe_hip_qk_prep &prep, int ntok, const int32_t *positions,
                                const int64_t *slots, int num_cus, void *q_out) {
    if (cache.dtype == NMOE_HIP_BF16)
        nmoe_kv_launch<T, nmoe_bf16>(s, rows, cache, prep, ntok, positions, slots, num_cus, q_out);
    else
        nmoe_kv_launch<T, _Float16>(s, rows, cache, prep, ntok, positions, slots, num_cus, q_out);
}

extern "C" int nmoe_kv_append(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *cache, const nmoe_hip_qkv *rows,
                              const nmoe_hip_qk_prep *prep, int ntok, const int32_t *positions, const int64_t *slots,
                              void *q_out, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_check_cache(ctx, cache);
    if (rc == NMOE_HIP_OK) rc = nmoe_check_rows(ctx, rows, q_out != NULL || (rows != NULL && rows->q != NULL));
    if (rc != NMOE_HIP_OK) return rc;
    if ((rows->q != NULL) != (q_out != NULL) || !nmoe_aligned(q_out, 16))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: q rows and q_out (16-byte aligned) come together");
    if (rows->kv_heads != cache->kv_heads || rows->head_dim != cache->head_dim)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: rows of %d heads of %d, a cache of %d of %d", rows->kv_heads,
                         rows->head_dim, cache->kv_heads, cache->head_dim);
    if (ntok < 0 || ntok > NMOE_MAX_ROWS || positions == NULL || slots == NULL || !nmoe_aligned(positions, 4) ||
        !nmoe_aligned(slots, 8))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: 0 <= ntok <= 2^22, positions and slots are required");
    nmoe_hip_qk_prep p = {};
    if (prep != NULL) {
        p = *prep;
        if (p.rotary_dim < 0 || p.rotary_dim > cache->head_dim || p.rotary_dim % 16 != 0 ||
            (p.rotary_dim != 0 && (p.inv_freq == NULL || !nmoe_aligned(p.inv_freq, 4))))
            return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: rotary_dim %d (a multiple of 16 up to %d) and inv_freq",
                             p.rotary_dim, cache->head_dim);
        if (p.qk_norm && (!(p.eps >= 0.0f) || !nmoe_aligned(p.q_norm, 16) || !nmoe_aligned(p.k_norm, 16)))
            return nmoe_fail(ctx, NMOE_HIP_EINVAL, "append: eps >= 0 and norm weights 16-byte aligned");
    }
    if (ntok == 0) return NMOE_HIP_OK;
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (rows->dtype == NMOE_HIP_F32)
        nmoe_kv_launch_from<float>(s, *rows, *cache, p, ntok, positions, slots, ctx->num_cus, q_out);
    else if (rows->dtype == NMOE_HIP_BF16)
        nmoe_kv_launch_from<nmoe_bf16>(s, *rows, *cache, p, ntok, positions, slots, ctx->num_cus, q_out);
    else
        nmoe_kv_launch_from<_Float16>(s, *rows, *cache, p, ntok, positions, slots, ctx->num_cus, q_out);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
