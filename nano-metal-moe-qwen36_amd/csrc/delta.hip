/*
 * delta.hip -- the gated delta rule, one token a sequence (nmoe_delta_step)
 * and over packed prompts (nmoe_delta_prompt).
 */
#include "nmoe_context.h"

#define NMOE_DELTA_MIN_G (-100.0f)

/* Token by token: one block a sequence and head of v; thread (r, c) of
 * 256 / DV x DV holds DK * DV / 256 values of column c of the state. */
template <typename T, int DK, int DV>
__global__ void __launch_bounds__(256)
    nmoe_delta_tokens_kernel(nmoe_hip_delta_rule d, const int32_t *cu, int ntok) {
    constexpr int R = 256 / DV, N = DK / R;
    __shared__ float s_q[DK], s_k[DK], s_part[2][R][DV], s_n[2];
    const int b = blockIdx.x / d.v_heads, h = blockIdx.x % d.v_heads, kh = h / (d.v_heads / d.k_heads);
    const int tid = threadIdx.x, c = tid % DV, r = tid / DV;
    const int t0 = cu != NULL ? min(max(cu[b], 0), ntok) : b, t1 = cu != NULL ? min(max(cu[b + 1], t0), ntok) : b + 1;
    const int state = d.state_index != NULL ? d.state_index[b] : b;
    T *out = (T *)d.out;
    if (state < 0 || state >= d.num_states) {
        for (int t = t0; t < t1; t++)
            for (int i = tid; i < DV; i += 256)
                out[((int64_t)t * d.v_heads + h) * DV + i] = nmoe_elem<T>::put(state < 0 ? 0.0f : NAN);
        return;
    }
    const int64_t at = ((int64_t)state * d.v_heads + h) * DK * DV;
    float S[N];
#pragma unroll
    for (int i = 0; i < N; i++) S[i] = d.state_in != NULL ? d.state_in[at + (r * N + i) * DV + c] : 0.0f;
    for (int t = t0; t < t1; t++) {
        __syncthreads();
        for (int i = tid; i < DK; i += 256) {
            s_q[i] = nmoe_elem<T>::get(((const T *)d.q)[t * d.q_stride + kh * DK + i]);
            s_k[i] = nmoe_elem<T>::get(((const T *)d.k)[t * d.k_stride + kh * DK + i]);
        }
        __syncthreads();
        if (tid < 128) {
            const float *x = tid < 64 ? s_q : s_k;
            float ss = 0.0f;
            for (int i = tid % 64; i < DK; i += 64) ss += x[i] * x[i];
            ss = nmoe_wave_sum_tree(ss);
            if (tid % 64 == 0) s_n[tid / 64] = d.l2 ? rsqrtf(ss + d.eps) : 1.0f;
        }
        __syncthreads();
        const float nq = s_n[0] * d.scale, nk = s_n[1], g = __expf(fmaxf(d.g[(int64_t)t * d.v_heads + h], NMOE_DELTA_MIN_G));
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            S[i] *= g;
            a += S[i] * s_k[r * N + i];
        }
        s_part[0][r][c] = a;
        __syncthreads();
        a = 0.0f;
        for (int i = 0; i < R; i++) a += s_part[0][i][c];
        const float v = nmoe_elem<T>::get(((const T *)d.v)[t * d.v_stride + h * DV + c]);
        const float u = d.beta[(int64_t)t * d.v_heads + h] * (v - nk * a) * nk;
        float o = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            S[i] += s_k[r * N + i] * u;
            o += S[i] * s_q[r * N + i];
        }
        s_part[1][r][c] = o;
        __syncthreads();
        if (r == 0) {
            o = 0.0f;
            for (int i = 0; i < R; i++) o += s_part[1][i][c];
            out[((int64_t)t * d.v_heads + h) * DV + c] = nmoe_elem<T>::put(o * nq);
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) d.state_out[at + (r * N + i) * DV + c] = S[i];
}

template <typename T>
static void nmoe_delta_launch(hipStream_t s, const nmoe_hip_delta_rule &d, int nseq, const int32_t *cu, int ntok) {
    const dim3 g((uint32_t)nseq * d.v_heads), b(256);
    if (d.k_dim == 64 && d.v_dim == 64)
        hipLaunchKernelGGL((nmoe_delta_tokens_kernel<T, 64, 64>), g, b, 0, s, d, cu, ntok);
    else if (d.k_dim == 64)
        hipLaunchKernelGGL((nmoe_delta_tokens_kernel<T, 64, 128>), g, b, 0, s, d, cu, ntok);
    else if (d.v_dim == 64)
        hipLaunchKernelGGL((nmoe_delta_tokens_kernel<T, 128, 64>), g, b, 0, s, d, cu, ntok);
    else
        hipLaunchKernelGGL((nmoe_delta_tokens_kernel<T, 128, 128>), g, b, 0, s, d, cu, ntok);
}

static int nmoe_delta_check(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, int ntok) {
    if (d == NULL) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: a rule is required");
    if (d->dtype != NMOE_HIP_F32 && !nmoe_is_half(d->dtype))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: unknown dtype %d", d->dtype);
    if (d->k_heads < 1 || d->v_heads < 1 || d->v_heads > NMOE_MAX_HEADS || d->v_heads % d->k_heads != 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: %d heads of v on %d of k (1..%d, a multiple)", d->v_heads, d->k_heads,
                         NMOE_MAX_HEADS);
    if ((d->k_dim != 64 && d->k_dim != 128) || (d->v_dim != 64 && d->v_dim != 128))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: k_dim %d and v_dim %d are 64 or 128", d->k_dim, d->v_dim);
    if (!nmoe_rows_ok(d->q, d->q_stride, 0, d->dtype) || !nmoe_rows_ok(d->k, d->k_stride, 0, d->dtype) ||
        !nmoe_rows_ok(d->v, d->v_stride, 0, d->dtype) || d->out == NULL || !nmoe_aligned(d->out, 16))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: q, k, v and out are 16-byte aligned, strides multiples of 16 bytes");
    if (d->g == NULL || d->beta == NULL || !nmoe_aligned(d->g, 4) || !nmoe_aligned(d->beta, 4))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: g and beta are required");
    if (d->state_out == NULL || !nmoe_aligned(d->state_out, 16) || !nmoe_aligned(d->state_in, 16) ||
        !nmoe_aligned(d->state_index, 4) || d->num_states < 1)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: state_out (16-byte aligned) of num_states >= 1 is required");
    if (!isfinite(d->scale) || (d->l2 && !(d->eps >= 0.0f)))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: a finite scale and, with l2, eps >= 0 are required");
    if (nseq < 0 || nseq > (1 << 20) || ntok < 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: nseq %d outside 0..2^20 or ntok %d < 0", nseq, ntok);
    return NMOE_HIP_OK;
}

static int nmoe_delta_run(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, const int32_t *cu, int ntok,
                          void *stream) {
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (d->dtype == NMOE_HIP_F32)
        nmoe_delta_launch<float>(s, *d, nseq, cu, ntok);
    else if (d->dtype == NMOE_HIP_BF16)
        nmoe_delta_launch<nmoe_bf16>(s, *d, nseq, cu, ntok);
    else
        nmoe_delta_launch<_Float16>(s, *d, nseq, cu, ntok);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}

extern "C" int nmoe_delta_step(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_delta_check(ctx, d, nseq, nseq);
    if (rc != NMOE_HIP_OK || nseq == 0) return rc;
    return nmoe_delta_run(ctx, d, nseq, NULL, nseq, stream);
}

extern "C" size_t nmoe_delta_prompt_workspace(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, int ntok) {
    if (ctx == NULL || nmoe_delta_check(ctx, d, nseq, ntok) != NMOE_HIP_OK) return 0;
    return 0;
}

extern "C" int nmoe_delta_prompt(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, const int32_t *cu, int ntok,
                                 int max_len, void *ws, size_t ws_bytes, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_delta_check(ctx, d, nseq, ntok);
    if (rc != NMOE_HIP_OK) return rc;
    if (cu == NULL || !nmoe_aligned(cu, 4) || max_len < 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: cu and max_len >= 0 are required");
    (void)ws;
    (void)ws_bytes;
    if (nseq == 0) return NMOE_HIP_OK;
    return nmoe_delta_run(ctx, d, nseq, cu, ntok, stream);
}
