/*
 * attn_prompt.hip -- attention over whole prompts packed one behind the
 * other, causal or full, with grouped heads (nmoe_attn_prompt).
 *
 * One pass over a query's keys with a running maximum m and sum l:
 *   s = c q.k,  p = 2^(s - m),  l += p,  o += p v;   out = o / l
 * (c = scale * log2(e)).  It is bound by the matrix cores: 4 D flops a pair of
 * query and key against 4 D bytes a key, which a block's 128 query rows
 * share.
 */
#include <type_traits>

#include "nmoe_context.h"

#define NMOE_PR_STRIDE (1 << 24) /* a tile's offsets stay below 2^31 bytes */
#define NMOE_PR_TOKENS (1 << 30)
#define NMOE_PR_SPLIT 8    /* key tiles from which on two groups of four pieces share them */
#define NMOE_PR_SHORT 64   /* keys up to which two groups of two do not */
#define NMOE_PR_SLACK 8.0f /* the running maximum may lag by 2^8: sums stay far below fp32's (and f16's) limit */

typedef __attribute__((address_space(3))) void nmoe_pr_lds;
typedef short nmoe_s4 __attribute__((ext_vector_type(4)));

/* Keys of a tile: what two buffers of K and V tiles leave room for two such
 * sets a CU (64 KB each). */
template <int D>
constexpr int nmoe_pr_keys = D == 256 ? 32 : 64;

template <typename T>
constexpr float nmoe_pr_lift = nmoe_elem<T>::dtype == NMOE_HIP_F16 ? 4.0f : 0.0f;

/* The 16-byte chunks of a tile's row are stored at chunk ^ f(row), so that
 * neither 16 rows' same chunk (a key operand's read) nor 4 rows' same 32
 * bytes (a transposing value read) meet in a bank.  256 bytes are the banks'
 * width: a 128-byte row's neighbour is already in the other half. */
template <int D>
__device__ __forceinline__ int nmoe_pr_swizzle(int row) {
    return (D == 64 ? row >> 1 & 1 : row & 3) << 2 | ((row >> 2) & 3);
}

/* A block: SUBS pieces of 32 query rows, numbered (32 rows, head) with the
 * heads of one key head side by side, and KG groups of SUBS wavefronts that
 * take the key tiles in turn (two where there are too few blocks to fill the
 * device; joined at the end).
 *
 * S^T (keys x queries) = K Q^T, 32x32x16: a lane holds one query's scores, so
 * maximum and sum need one exchange with lane + 32, and the weights are the
 * second product's column operand where they are: of 16 keys a lane has
 * 8 g + 4 (l / 32) + e (g < 2, e < 4), which is the order the product takes
 * them in.  O^T (dimensions x queries) = V^T P^T; V^T comes from V's rows by
 * the LDS's transposing reads.
 *
 * Tiles go from memory to LDS directly, the next while one is multiplied.
 * Rows behind the last key repeat it (their weights are 0).
 * 8191 tokens in three prompts (32 heads of 128): 218 GF in 230 to 245 us,
 * 0.9 PF/s, where a library product of 8192 a side reaches 1.2.  Of a tile's
 * 4000 cycles a block, the two products take 60%, the softmax 20%; the rest
 * is the barrier and the loads. */
template <typename T, int D, int SUBS, int KG>
__global__ void __launch_bounds__(64 * SUBS * KG, SUBS == 2 && D > 64 ? 1 : 2)
    nmoe_attn_prompt_kernel(nmoe_hip_qkv rows, int nseq, const int32_t *cu_q, const int32_t *cu_k, int ntok_q,
                            int ntok_k, int causal, float c, uint32_t q_and, uint32_t q_xor, T *out, float *lse) {
    typedef nmoe_mat<T> X;
    constexpr int GT = 64 * SUBS, KT = nmoe_pr_keys<D>, CPR = D / 8, RPI = GT / CPR, NI = KT / RPI, KS = KT / 32, DT = D / 32;
    constexpr int EVERY = KS * (D / 16) / (2 * NI);
    static_assert(EVERY * 2 * NI == KS * (D / 16), "a load to so many products");
    constexpr int TILE = KT * D, TURN = RPI < 16 ? 16 / RPI : 1;
    /* two buffers by name: of one array with an index, the compiler takes every read for one of the tile under way
     * too, and waits for that first */
    __shared__ alignas(16) uint16_t s_kv0[KG][2][TILE], s_kv1[KG][2][TILE];
    __shared__ float s_ml[2][SUBS][KG == 2 ? 64 : 1];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wq = wave % SUBS, kg = wave / SUBS, tg = tid % GT, hh = lane / 32;
    const int pairs = rows.kv_heads * nseq, group = rows.q_heads / rows.kv_heads;
    const int pair = blockIdx.x % pairs, kh = pair % rows.kv_heads, b = pair / rows.kv_heads;
    const int q0 = min(max(cu_q[b], 0), ntok_q), nq = min(max(cu_q[b + 1], q0), ntok_q) - q0;
    const int k0 = min(max(cu_k[b], 0), ntok_k), nk = min(max(cu_k[b + 1], k0), ntok_k) - k0;
    const int64_t subs = (int64_t)group * ((nq + 31) / 32), tiles = (subs + SUBS - 1) / SUBS;
    const int ahead = nk - nq + 1; /* query i sees keys below i + ahead */

    const T *kbase = (const T *)rows.k + k0 * rows.k_stride + kh * rows.k_head_stride;
    const T *vbase = (const T *)rows.v + k0 * rows.v_stride + kh * rows.v_head_stride;
    const uint32_t kstep = (uint32_t)rows.k_stride * 2, vstep = (uint32_t)rows.v_stride * 2;
    const int lrow = tg / CPR;
    uint32_t lchunk[TURN]; /* f repeats after 16 rows */
#pragma unroll
    for (int i = 0; i < TURN; i++) lchunk[i] = (uint32_t)((tg % CPR) ^ nmoe_pr_swizzle<D>(i * RPI + lrow)) * 16;

    /* load i of a tile's 2 NI: of K, then of V */
    auto load = [&](int left, const __amdgpu_buffer_rsrc_t &rk, const __amdgpu_buffer_rsrc_t &rv, auto buf, int n) {
        const int i = n % NI;
        const uint32_t row = (uint32_t)min(i * RPI + lrow, left - 1);
        const int at = (i * GT + wq * 64) * 8;
        if constexpr (decltype(buf)::value == 0) {
            if (n < NI)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (nmoe_pr_lds *)&s_kv0[kg][0][at], 16,
                                                         (int)(row * kstep + lchunk[i % TURN]), 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (nmoe_pr_lds *)&s_kv0[kg][1][at], 16,
                                                         (int)(row * vstep + lchunk[i % TURN]), 0, 0, 0);
        } else {
            if (n < NI)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (nmoe_pr_lds *)&s_kv1[kg][0][at], 16,
                                                         (int)(row * kstep + lchunk[i % TURN]), 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (nmoe_pr_lds *)&s_kv1[kg][1][at], 16,
                                                         (int)(row * vstep + lchunk[i % TURN]), 0, 0, 0);
        }
    };

    /* a chunk's place is (chunk ^ f) * 8, in elements: other chunks of the row by the same bits of its number */
    const int kplace = lane % 32 * D + (hh ^ nmoe_pr_swizzle<D>(lane % 32)) * 8;
    const int vplace = (4 * hh + lane % 16 / 4) * D +
                       ((2 * (lane / 16 % 2) + lane % 4 / 2) ^ nmoe_pr_swizzle<D>(4 * hh + lane % 16 / 4)) * 8 + lane % 2 * 4;

    /* the latest rows, which see the most keys, first */
    for (int64_t tile = tiles - 1 - blockIdx.x / pairs; tile >= 0; tile -= gridDim.x / pairs) {
        const int64_t sub = tile * SUBS + wq, last = min(tile * SUBS + SUBS, subs) - 1;
        const bool active = sub < subs;
        const int tok = active ? (int)(sub / group) * 32 : 0, h = kh * group + (active ? (int)(sub % group) : 0);
        const int i = tok + lane % 32, see = causal ? min(i + ahead, nk) : nk;
        const int see_lo = causal ? tok + ahead : nk; /* every row of the piece sees these */
        const int see_hi = active ? (causal ? min(min(tok + 31, nq - 1) + ahead, nk) : nk) : 0;
        const int end = causal ? min(min((int)(last / group) * 32 + 31, nq - 1) + ahead, nk) : nk;
        const int nt = end > 0 ? (end + KT - 1) / KT : 0;

        nmoe_u4 qf[D / 16];
        const T *qr = (const T *)rows.q + (int64_t)(q0 + min(i, nq - 1)) * rows.q_stride + h * rows.q_head_stride + 8 * hh;
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
            qf[k] = *(const nmoe_u4 *)(qr + 16 * k);
#pragma unroll
            for (int e = 0; e < 4; e++) qf[k][e] = (qf[k][e] & q_and) ^ q_xor;
        }
        nmoe_f16v o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
        float m = -3.402823466e38f, l = 0.0f;

        auto work = [&](const int t, auto buf) {
            constexpr bool B = decltype(buf)::value != 0;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            /* the next tile (behind the last, that one again): a load to every EVERY products of the scores.  Asked for
             * at once, all wavefronts' loads stood in line, 500 to 900 cycles of 4500 (heads of 256: one prompt of
             * 2048 76 us instead of 73, of 500 25 instead of 22) */
            const int tn = min(t + KG, nt - 1), left = nk - tn * KT;
            const __amdgpu_buffer_rsrc_t rk = nmoe_buffer(kbase + (int64_t)tn * KT * rows.k_stride);
            const __amdgpu_buffer_rsrc_t rv = nmoe_buffer(vbase + (int64_t)tn * KT * rows.v_stride);
            const std::integral_constant<int, !B> other;
            if (t * KT >= see_hi) {
#pragma unroll
                for (int n = 0; n < 2 * NI; n++) load(left, rk, rv, other, n);
                return;
            }
            const uint16_t *sk = B ? s_kv1[kg][0] : s_kv0[kg][0], *sv = B ? s_kv1[kg][1] : s_kv0[kg][1];
            /* the lane's first places in a K and a V tile, made anew for each: the compiler kept each place derived
             * from them in a register of its own through the loop, and spilled more with heads of 256 (2 registers in
             * form 0 and 6 to 8 in form 1 still are) */
            int krow = kplace, vrow = vplace;
            asm volatile("" : "+v"(krow), "+v"(vrow));
            float s[KS][16];
#pragma unroll
            for (int k = 0; k < KS; k++) {
                nmoe_f16v x;
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = 0.0f;
                const uint16_t *p = sk + 32 * k * D;
#pragma unroll
                for (int d = 0; d < D / 16; d++) {
                    x = X::mma32(*(const nmoe_u4 *)(p + (krow ^ (2 * (d % 8)) * 8) + d / 8 * 128), qf[d], x);
                    if (EVERY == 1 || d % EVERY == 1) {
                        load(left, rk, rv, other, (k * (D / 16) + d) / EVERY);
                        __builtin_amdgcn_sched_barrier(0x106); /* stays between its products; LDS reads, VALU and SALU need not */
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; e++) s[k][e] = x[e];
            }
            if (t * KT + KT > see_lo) {
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (t * KT + 32 * k + 8 * (e / 4) + 4 * hh + e % 4 >= see) s[k][e] = -INFINITY;
            }
            float mt = s[0][0];
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 16; e++) mt = fmaxf(mt, s[k][e]);
            mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * c - nmoe_pr_lift<T>;
            if (__any(mt > m + NMOE_PR_SLACK)) {
                const float mn = fmaxf(m, mt), a = nmoe_exp2(m - mn);
                m = mn;
                l *= a;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[d][e] *= a;
            }
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    s[k][e] = nmoe_exp2(fmaf(s[k][e], c, -m));
                    l += s[k][e];
                }
#pragma unroll
            for (int u = 0; u < KT / 16; u++) {
                const nmoe_u4 pf = X::pack(&s[u / 2][8 * (u % 2)]); /* to 16 bits: the products take no more; l has them in fp32 */
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    typedef __attribute__((address_space(3))) nmoe_s4 lds_s4;
                    union {
                        nmoe_s4 h[2];
                        nmoe_u4 v;
                    } x;
#pragma unroll
                    for (int g = 0; g < 2; g++)
                        x.h[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s4 *)(sv + (16 * u + 8 * g) * D + (vrow ^ ((4 * (d % 4)) ^ (2 * g)) * 8) + d / 4 * 128));
                    o[d] = X::mma32(x.v, pf, o[d]);
                }
            }
        };
        __syncthreads();
        if (kg < nt) {
            const __amdgpu_buffer_rsrc_t rk = nmoe_buffer(kbase + (int64_t)kg * KT * rows.k_stride);
            const __amdgpu_buffer_rsrc_t rv = nmoe_buffer(vbase + (int64_t)kg * KT * rows.v_stride);
#pragma unroll
            for (int n = 0; n < 2 * NI; n++) load(nk - kg * KT, rk, rv, std::integral_constant<int, 0>(), n);
        }
        for (int t0 = 0; t0 < nt; t0 += 2 * KG) {
            work(t0 + kg, std::integral_constant<int, 0>());
            if (t0 + KG < nt) work(t0 + KG + kg, std::integral_constant<int, 1>());
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); /* the last loads are for no one, but not for the next block's LDS */
        l += __shfl_xor(l, 32, 64);
        if constexpr (KG == 2) {
            /* [piece][D / 2][64] */
            float *so = (float *)(wq < SUBS / 2 ? s_kv0[0][0] : s_kv1[0][0]) + wq % (SUBS / 2) * (D / 2) * 64;
            __syncthreads();
            if (kg == 1) {
                s_ml[0][wq][lane] = m;
                s_ml[1][wq][lane] = l;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) so[(16 * d + e) * 64 + lane] = o[d][e];
            }
            __syncthreads();
            if (kg == 0) {
                const float m1 = s_ml[0][wq][lane], mn = fmaxf(m, m1), a = nmoe_exp2(m - mn), a1 = nmoe_exp2(m1 - mn);
                m = mn;
                l = l * a + s_ml[1][wq][lane] * a1;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[d][e] = o[d][e] * a + so[(16 * d + e) * 64 + lane] * a1;
            }
        }
        if (kg == 0 && active && i < nq) {
            const int64_t oh = (int64_t)(q0 + i) * rows.q_heads + h;
            const float inv = see > 0 ? 1.0f / l : 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float z[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) z[j] = see > 0 ? o[d][4 * e + j] * inv : 0.0f;
                    nmoe_store<T, 4>(out + oh * D + 32 * d + 8 * e + 4 * hh, z);
                }
            if (lse != NULL && hh == 0) lse[oh] = see > 0 ? 0.69314718055994531f * (m + log2f(l)) : -INFINITY;
        }
    }
}

template <typename T, int D>
static void nmoe_pr_launch_as(nmoe_hip_ctx *ctx, hipStream_t s, const nmoe_hip_qkv &r, int nseq, const int32_t *cu_q,
                              const int32_t *cu_k, int ntok_q, int ntok_k, int max_q, int max_k, int causal, float scale,
                              void *out, float *lse) {
    const int group = r.q_heads / r.kv_heads;
    const int64_t pairs = (int64_t)r.kv_heads * nseq, subs = (int64_t)group * ((max_q + 31) / 32);
    /* c > 0, so that the largest score is the largest product: the sign goes to q, exactly, and a scale of 0 to q too */
    const float c = scale == 0.0f ? 1.0f : fabsf(scale) * 1.44269504088896341f;
    const uint32_t q_and = scale == 0.0f ? 0u : 0xffffffffu, q_xor = scale < 0.0f ? 0x80008000u : 0u;
    /* 0: pieces of 4, which share keys best; two blocks a CU overlap each other.  Where there are fewer of them than
     * that, two groups a block, if the keys are long enough to pay for joining them (2): pieces of 2, which use more
     * CUs, as long as the blocks are two rounds at most (the latest rows and the first ones in turn; of heads of 128,
     * whose pieces of 4 lose less, one round), else (1) pieces of 4.  Heads of 64 have two blocks a CU, so never more
     * than two rounds; the others one, by LDS.
     * In us, forms 0, 1, 2: one prompt of 500 (16 heads of 256) 31, 27, 21, of 2048 100, 70, 66, of 2300 -, 77, 90;
     * of 2000 (8 of 64) 35, 26, 18; of 1000 (16 of 128) 23, 21, 19, (32 of 128) 24, 23, 27; six of 50 (16 of 256)
     * 12.7, 16.1, 11.9; one of 32 (32 of 128) 7.5, 9.2, 8.1.
     * Form 0's line is too low for one long prompt, whose last rows bound it: on either side, 16 on 2 heads of 256 take
     * 154 (4064 tokens, form 1) and 199 (4096), of 128 78 and 88, 32 on 8 of 128 46 (2016) and 49 (2048), 8 of 64 100
     * (8064, form 2) and 130 (8192).  And the blocks are counted as if all sequences were max_q long: one of 2048 with
     * seven of 20 (16 of 256) takes form 0, 247, where the 2048 alone take form 2, 66. */
    const int64_t two = (subs + 1) / 2 * pairs;
    const int form = (subs + 3) / 4 * pairs >= 2 * ctx->num_cus                                           ? 0
                     : (D == 64 || two <= (D == 128 ? 1 : 2) * ctx->num_cus) && max_k > NMOE_PR_SHORT     ? 2
                     : D != 64 && max_k >= NMOE_PR_SPLIT * nmoe_pr_keys<D>                                ? 1
                                                                                                          : 0;
    const int pieces = form == 2 ? 2 : 4;
    int64_t tiles = (subs + pieces - 1) / pieces;
    if (tiles * pairs > NMOE_MAX_ROWS) tiles = NMOE_MAX_ROWS / pairs; /* the blocks go on to further tiles */
    const dim3 g((uint32_t)(tiles * pairs));
    if (form == 0)
        hipLaunchKernelGGL((nmoe_attn_prompt_kernel<T, D, 4, 1>), g, dim3(256), 0, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k,
                           causal, c, q_and, q_xor, (T *)out, lse);
    else if (form == 2)
        hipLaunchKernelGGL((nmoe_attn_prompt_kernel<T, D, 2, 2>), g, dim3(256), 0, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k,
                           causal, c, q_and, q_xor, (T *)out, lse);
    else if constexpr (D != 64)
        hipLaunchKernelGGL((nmoe_attn_prompt_kernel<T, D, 4, 2>), g, dim3(512), 0, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k,
                           causal, c, q_and, q_xor, (T *)out, lse);
}

template <typename T>
static void nmoe_pr_launch(nmoe_hip_ctx *ctx, hipStream_t s, const nmoe_hip_qkv &r, int nseq, const int32_t *cu_q,
                           const int32_t *cu_k, int ntok_q, int ntok_k, int max_q, int max_k, int causal, float scale,
                           void *out, float *lse) {
    if (r.head_dim == 64)
        nmoe_pr_launch_as<T, 64>(ctx, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, max_k, causal, scale, out, lse);
    else if (r.head_dim == 128)
        nmoe_pr_launch_as<T, 128>(ctx, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, max_k, causal, scale, out, lse);
    else
        nmoe_pr_launch_as<T, 256>(ctx, s, r, nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, max_k, causal, scale, out, lse);
}

extern "C" int nmoe_attn_prompt(nmoe_hip_ctx *ctx, const nmoe_hip_qkv *rows, int nseq, const int32_t *cu_q,
                                const int32_t *cu_k, int ntok_q, int ntok_k, int max_q, int max_k, int causal,
                                float scale, void *out, float *lse, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_check_rows(ctx, rows, 1);
    if (rc != NMOE_HIP_OK) return rc;
    if (!nmoe_is_half(rows->dtype)) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: dtype %d is neither bf16 nor f16", rows->dtype);
    if (rows->k_stride >= NMOE_PR_STRIDE || rows->v_stride >= NMOE_PR_STRIDE)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: token strides of k and v are below %d elements", NMOE_PR_STRIDE);
    if (cu_q == NULL || out == NULL || !nmoe_aligned(out, 16) || !nmoe_aligned(cu_q, 4) || !nmoe_aligned(cu_k, 4) ||
        !nmoe_aligned(lse, 4))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: cu_q and out (16-byte aligned) are required");
    if (nseq < 0 || (int64_t)nseq * rows->q_heads > NMOE_MAX_ROWS || ntok_q < 0 || ntok_k < 0 || ntok_q > NMOE_PR_TOKENS ||
        ntok_k > NMOE_PR_TOKENS || max_q < 0 || max_k < 0 || !nmoe_scale_ok(scale))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: %d sequences of %d heads outside 0..2^22, a size that is negative or "
                                               "above 2^30, or a scale not below 2^127", nseq, rows->q_heads);
    if (nseq == 0 || ntok_q == 0) return NMOE_HIP_OK;
    if (max_q < 1) max_q = 1;
    if (max_q > ntok_q) max_q = ntok_q;
    if (cu_k == NULL) cu_k = cu_q;
    if (max_k > ntok_k) max_k = ntok_k;
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (rows->dtype == NMOE_HIP_BF16)
        nmoe_pr_launch<nmoe_bf16>(ctx, s, *rows, nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, max_k, causal, scale, out, lse);
    else
        nmoe_pr_launch<_Float16>(ctx, s, *rows, nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, max_k, causal, scale, out, lse);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
