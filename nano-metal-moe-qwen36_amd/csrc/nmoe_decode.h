/*
 * nmoe_decode.h -- what decode attention has alike over a cache in 16 bits
 * (attn_decode.hip) and in 8 (attn8_decode.hip): how sequences are cut into
 * parts, and how the parts are joined.
 */
#ifndef NMOE_DECODE_H
#define NMOE_DECODE_H

#include "nmoe_context.h"

#define NMOE_DEC_WAVES 4
#define NMOE_DEC_TILE 32                              /* keys of a wavefront's step */
#define NMOE_DEC_STEP (NMOE_DEC_WAVES * NMOE_DEC_TILE) /* keys of a block's step; parts are multiples of it */
#define NMOE_DEC_HEADS 16                             /* query heads of a block */
#define NMOE_DEC_PARTS 512                            /* most parts of a sequence */
#define NMOE_DEC_JOIN 256
#define NMOE_DEC_LONGEST (1 << 30) /* keys of a sequence: leaves room in 32 bits for a step past the end */

/* How a sequence of len keys is cut: `per` keys a part (the call's, or as
 * many as the call's number of parts needs when max_len was too small). */
__device__ __forceinline__ int nmoe_dec_per(int len, int per, int parts) {
    const int64_t need = ((int64_t)len + parts - 1) / parts;
    return need <= per ? per : (int)((need + NMOE_DEC_STEP - 1) / NMOE_DEC_STEP * NMOE_DEC_STEP);
}

/* A length the table's row can hold, else -1. */
__device__ __forceinline__ int nmoe_dec_len(const int32_t *lens, int b, int max_pages, int page_size) {
    const int len = max(lens[b], 0);
    return (int64_t)len > (int64_t)max_pages * page_size || len > NMOE_DEC_LONGEST ? -1 : len;
}

template <int N>
__device__ __forceinline__ void nmoe_dec_wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

/* Joins a head's parts: 256 / (D / 4) groups of threads take parts in turn,
 * 4 dimensions a thread. */
template <typename T, int D>
static __global__ void __launch_bounds__(NMOE_DEC_JOIN)
    nmoe_attn_join_kernel(int q_heads, const int32_t *seq_lens, int max_pages, int page_size, int parts, int per,
                          const float *part_o, const float *part_ml, T *out, float *lse) {
    constexpr int LANES = D / 4, GROUPS = NMOE_DEC_JOIN / LANES;
    __shared__ float s_a[NMOE_DEC_PARTS];
    __shared__ nmoe_f4 s_y[GROUPS][LANES];
    __shared__ float s_l[NMOE_DEC_JOIN / 64], s_m[NMOE_DEC_JOIN / 64];
    const int tid = threadIdx.x, b = blockIdx.x / q_heads, g = tid / LANES, d = tid % LANES;
    const int64_t oh = blockIdx.x;
    const float *ml = part_ml + 2 * oh * parts, *po = part_o + oh * parts * D + 4 * d;
    /* the first of each thread's beside the length, whether they turn out to be there or not */
    const float m0 = ml[2 * min(tid, parts - 1)], l0 = ml[2 * min(tid, parts - 1) + 1];
    const nmoe_f4 y0 = *(const nmoe_f4 *)(po + (int64_t)min(g, parts - 1) * D);
    const int len = nmoe_dec_len(seq_lens, b, max_pages, page_size);
    per = nmoe_dec_per(max(len, 0), per, parts);
    if (len <= per) return; /* written by its one part */
    const int n = (int)(((int64_t)len + per - 1) / per);
    float m = tid < n ? m0 : -INFINITY, l = 0.0f;
    for (int i = tid + NMOE_DEC_JOIN; i < n; i += NMOE_DEC_JOIN) m = fmaxf(m, ml[2 * i]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) m = fmaxf(m, __shfl_xor(m, x, 64));
    if (tid % 64 == 0) s_m[tid / 64] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NMOE_DEC_JOIN / 64; i++) m = fmaxf(m, s_m[i]);
    for (int i = tid; i < n; i += NMOE_DEC_JOIN) {
        s_a[i] = nmoe_exp2((i == tid ? m0 : ml[2 * i]) - m);
        l += s_a[i] * (i == tid ? l0 : ml[2 * i + 1]);
    }
    l = nmoe_wave_sum_tree(l);
    if (tid % 64 == 0) s_l[tid / 64] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < NMOE_DEC_JOIN / 64; i++) l += s_l[i];
    nmoe_f4 y = {0, 0, 0, 0};
    if (g < n) y = s_a[g] * y0;
#pragma unroll 4
    for (int i = g + GROUPS; i < n; i += GROUPS) y += s_a[i] * *(const nmoe_f4 *)(po + (int64_t)i * D);
    s_y[g][d] = y;
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int i = 1; i < GROUPS; i++) y += s_y[i][d];
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; i++) z[i] = y[i] / l;
    nmoe_store<T, 4>(out + oh * D + 4 * d, z);
    if (lse != NULL && d == 0) lse[oh] = 0.69314718055994531f * (m + log2f(l));
}

/* The calls' cut: `want` workgroups in all, as many as run at once. */
struct nmoe_dec_plan {
    int tiles, parts, per;
    size_t rows; /* partial rows */
};

static inline int nmoe_dec_tiles(int kv_heads, int q_heads) {
    return (q_heads / kv_heads + NMOE_DEC_HEADS - 1) / NMOE_DEC_HEADS;
}

static inline nmoe_dec_plan nmoe_dec_plan_of(int64_t want, int kv_heads, int q_heads, int nseq, int64_t max_len) {
    nmoe_dec_plan p;
    p.tiles = nmoe_dec_tiles(kv_heads, q_heads);
    const int64_t blocks = (int64_t)nseq * kv_heads * p.tiles;
    if (max_len > NMOE_DEC_LONGEST) max_len = NMOE_DEC_LONGEST;
    int64_t parts = blocks >= want ? 1 : (want + blocks - 1) / blocks;
    if (parts > NMOE_DEC_PARTS) parts = NMOE_DEC_PARTS;
    int64_t per = (max_len + parts - 1) / parts;
    per = (per + NMOE_DEC_STEP - 1) / NMOE_DEC_STEP * NMOE_DEC_STEP;
    if (per < NMOE_DEC_STEP) per = NMOE_DEC_STEP;
    p.per = (int)per;
    p.parts = (int)((max_len + per - 1) / per);
    if (p.parts < 1) p.parts = 1;
    p.rows = p.parts > 1 ? (size_t)nseq * q_heads * p.parts : 0;
    return p;
}

/* Bytes that do for every plan of nseq sequences or fewer, of max_len keys or
 * fewer.  A plan's own need falls now and then where either grows (parts are
 * whole steps; from `want` blocks on there is one part).  With u blocks a
 * sequence, n sequences are cut where n u < want, into at most ceil(want / (n
 * u)), NMOE_DEC_PARTS or ceil(max_len / NMOE_DEC_STEP) parts each; and n
 * ceil(want / (n u)) <= n + (want - 1) / u, rounded down. */
static inline size_t nmoe_dec_ws_bytes(int64_t want, int kv_heads, int head_dim, int q_heads, int nseq, int64_t max_len) {
    const int64_t u = (int64_t)kv_heads * nmoe_dec_tiles(kv_heads, q_heads);
    int64_t n = (want + u - 1) / u - 1, most = (max_len + NMOE_DEC_STEP - 1) / NMOE_DEC_STEP;
    if (n > nseq) n = nseq;
    if (most > NMOE_DEC_PARTS) most = NMOE_DEC_PARTS;
    if (n < 1 || most < 2) return 0;
    const int64_t parts = n * most < n + (want - 1) / u ? n * most : n + (want - 1) / u;
    return (size_t)parts * q_heads * (head_dim + 2) * sizeof(float);
}

#endif
