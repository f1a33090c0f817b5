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
/* Blocks a CU.  Where there are more, a wavefront takes two heads of q, by whose
 * angles the second has none to wait for (heads of 256, 4100 tokens: 21.9 us, one
 * each 23.7; 6000: 26.1, 29.4; 8190, beyond what the last cache holds: 47.7, 45.3). */
#define NMOE_KV8_AT_ONCE 5
#define NMOE_KV8_TURNS 2
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
template <bool ROW>
__device__ __forceinline__ int64_t nmoe_kv8_first(int row, int b) {
    return ROW ? row : row / 16 + 2 * (int64_t)b;
}

struct nmoe_kv8_seq {
    int b, first_row, end_row, len;
};

/* The sequence that unit `slot` belongs to (ROW: that row `slot` does), with its offsets and length: among
 * the 63 around where it is if all are of one length, whose values come with
 * one load (of up to 63 sequences, any), else by 64 places at a time. */
template <bool ROW>
__device__ __forceinline__ nmoe_kv8_seq nmoe_kv8_find(const int32_t *cu, const int32_t *lens, int nseq, int ntok, int64_t slot,
                                                      int64_t slots) {
    const int lane = threadIdx.x % 64;
    const int guess = min(max((int)((float)slot / (float)slots * (float)nseq) - 31, 0), max(nseq - 63, 0));
    const int at = min(guess + lane, nseq), row = min(max(cu[at], 0), ntok), len = lens[min(at, nseq - 1)];
    const int near = (int)__popcll(__ballot(guess + lane < nseq && nmoe_kv8_first<ROW>(row, at) <= slot));
    if ((near > 0 && near < 64) || nseq == 1) {
        const int b = max(near - 1, 0);
        return {guess + b, __builtin_amdgcn_readlane(row, b), __builtin_amdgcn_readlane(row, b + 1), __builtin_amdgcn_readlane(len, b)};
    }
    int lo = 0, n = nseq;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lane * step;
        const uint64_t below = __ballot(i < n && nmoe_kv8_first<ROW>(min(max(cu[lo + min(i, n - 1)], 0), ntok), lo + i) <= slot);
        const int last = max((int)__popcll(below) - 1, 0) * step;
        lo += last;
        n = min(step, n - last);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    return {lo, min(max(cu[lo], 0), ntok), min(max(cu[lo + 1], 0), ntok), lens[lo]};
}

/* A lane's 8 elements of a row, as they are loaded: 4 from p + ea on and 4 from
 * p + eb.  Where pairs of the rotation are half a turn's dimensions apart, these
 * are 4 of its first half and their partners, so that it needs no exchange;
 * else they are neighbours. */
template <typename T>
struct nmoe_kv8_raw {
    nmoe_u4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void nmoe_kv8_ask(const T *p, int ea, int eb, nmoe_kv8_raw<T> &r) {
    if constexpr (sizeof(T) == 4) {
        r.w[0] = *(const nmoe_u4 *)(p + ea);
        r.w[1] = *(const nmoe_u4 *)(p + eb);
    } else {
        const uint2 a = *(const uint2 *)(p + ea), b = *(const uint2 *)(p + eb);
        r.w[0] = nmoe_u4{a.x, a.y, b.x, b.y};
    }
}

template <typename T>
__device__ __forceinline__ void nmoe_kv8_values(const nmoe_kv8_raw<T> &r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (sizeof(T) == 4)
            x[i] = __uint_as_float(r.w[i / 4][i % 4]);
        else if constexpr (nmoe_elem<T>::dtype == NMOE_HIP_BF16)
            x[i] = __uint_as_float(i % 2 ? r.w[0][i / 2] & 0xffff0000u : r.w[0][i / 2] << 16);
        else
            x[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(i % 2 ? r.w[0][i / 2] >> 16 : r.w[0][i / 2] & 0xffffu));
    }
}

template <typename C>
__device__ __forceinline__ void nmoe_kv8_put(C *p, int ea, int eb, const float (&x)[8]) {
    const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
    nmoe_store<C, 4>(p + ea, a);
    nmoe_store<C, 4>(p + eb, b);
}

/* Where a lane's two fours are: lane u of a row's. */
__device__ __forceinline__ void nmoe_kv8_places(const nmoe_hip_qk_prep &prep, int u, int &ea, int &eb) {
    const bool apart = !prep.interleaved && 8 * u < prep.rotary_dim;
    ea = apart ? 4 * u : 8 * u;
    eb = apart ? prep.rotary_dim / 2 + 4 * u : 8 * u + 4;
}

/* The sum of v over a row's LANES lanes. */
template <int LANES>
__device__ __forceinline__ float nmoe_kv8_row_sum(float v) {
    v = nmoe_dpp_group_sum<LANES == 8 ? 8 : 16>(v);
    if (LANES == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

/* Norm and rotation of a row, by angles c and s of its pairs. */
template <int LANES>
__device__ __forceinline__ void nmoe_kv8_prepare(float (&x)[8], const float (&w)[8], const nmoe_hip_qk_prep &prep, bool turns,
                                                 const float *c, const float *s) {
    if (prep.qk_norm) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss += x[i] * x[i];
        const float inv = rsqrtf(nmoe_kv8_row_sum<LANES>(ss) / (float)(8 * LANES) + prep.eps);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] *= inv * w[i];
    }
    if (!turns) return;
    const nmoe_f4 c4 = *(const nmoe_f4 *)c, s4 = *(const nmoe_f4 *)s;
    if (prep.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = fmaf(a, c4[i], -b * s4[i]);
            x[2 * i + 1] = fmaf(b, c4[i], a * s4[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float a = x[i], b = x[i + 4];
            x[i] = fmaf(a, c4[i], -b * s4[i]);
            x[i + 4] = fmaf(b, c4[i], a * s4[i]);
        }
    }
}

/* The norm's weights of a lane's elements. */
__device__ __forceinline__ void nmoe_kv8_weights(const uint16_t *norm, const nmoe_hip_qk_prep &prep, int ea, int eb, float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = 1.0f;
    if (!prep.qk_norm || norm == NULL) return;
    nmoe_kv8_raw<nmoe_bf16> r;
    nmoe_kv8_ask((const nmoe_bf16 *)norm, ea, eb, r);
    nmoe_kv8_values(r, w);
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] += prep.add_one ? 1.0f : 0.0f;
}

/* A block of 4 wavefronts: 16 tokens, a wavefront a head of q, k or v.  A
 * row is held by D / 8 lanes, 8 elements each; a wavefront goes over its head's
 * new rows a step of 512 / D at a time, the next one under way.  Keys and values
 * take two turns: one for their largest magnitude, one, back again, for their
 * codes (rows come from the cache then, and are prepared again): held in
 * registers, 16 rows left room for two wavefronts a SIMD instead of eight, and
 * 4097 tokens took 35 us.  The first rows, page and stored scale are asked for
 * before the angles, which the wavefronts compute together meanwhile.
 *
 * It is bound by memory: 4097 tokens of 16 + 2 heads of 256 (bf16, 80 MB) take
 * 20.4 us, 3.9 TB/s, half of it writes; the same loads and stores with nothing
 * between them 17.
 *
 * SPLIT: a block a head, whose steps the wavefronts share, which is for calls
 * that are as long as one block takes (100 tokens in 4 sequences: 7.2 us instead
 * of 12.1; 700: 9.9, 12.9; with blocks beyond those that run at once, 3000: 21.6
 * instead of 18.8). */
template <typename T, typename C, int D, bool SPLIT>
__global__ void __launch_bounds__(NMOE_KV8_THREADS, 5)
    nmoe_kv8_append_kernel(nmoe_hip_qkv rows, nmoe_hip_kv8_cache cache, nmoe_hip_qk_prep prep, int nseq,
                           const int32_t *cu, int ntok, const int32_t *seq_lens, const int32_t *page_table, int max_pages,
                           const int32_t *positions, C *q_out, int64_t slots, int parts, int per, int q_parts) {
    constexpr int LANES = D / 8, R = 64 / LANES;
    constexpr int HEADS = SPLIT ? 1 : NMOE_KV8_WAVES, STEPS = SPLIT ? (16 / R + NMOE_KV8_WAVES - 1) / NMOE_KV8_WAVES : 16 / R;
    __shared__ alignas(16) float s_cos[16][D / 2], s_sin[16][D / 2];
    __shared__ float s_most[2][NMOE_KV8_WAVES];
    const int tid = threadIdx.x, lane = tid % 64, half = prep.rotary_dim / 2, f0 = lane % LANES * 4; /* the lane's pairs */
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int qh = q_out != NULL ? rows.q_heads : 0, all = qh + 2 * rows.kv_heads;
    const bool turns = 2 * f0 < prep.rotary_dim;
    int ea, eb;
    nmoe_kv8_places(prep, lane % LANES, ea, eb);
    for (int64_t unit = blockIdx.x; unit < slots * parts; unit += gridDim.x) {
        const int64_t slot = unit / parts;
        const nmoe_kv8_seq seq = nmoe_kv8_find<false>(cu, seq_lens, nseq, ntok, slot, slots);
        const int b = seq.b, t0 = seq.first_row, n = max(seq.end_row - t0, 0), len = seq.len;
        const bool bad = len < n || nmoe_len_of(len, max_pages, cache.page_size) < 0;
        const int begin = bad ? 0 : len - n; /* tokens before these */
        const int64_t first = nmoe_kv8_first<false>(t0, b), block = slot - first + begin / 16;
        if (n == 0 || slot < first || block * 16 >= (int64_t)begin + n) continue; /* the whole workgroup */
        const int at = (int)block * 16, lo = max(begin - at, 0), hi = min(begin + n - at, 16); /* places of new tokens */
        const int token = t0 + at - begin; /* row of place 0 */
        const int page = bad ? -1 : page_table[(int64_t)b * max_pages + at / cache.page_size], place = at % cache.page_size;
        /* the heads of q, `per` a workgroup, then those of k and v, one a wavefront: they take two turns */
        const int part = (int)(unit % parts), lead = part < q_parts ? part * per : qh + (part - q_parts) * HEADS;
        const int tile0 = SPLIT ? lead : lead + wave, tiles = part < q_parts ? min(lead + per, qh) : min(lead + HEADS, all);
        for (int tile = tile0; tile < tiles || tile == tile0; tile += HEADS) {
        const int there = min(tile, tiles - 1); /* without a tile: the last one */
        const int kind = there < qh ? 0 : there < qh + rows.kv_heads ? 1 : 2;
        const int head = kind == 0 ? there : kind == 1 ? there - qh : there - qh - rows.kv_heads;
        const int s0 = SPLIT ? max(lo / R, wave * STEPS) : lo / R; /* the wavefront's steps with new rows */
        const int s1 = SPLIT ? min((hi - 1) / R, wave * STEPS + STEPS - 1) : (hi - 1) / R;
        const int64_t stride = kind == 0 ? rows.q_stride : kind == 1 ? rows.k_stride : rows.v_stride;
        const T *const src = (const T *)(kind == 0 ? rows.q : kind == 1 ? rows.k : rows.v) +
                             head * (kind == 0 ? rows.q_head_stride : kind == 1 ? rows.k_head_stride : rows.v_head_stride);
        auto ask = [&](int s, nmoe_kv8_raw<T> &r) { /* beside the new rows: one of them */
            nmoe_kv8_ask(src + (token + min(max(s * R + lane / LANES, lo), hi - 1)) * stride, ea, eb, r);
        };
        nmoe_kv8_raw<T> raw;
        ask(s0, raw);
        const bool keep = tile < tiles && kind != 0 && page >= 0 && page < cache.num_pages;
        float *const scale = (kind == 1 ? cache.k_scale : cache.v_scale) + nmoe_kv8_scale_at(cache, keep ? page : 0, place, head);
        float stored = 0.0f;
        if (keep && lo > 0) stored = *scale;
        float w[8];
        nmoe_kv8_weights(kind == 0 ? prep.q_norm : prep.k_norm, prep, ea, eb, w);
        if (half != 0 && tile == tile0) {
            for (int i = tid; i < 16 * half; i += NMOE_KV8_THREADS) {
                const int p = i / half, f = i - p * half;
                if (p >= lo && p < hi)
                    nmoe_turn(positions != NULL ? positions[token + p] : at + p, prep.inv_freq[f], s_cos[p][f], s_sin[p][f]);
            }
            __syncthreads();
        }
        auto prepare = [&](float (&x)[8], int s) {
            const int p = s * R + lane / LANES;
            nmoe_kv8_prepare<LANES>(x, w, prep, turns, &s_cos[p][f0], &s_sin[p][f0]);
        };
        if (kind == 0 && tile < tiles) {
#pragma unroll 1
            for (int s = s0; s <= s1; s++) {
                nmoe_kv8_raw<T> next = raw;
                if (s < s1) ask(s + 1, next);
                float x[8];
                nmoe_kv8_values<T>(raw, x);
                prepare(x, s);
                const int p = s * R + lane / LANES;
                if (bad) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = NAN;
                }
                if (p >= lo && p < hi) nmoe_kv8_put(q_out + ((int64_t)(token + p) * rows.q_heads + head) * D, ea, eb, x);
                raw = next;
            }
        } else if (keep) {
            float x[8], amax = 0.0f, finite = 0.0f;
#pragma unroll 1
            for (int s = s0; s <= s1; s++) {
                nmoe_kv8_raw<T> next = raw;
                if (s < s1) ask(s + 1, next);
                nmoe_kv8_values<T>(raw, x);
                if (kind == 1) prepare(x, s);
                const int p = s * R + lane / LANES;
                if (p >= lo && p < hi) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float y = fabsf(x[i]);
                        amax = fmaxf(amax, y); /* a NaN is not the larger one */
                        finite = fmaxf(finite, y < INFINITY ? y : 0.0f);
                    }
                }
                raw = next;
            }
            amax = nmoe_wave_max_f(amax);
            finite = nmoe_wave_max_f(finite);
            if constexpr (SPLIT) {
                if (lane == 0) {
                    s_most[0][wave] = amax;
                    s_most[1][wave] = finite;
                }
                __syncthreads(); /* and the scale has been read */
#pragma unroll
                for (int i = 0; i < NMOE_KV8_WAVES; i++) {
                    amax = fmaxf(amax, s_most[0][i]);
                    finite = fmaxf(finite, s_most[1][i]);
                }
            }
            const bool odd = !(amax < 448.0f * nmoe_kv8_two_to(NMOE_KV8_HIGH)); /* infinities, or beyond the largest scale */
            int e = nmoe_kv8_power(finite);
            uint8_t *const dst = (uint8_t *)(kind == 1 ? cache.k : cache.v) + page * cache.page_stride +
                                 place * cache.token_stride + head * cache.head_stride;
            if (lo > 0) { /* older tokens in the block */
                const int was = min(max((int)(__float_as_uint(stored) >> 23 & 255u) - 127, NMOE_KV8_LOW), NMOE_KV8_HIGH);
                if (was < e) {
                    const float f = nmoe_kv8_two_to(max(was - e, -126));
                    for (int p = lane / LANES + (SPLIT ? wave * R : 0); p < lo; p += SPLIT ? NMOE_KV8_WAVES * R : R) {
                        uint32_t *const c = (uint32_t *)(dst + p * cache.token_stride);
                        c[ea / 4] = nmoe_kv8_again(c[ea / 4], f);
                        c[eb / 4] = nmoe_kv8_again(c[eb / 4], f);
                    }
                }
                e = max(e, was);
            }
            const float inv = nmoe_kv8_two_to(-e);
#pragma unroll 1
            for (int s = s1; s >= s0; s--) { /* the last step's are still there */
                nmoe_kv8_raw<T> next = raw;
                if (s > s0) ask(s - 1, next);
                const uint2 c = odd ? uint2{nmoe_kv8_codes_of_any(&x[0], inv), nmoe_kv8_codes_of_any(&x[4], inv)}
                                    : uint2{nmoe_kv8_codes(&x[0], inv), nmoe_kv8_codes(&x[4], inv)};
                const int p = s * R + lane / LANES;
                if (p >= lo && p < hi) {
                    *(uint32_t *)(dst + p * cache.token_stride + ea) = c.x;
                    *(uint32_t *)(dst + p * cache.token_stride + eb) = c.y;
                }
                if (s > s0) {
                    nmoe_kv8_values<T>(next, x);
                    if (kind == 1) prepare(x, s - 1);
                }
            }
            if (lane == 0 && (!SPLIT || wave == 0)) *scale = nmoe_kv8_two_to(e);
        }
        }
        if (half != 0 || SPLIT) __syncthreads(); /* the angles and maxima are read */
    }
}

/* The largest of a row's D / 8 lanes. */
template <int LANES>
__device__ __forceinline__ float nmoe_kv8_row_max(float v) {
    v = fmaxf(v, nmoe_dpp_f<NMOE_DPP_XOR1>(v));
    v = fmaxf(v, nmoe_dpp_f<NMOE_DPP_XOR2>(v));
    v = fmaxf(v, nmoe_dpp_f<NMOE_DPP_HALF_MIRROR>(v));
    if (LANES >= 16) v = fmaxf(v, nmoe_dpp_f<NMOE_DPP_MIRROR>(v));
    if (LANES >= 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
    return v;
}

/* The form for about a token a sequence: a block a token and as many of its
 * rows (heads of q, k and v) as it has lanes for, all at once.  A block of
 * the cache with more new tokens is its first one's.  It is one chain: row and
 * offsets, length, page, stored scale, older codes (200 sequences of a token,
 * 16 + 2 heads of 256: 6.2 us, by blocks of 16 tokens 9.6; 1000: 12.1, 24.0). */
template <typename T, typename C, int D>
__global__ void __launch_bounds__(NMOE_KV8_THREADS)
    nmoe_kv8_token_kernel(nmoe_hip_qkv rows, nmoe_hip_kv8_cache cache, nmoe_hip_qk_prep prep, int nseq, const int32_t *cu,
                          int ntok, const int32_t *seq_lens, const int32_t *page_table, int max_pages,
                          const int32_t *positions, C *q_out, int parts) {
    constexpr int LANES = D / 8, ROWS = NMOE_KV8_THREADS / LANES;
    __shared__ alignas(16) float s_cos[D / 2], s_sin[D / 2];
    const int tid = threadIdx.x, lane = tid % 64, half = prep.rotary_dim / 2, f0 = lane % LANES * 4;
    const int qh = q_out != NULL ? rows.q_heads : 0, all = qh + 2 * rows.kv_heads;
    int ea, eb;
    nmoe_kv8_places(prep, lane % LANES, ea, eb);
    const int t = blockIdx.x / parts, r = blockIdx.x % parts * ROWS + tid / LANES, row = min(r, all - 1);
    const int kind = row < qh ? 0 : row < qh + rows.kv_heads ? 1 : 2;
    const int head = kind == 0 ? row : kind == 1 ? row - qh : row - qh - rows.kv_heads;
    const int64_t stride = kind == 0 ? rows.q_stride : kind == 1 ? rows.k_stride : rows.v_stride;
    const T *const src = (const T *)(kind == 0 ? rows.q : kind == 1 ? rows.k : rows.v) +
                         head * (kind == 0 ? rows.q_head_stride : kind == 1 ? rows.k_head_stride : rows.v_head_stride);
    nmoe_kv8_raw<T> raw;
    nmoe_kv8_ask(src + t * stride, ea, eb, raw);
    const float freq = tid < half ? prep.inv_freq[tid] : 0.0f;
    float w[8];
    nmoe_kv8_weights(kind == 0 ? prep.q_norm : prep.k_norm, prep, ea, eb, w);
    const nmoe_kv8_seq seq = nmoe_kv8_find<true>(cu, seq_lens, nseq, ntok, t, ntok);
    const int b = seq.b, t0 = seq.first_row, n = max(seq.end_row - t0, 0), len = seq.len;
    if (t < t0 || t >= t0 + n) return; /* of no sequence: the whole workgroup */
    const bool bad = len < n || nmoe_len_of(len, max_pages, cache.page_size) < 0;
    const int j = bad ? t - t0 : len - n + (t - t0), at = j / 16 * 16, lo = j - at; /* its place in the sequence, its block */
    const bool leads = t == t0 || lo == 0;
    const int more = leads ? min(16 - lo, t0 + n - t) : 0; /* new tokens of the block, where they are this one's */
    const int page = bad ? -1 : page_table[(int64_t)b * max_pages + at / cache.page_size], place = at % cache.page_size;
    const bool keep = r < all && kind != 0 && more > 0 && page >= 0 && page < cache.num_pages;
    float *const scale = (kind == 1 ? cache.k_scale : cache.v_scale) + nmoe_kv8_scale_at(cache, keep ? page : 0, place, head);
    const float stored = keep && lo > 0 ? *scale : 0.0f;
    float x[8];
    /* token t + i's row, normalised and rotated; for all of the workgroup */
    auto prepare = [&](int i) {
        if (half != 0) {
            if (i != 0) __syncthreads(); /* the last one's angles are read */
            if (tid < half) nmoe_turn(positions != NULL ? positions[t + i] : j + i, freq, s_cos[tid], s_sin[tid]);
            __syncthreads();
        }
        nmoe_kv8_values<T>(raw, x);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = x[e];
        nmoe_kv8_prepare<LANES>(y, w, prep, 2 * f0 < prep.rotary_dim, s_cos + f0, s_sin + f0);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = kind == 2 ? x[e] : y[e];
    };
    float amax = 0.0f, finite = 0.0f;
    auto largest = [&]() {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = fabsf(x[e]);
            amax = fmaxf(amax, y); /* a NaN is not the larger one */
            finite = fmaxf(finite, y < INFINITY ? y : 0.0f);
        }
    };
    prepare(0);
    if (kind == 0 && r < all) {
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = bad ? NAN : x[e];
        nmoe_kv8_put(q_out + ((int64_t)t * rows.q_heads + head) * D, ea, eb, z);
    }
    if (more == 0) return;
    largest();
    for (int i = 1; i < more; i++) {
        nmoe_kv8_ask(src + (t + i) * stride, ea, eb, raw);
        prepare(i);
        largest();
    }
    amax = nmoe_kv8_row_max<LANES>(amax);
    finite = nmoe_kv8_row_max<LANES>(finite);
    const bool odd = !(amax < 448.0f * nmoe_kv8_two_to(NMOE_KV8_HIGH)); /* infinities, or beyond the largest scale */
    uint8_t *const dst = (uint8_t *)(kind == 1 ? cache.k : cache.v) + (keep ? page : 0) * cache.page_stride +
                         place * cache.token_stride + head * cache.head_stride;
    int power = nmoe_kv8_power(finite);
    if (keep && lo > 0) { /* older tokens in the block */
        const int was = min(max((int)(__float_as_uint(stored) >> 23 & 255u) - 127, NMOE_KV8_LOW), NMOE_KV8_HIGH);
        if (was < power) {
            const float f = nmoe_kv8_two_to(max(was - power, -126));
#pragma unroll 4
            for (int p = 0; p < lo; p++) {
                uint32_t *const c = (uint32_t *)(dst + p * cache.token_stride);
                c[ea / 4] = nmoe_kv8_again(c[ea / 4], f);
                c[eb / 4] = nmoe_kv8_again(c[eb / 4], f);
            }
        }
        power = max(power, was);
    }
    const float inv = nmoe_kv8_two_to(-power);
    for (int i = more - 1; i >= 0; i--) { /* the last one's are still there */
        const uint2 c = odd ? uint2{nmoe_kv8_codes_of_any(&x[0], inv), nmoe_kv8_codes_of_any(&x[4], inv)}
                            : uint2{nmoe_kv8_codes(&x[0], inv), nmoe_kv8_codes(&x[4], inv)};
        if (keep) {
            *(uint32_t *)(dst + (lo + i) * cache.token_stride + ea) = c.x;
            *(uint32_t *)(dst + (lo + i) * cache.token_stride + eb) = c.y;
        }
        if (i > 0) {
            nmoe_kv8_ask(src + (t + i - 1) * stride, ea, eb, raw);
            if (half != 0 && i == 1) __syncthreads();
            prepare(i - 1);
        }
    }
    if (keep && lane % LANES == 0) *scale = nmoe_kv8_two_to(power);
}

template <typename T, typename C, int D>
static void nmoe_kv8_launch_as(hipStream_t s, const nmoe_hip_qkv &r, const nmoe_hip_kv8_cache &c, const nmoe_hip_qk_prep &p,
                               int nseq, const int32_t *cu, int ntok, const int32_t *lens, const int32_t *table, int max_pages,
                               const int32_t *positions, int num_cus, void *q_out) {
    const int all = (q_out != NULL ? r.q_heads : 0) + 2 * r.kv_heads;
    const int wide = (all + NMOE_KV8_THREADS / (D / 8) - 1) / (NMOE_KV8_THREADS / (D / 8));
    if (ntok <= nseq && (int64_t)ntok * wide <= NMOE_KV8_UNITS) {
        hipLaunchKernelGGL((nmoe_kv8_token_kernel<T, C, D>), dim3((uint32_t)(ntok * wide)), dim3(NMOE_KV8_THREADS), 0, s, r, c, p,
                           nseq, cu, ntok, lens, table, max_pages, positions, (C *)q_out, wide);
        return;
    }
    const int64_t slots = ntok / 16 + 2 * (int64_t)nseq, at_once = NMOE_KV8_AT_ONCE * (int64_t)(num_cus > 0 ? num_cus : 256);
    const int q = all - 2 * r.kv_heads;
    /* heads of 64 leave half of the wavefronts without a step: 700 tokens on 8 + 8 of them 9.1 us instead of 7.9 */
    const bool split = slots * all * 128 <= at_once * D;
    const int heads = split ? 1 : NMOE_KV8_WAVES, kv_parts = (2 * r.kv_heads + heads - 1) / heads;
    int q_parts = (q + heads - 1) / heads;
    if (slots * (q_parts + kv_parts) > at_once) q_parts = (q_parts + NMOE_KV8_TURNS - 1) / NMOE_KV8_TURNS;
    const int parts = q_parts + kv_parts, per = q_parts > 0 ? (q + q_parts - 1) / q_parts : 0;
    const int64_t units = slots * parts;
    const dim3 grid((uint32_t)(units < NMOE_KV8_UNITS ? units : NMOE_KV8_UNITS));
    if (split)
        hipLaunchKernelGGL((nmoe_kv8_append_kernel<T, C, D, true>), grid, dim3(NMOE_KV8_THREADS), 0, s, r, c, p, nseq, cu, ntok, lens,
                           table, max_pages, positions, (C *)q_out, slots, parts, per, q_parts);
    else
        hipLaunchKernelGGL((nmoe_kv8_append_kernel<T, C, D, false>), grid, dim3(NMOE_KV8_THREADS), 0, s, r, c, p, nseq, cu, ntok, lens,
                           table, max_pages, positions, (C *)q_out, slots, parts, per, q_parts);
}

template <typename T, typename C>
static void nmoe_kv8_launch(hipStream_t s, const nmoe_hip_qkv &r, const nmoe_hip_kv8_cache &c, const nmoe_hip_qk_prep &p,
                            int nseq, const int32_t *cu, int ntok, const int32_t *lens, const int32_t *table, int max_pages,
                            const int32_t *positions, int num_cus, void *q_out) {
    if (c.head_dim == 64)
        nmoe_kv8_launch_as<T, C, 64>(s, r, c, p, nseq, cu, ntok, lens, table, max_pages, positions, num_cus, q_out);
    else if (c.head_dim == 128)
        nmoe_kv8_launch_as<T, C, 128>(s, r, c, p, nseq, cu, ntok, lens, table, max_pages, positions, num_cus, q_out);
    else
        nmoe_kv8_launch_as<T, C, 256>(s, r, c, p, nseq, cu, ntok, lens, table, max_pages, positions, num_cus, q_out);
}

template <typename T>
static void nmoe_kv8_launch_from(hipStream_t s, const nmoe_hip_qkv &r, const nmoe_hip_kv8_cache &c, const nmoe_hip_qk_prep &p,
                                 int nseq, const int32_t *cu, int ntok, const int32_t *lens, const int32_t *table,
                                 int max_pages, const int32_t *positions, int num_cus, void *q_out, int q_dtype) {
    if (q_dtype == NMOE_HIP_BF16)
        nmoe_kv8_launch<T, nmoe_bf16>(s, r, c, p, nseq, cu, ntok, lens, table, max_pages, positions, num_cus, q_out);
    else
        nmoe_kv8_launch<T, _Float16>(s, r, c, p, nseq, cu, ntok, lens, table, max_pages, positions, num_cus, q_out);
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
        nmoe_kv8_launch_from<float>(s, *rows, *cache, p, nseq, cu, ntok, seq_lens, page_table, max_pages, positions, ctx->num_cus,
                                        q_out, q_dtype);
    else if (rows->dtype == NMOE_HIP_BF16)
        nmoe_kv8_launch_from<nmoe_bf16>(s, *rows, *cache, p, nseq, cu, ntok, seq_lens, page_table, max_pages, positions, ctx->num_cus,
                                        q_out, q_dtype);
    else
        nmoe_kv8_launch_from<_Float16>(s, *rows, *cache, p, nseq, cu, ntok, seq_lens, page_table, max_pages, positions, ctx->num_cus,
                                        q_out, q_dtype);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
