/*
 * attn_decode.hip -- attention of one new token a sequence over a paged
 * key-value cache (nmoe_attn_decode).
 *
 * out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q.k_j - m): one pass
 * over keys and values with a running maximum m and sum, so a sequence can be
 * cut anywhere and the parts joined afterwards:
 *   m = max m_s,  l = sum l_s 2^(m_s - m),  o = sum o_s 2^(m_s - m)
 * (in powers of two: scale * log2(e) is one factor).
 *
 * It is bound by the bytes of the cache: a key and a value of D elements are
 * 4 D bytes for 4 D flops a query head.  A group of query heads on one key
 * head shares them, and on the vector units eight such heads would already
 * cost more than the bytes; so the group's heads are the 16 columns of the
 * matrix instructions (16x16x32), whatever part of them is used.
 */
#include <type_traits>

#include "nmoe_decode.h"

#define NMOE_DEC_STRIDE (1 << 24) /* 16 tokens' offsets stay below 2^31 bytes */
#define NMOE_DEC_NT 2 /* cache policy: read once (nt) */
#define NMOE_DEC_PARTS 512                            /* most parts of a sequence */

/* f16 weights are held up to 2^12 instead of 1, so that those of 2^-26 and
 * more keep their 11 bits (f16 has them from 2^-14 on); bf16 needs no lift. */
template <typename T>
constexpr float nmoe_dec_lift = nmoe_elem<T>::dtype == NMOE_HIP_F16 ? 12.0f : 0.0f;

/* How a sequence of len keys is cut: `per` keys a part (the call's, or as
 * many as the call's number of parts needs when max_len was too small). */
__device__ __forceinline__ int nmoe_dec_per(int len, int per, int parts) {
    const int64_t need = ((int64_t)len + parts - 1) / parts;
    return need <= per ? per : (int)((need + NMOE_DEC_STEP - 1) / NMOE_DEC_STEP * NMOE_DEC_STEP);
}

/* The 16-byte chunks of a key's row are stored at chunk ^ f(row), so that 8
 * rows' same chunk lies in 8 different places of the banks (256 bytes wide: a
 * 128-byte row's neighbour is already in the other half). */
template <int D>
__device__ __forceinline__ int nmoe_dec_swizzle(int row) {
    return D == 64 ? (row >> 1) & 3 : row & 7;
}

/* One block a part of a sequence, a key head and up to 16 of its query
 * heads; its wavefronts take tiles of 32 keys in turn.
 *
 * Scores: S^T (keys x heads) = K Q^T.  As the row operand a lane has key l %
 * 16, so lanes side by side are different rows, and read so from memory the
 * pipeline takes one lane a cycle instead of four (64 sequences of 4096 on
 * heads of 256: 4.4 TB/s).  K's rows therefore go to LDS directly, whole rows
 * side by side, into a buffer of the wavefront's own: the next tile's when
 * this one's have been read.
 * A lane then holds, of its head l % 16, the scores of keys 16 a + 4 (l / 16)
 * + i (a < 2, i < 4): which is the order the second product takes its 32 keys
 * in, so the weights stay in the lane.  O^T (dimensions x heads) = V^T P^T
 * needs 8 keys of one dimension in a lane: lane (r, c) reads 16 bytes,
 * dimensions 8 r .., of its 8 keys (whole rows, 16 lanes side by side) and
 * takes the halves of the words apart; product dd has the dimensions 8 r + dd
 * as its rows.
 * Keys behind the end: their addresses are the last key's, their scores
 * -inf, their values zero.
 * 64 sequences of about 4096 (16 query heads on 2 of 256, bf16): 558 MB in 98
 * us, 5.7 TB/s; one of 131071, f16: 537 MB in 87 us, 6.2 TB/s; one of 777:
 * 9.4 us, two launches and the latency of a few dependent loads. */
template <typename T, int D>
__global__ void __launch_bounds__(64 * NMOE_DEC_WAVES, 2)
    nmoe_attn_decode_kernel(nmoe_hip_kv_cache cache, const T *q, int q_heads, int tiles, const int32_t *seq_lens,
                            const int32_t *page_table, int max_pages, int parts, int per, float scale2, T *out,
                            float *lse, float *part_o, float *part_ml) {
    typedef nmoe_mat<T> X;
    constexpr int KS = D / 32, VC = D >= 128 ? D / 128 : 1, DD = D >= 128 ? 8 : 4;
    constexpr int CH = D / 8, RPI = 64 / CH, NI = NMOE_DEC_TILE / RPI; /* chunks of a row, rows and loads of a tile of K */
    /* the wavefronts' tiles of K, in the end their outputs */
    __shared__ alignas(16) char s_kv[NMOE_DEC_WAVES * NMOE_DEC_TILE * D * 2 > NMOE_DEC_WAVES * NMOE_DEC_HEADS * D * 4
                                         ? NMOE_DEC_WAVES * NMOE_DEC_TILE * D * 2
                                         : NMOE_DEC_WAVES * NMOE_DEC_HEADS * D * 4];
    __shared__ float s_m[NMOE_DEC_WAVES][NMOE_DEC_HEADS], s_l[NMOE_DEC_WAVES][NMOE_DEC_HEADS];
    __shared__ int s_bad;
    float(*s_o)[NMOE_DEC_HEADS][D] = (float(*)[NMOE_DEC_HEADS][D])s_kv;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, c = lane / 16;
    const int part = blockIdx.x % parts, bk = blockIdx.x / parts, tile = bk % tiles;
    const int kh = bk / tiles % cache.kv_heads, b = bk / tiles / cache.kv_heads;
    const int group = q_heads / cache.kv_heads, h0 = kh * group + tile * NMOE_DEC_HEADS;
    const int heads = min(group - tile * NMOE_DEC_HEADS, NMOE_DEC_HEADS);
    /* the first tile's page numbers beside the length they depend on: where the part most likely begins */
    const int32_t *table = page_table + (int64_t)b * max_pages;
    const int64_t guess = (int64_t)part * per + w * NMOE_DEC_TILE;
    int early[2];
#pragma unroll
    for (int a = 0; a < 2; a++) {
        const uint32_t page = (uint32_t)min(guess + 16 * a, (int64_t)NMOE_LONGEST) / (uint32_t)cache.page_size;
        early[a] = table[min(page, (uint32_t)max_pages - 1)];
    }
    nmoe_u4 qf[KS];
    const T *qr = q + ((int64_t)b * q_heads + h0 + min(r, heads - 1)) * D + 8 * c;
#pragma unroll
    for (int k = 0; k < KS; k++) {
        qf[k] = *(const nmoe_u4 *)(qr + 32 * k);
        if (r >= heads) qf[k] = nmoe_u4{0, 0, 0, 0};
    }
    const int len = nmoe_len_of(seq_lens[b], max_pages, cache.page_size);
    per = nmoe_dec_per(max(len, 0), per, parts);
    const int64_t first = (int64_t)part * per;
    if (part != 0 && first >= len) return;
    const int begin = (int)first, end = (int)min((int64_t)max(len, 0), first + per);
    if (tid == 0) s_bad = len < 0;
    __syncthreads();

    nmoe_f4 o[VC][DD];
#pragma unroll
    for (int v = 0; v < VC; v++)
#pragma unroll
        for (int i = 0; i < DD; i++) o[v][i] = nmoe_f4{0, 0, 0, 0};
    float m = -3.402823466e38f, l = 0.0f; /* finite, so that a key whose score is -infinity weighs 0 also where no other is */
    bool bad = false;

    const T *kb = (const T *)cache.k + kh * cache.head_stride, *vb = (const T *)cache.v + kh * cache.head_stride;
    const uint32_t step = (uint32_t)cache.token_stride * 2; /* bytes from a key to the next of its page */
    const int last16 = end > begin ? (end - 1) & ~15 : 0;
    const int t0 = begin + w * NMOE_DEC_TILE;
    /* a tile lies in two halves of 16 keys, each in one page */
    auto page_of = [&](int t, int a) { return table[(uint32_t)min(t + 16 * a, last16) / (uint32_t)cache.page_size]; };
    auto row_of = [&](int t, int a, int page) {
        page = __builtin_amdgcn_readfirstlane(page);
        if ((uint32_t)page >= (uint32_t)cache.num_pages) {
            bad = true;
            page = 0;
        }
        return page * cache.page_stride +
               (int64_t)((uint32_t)min(t + 16 * a, last16) % (uint32_t)cache.page_size) * cache.token_stride;
    };
    auto top_of = [&](int t, int a) { return min(end - 1 - min(t + 16 * a, last16), 15); }; /* a half's last key */
    uint16_t *sk = (uint16_t *)s_kv + w * NMOE_DEC_TILE * D;
    const uint32_t chunk = (uint32_t)((lane % CH) ^ nmoe_dec_swizzle<D>(lane / CH)) * 16;
    auto load_k = [&](int t, const int64_t (&row)[2]) {
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const __amdgpu_buffer_rsrc_t k = nmoe_buffer(kb + row[a]);
            const int top = top_of(t, a);
#pragma unroll
            for (int i = 0; i < NI / 2; i++) {
                /* the swizzle goes by the row's last bits: the same for rows 8 apart */
                const int at = i * RPI + lane / CH;
                const uint32_t ch = RPI % 8 == 0 ? chunk : (uint32_t)((lane % CH) ^ nmoe_dec_swizzle<D>(at)) * 16;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(k, (__attribute__((address_space(3))) void *)(sk + (a * 16 + i * RPI) * D),
                                                         16, (int)((uint32_t)min(at, top) * step + ch), 0, 0, NMOE_DEC_NT);
            }
        }
    };
    int64_t row[2] = {0, 0};
    auto work = [&](const int t, auto last) {
        constexpr bool LAST = decltype(last)::value;
        int next[2];
        if (!LAST) {
#pragma unroll
            for (int a = 0; a < 2; a++) next[a] = page_of(t + NMOE_DEC_STEP, a);
        }
        asm volatile("" ::: "memory");
        nmoe_u4 vf[VC][8];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const __amdgpu_buffer_rsrc_t v = nmoe_buffer(vb + row[a]);
            const int top = top_of(t, a);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t at = (uint32_t)min(4 * c + i, top) * step;
#pragma unroll
                for (int x = 0; x < VC; x++) {
                    if constexpr (D >= 128)
                        vf[x][4 * a + i] = __builtin_amdgcn_raw_buffer_load_b128(v, (int)(at + 256 * x + 16 * r), 0, NMOE_DEC_NT);
                    else {
                        const auto y = __builtin_amdgcn_raw_buffer_load_b64(v, (int)(at + 8 * r), 0, NMOE_DEC_NT);
                        vf[x][4 * a + i] = nmoe_u4{y[0], y[1], 0, 0};
                    }
                }
            }
        }
        nmoe_dec_wait_vm<8 * VC>(); /* K has come, these values may be on their way */
        float s[8];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            nmoe_f4 x = {0, 0, 0, 0};
            const uint16_t *p = sk + (16 * a + r) * D;
            const int f = nmoe_dec_swizzle<D>(r);
#pragma unroll
            for (int k = 0; k < KS; k++) x = X::mma16(*(const nmoe_u4 *)(p + ((4 * k + c) ^ f) * 8), qf[k], x);
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * a + i] = x[i] * scale2;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (!LAST) {
#pragma unroll
            for (int a = 0; a < 2; a++) row[a] = row_of(t + NMOE_DEC_STEP, a, next[a]);
            load_k(t + NMOE_DEC_STEP, row);
        } else if (t + NMOE_DEC_TILE > end) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (t + 16 * (j / 4) + 4 * c + j % 4 >= end) {
                    s[j] = -INFINITY;
#pragma unroll
                    for (int v = 0; v < VC; v++) vf[v][j] = nmoe_u4{0, 0, 0, 0};
                }
        }
        float mt = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) - nmoe_dec_lift<T>;
        if (__any(mt > m)) {
            const float mn = fmaxf(m, mt), a = nmoe_exp2(m - mn);
            m = mn;
            l *= a;
#pragma unroll
            for (int v = 0; v < VC; v++)
#pragma unroll
                for (int i = 0; i < DD; i++) o[v][i] *= a;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            s[j] = nmoe_exp2(s[j] - m);
            l += s[j];
        }
        const nmoe_u4 pf = X::pack(s); /* to 16 bits: the products take no more; l has them in fp32 */
#pragma unroll
        for (int v = 0; v < VC; v++)
#pragma unroll
            for (int dd = 0; dd < DD; dd++) {
                nmoe_u4 x;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    x[j] = __builtin_amdgcn_perm(vf[v][2 * j + 1][dd / 2], vf[v][2 * j][dd / 2],
                                                 dd % 2 ? 0x07060302 : 0x05040100);
                o[v][dd] = X::mma16(x, pf, o[v][dd]);
            }
    };
    if (t0 < end) {
#pragma unroll
        for (int a = 0; a < 2; a++)
            row[a] = row_of(t0, a, t0 != guess ? page_of(t0, a) : t0 + 16 * a <= last16 ? early[a] : early[0]);
        load_k(t0, row);
        int t = t0;
        /* the last tile on its own: with a path that loads no next one, a wait for values would be one for the next keys */
        for (; (int64_t)t + NMOE_DEC_STEP < end; t += NMOE_DEC_STEP) work(t, std::false_type());
        work(t, std::true_type());
    }
    if (bad) s_bad = 1;
    __syncthreads();

    /* the wavefronts' parts; a lane's l covers its own keys only */
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (c == 0) {
        s_m[w][r] = m;
        s_l[w][r] = l;
    }
    if (r < heads) {
#pragma unroll
        for (int v = 0; v < VC; v++)
#pragma unroll
            for (int dd = 0; dd < DD; dd++)
#pragma unroll
                for (int i = 0; i < 4; i++) s_o[w][r][128 * v + DD * (4 * c + i) + dd] = o[v][dd][i];
    }
    __syncthreads();
    const bool whole = len <= per; /* the sequence is this one part */
    for (int x = tid; x < heads * D / 4; x += 64 * NMOE_DEC_WAVES) {
        const int h = x / (D / 4), d = x % (D / 4) * 4;
        float mj = -INFINITY, lj = 0.0f;
#pragma unroll
        for (int i = 0; i < NMOE_DEC_WAVES; i++) mj = fmaxf(mj, s_m[i][h]);
        nmoe_f4 y = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NMOE_DEC_WAVES; i++) {
            const float a = s_l[i][h] == 0.0f ? 0.0f : nmoe_exp2(s_m[i][h] - mj); /* one without weights has no maximum */
            lj += a * s_l[i][h];
            y += a * *(const nmoe_f4 *)&s_o[i][h][d];
        }
        const int64_t oh = (int64_t)b * q_heads + h0 + h;
        if (s_bad) lj = NAN;
        if (whole) {
            float z[4];
#pragma unroll
            for (int i = 0; i < 4; i++) z[i] = len == 0 ? 0.0f : y[i] / lj;
            nmoe_store<T, 4>(out + oh * D + d, z);
            if (lse != NULL && d == 0) lse[oh] = len == 0 ? -INFINITY : 0.69314718055994531f * (mj + log2f(lj));
        } else {
            *(nmoe_f4 *)(part_o + (oh * parts + part) * D + d) = y;
            if (d == 0) {
                part_ml[2 * (oh * parts + part)] = mj;
                part_ml[2 * (oh * parts + part) + 1] = lj;
            }
        }
    }
}

/* Joins a head's parts: 256 / (D / 4) groups of threads take parts in turn,
 * 4 dimensions a thread. */
template <typename T, int D>
__global__ void __launch_bounds__(NMOE_DEC_JOIN)
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
    const int len = nmoe_len_of(seq_lens[b], max_pages, page_size);
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

/* How the longest sequence is cut: into about two blocks a CU with heads of
 * 256, which is as many as run at once (by LDS and registers), and four else
 * (of heads of 128 three do, by registers, and of 64 five), in parts of whole
 * steps.  64 sequences of about 4096 on heads of 256: 96, 98, 104, 116, 108 us
 * with 1, 2, 3, 4, 8 blocks a CU; 20 of 5000 on heads of 128: 93, 81, 73, 69
 * us with 1 to 4.
 * It is one number for all lengths, and one part where the sequences alone are
 * blocks enough: a long one among many short ones stays on a few CUs.  255
 * sequences of 512 and one of 131071 (2 heads of 256) take 2408 us, 256 of 512
 * 42; 63 and one 621, 64 of 512 19. */
struct nmoe_dec_plan {
    int tiles, parts, per;
    size_t rows; /* partial rows */
};

static int nmoe_dec_tiles(const nmoe_hip_kv_cache *c, int q_heads) {
    return (q_heads / c->kv_heads + NMOE_DEC_HEADS - 1) / NMOE_DEC_HEADS;
}

static int64_t nmoe_dec_want(const nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *c) {
    return (c->head_dim == 256 ? 2 : 4) * (ctx->num_cus > 0 ? ctx->num_cus : 256);
}

static nmoe_dec_plan nmoe_dec_plan_of(const nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *c, int q_heads, int nseq,
                                      int64_t max_len) {
    nmoe_dec_plan p;
    p.tiles = nmoe_dec_tiles(c, q_heads);
    const int64_t blocks = (int64_t)nseq * c->kv_heads * p.tiles, want = nmoe_dec_want(ctx, c);
    if (max_len > NMOE_LONGEST) max_len = NMOE_LONGEST;
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
static size_t nmoe_dec_ws_bytes(const nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *c, int q_heads, int nseq,
                                int64_t max_len) {
    const int64_t u = (int64_t)c->kv_heads * nmoe_dec_tiles(c, q_heads), want = nmoe_dec_want(ctx, c);
    int64_t n = (want + u - 1) / u - 1, most = (max_len + NMOE_DEC_STEP - 1) / NMOE_DEC_STEP;
    if (n > nseq) n = nseq;
    if (most > NMOE_DEC_PARTS) most = NMOE_DEC_PARTS;
    if (n < 1 || most < 2) return 0;
    const int64_t parts = n * most < n + (want - 1) / u ? n * most : n + (want - 1) / u;
    return (size_t)parts * q_heads * (c->head_dim + 2) * sizeof(float);
}

template <typename T, int D>
static void nmoe_dec_launch_as(hipStream_t s, const nmoe_dec_plan &p, const nmoe_hip_kv_cache &c, const void *q,
                               int q_heads, int nseq, const int32_t *lens, const int32_t *table, int max_pages,
                               float scale, void *out, float *lse, void *ws) {
    float *po = (float *)ws, *pml = po + p.rows * D;
    hipLaunchKernelGGL((nmoe_attn_decode_kernel<T, D>), dim3((uint32_t)nseq * c.kv_heads * p.tiles * p.parts),
                       dim3(64 * NMOE_DEC_WAVES), 0, s, c, (const T *)q, q_heads, p.tiles, lens, table, max_pages, p.parts,
                       p.per, scale * 1.44269504088896341f, (T *)out, lse, po, pml);
    if (p.parts > 1)
        hipLaunchKernelGGL((nmoe_attn_join_kernel<T, D>), dim3((uint32_t)nseq * q_heads), dim3(NMOE_DEC_JOIN), 0, s,
                           q_heads, lens, max_pages, c.page_size, p.parts, p.per, po, pml, (T *)out, lse);
}

template <typename T>
static void nmoe_dec_launch(hipStream_t s, const nmoe_dec_plan &p, const nmoe_hip_kv_cache &c, const void *q,
                            int q_heads, int nseq, const int32_t *lens, const int32_t *table, int max_pages,
                            float scale, void *out, float *lse, void *ws) {
    if (c.head_dim == 64)
        nmoe_dec_launch_as<T, 64>(s, p, c, q, q_heads, nseq, lens, table, max_pages, scale, out, lse, ws);
    else if (c.head_dim == 128)
        nmoe_dec_launch_as<T, 128>(s, p, c, q, q_heads, nseq, lens, table, max_pages, scale, out, lse, ws);
    else
        nmoe_dec_launch_as<T, 256>(s, p, c, q, q_heads, nseq, lens, table, max_pages, scale, out, lse, ws);
}

static int nmoe_dec_check(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *cache, int q_heads, int nseq, int max_len) {
    int rc = nmoe_check_cache(ctx, cache);
    if (rc != NMOE_HIP_OK) return rc;
    if (q_heads < 1 || q_heads > NMOE_MAX_HEADS || q_heads % cache->kv_heads != 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: %d query heads on %d key heads (1..%d, a multiple)", q_heads,
                         cache->kv_heads, NMOE_MAX_HEADS);
    if (nseq < 0 || (int64_t)nseq * q_heads > NMOE_MAX_ROWS || max_len < 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: %d sequences of %d heads outside 0..2^22, or max_len %d < 0", nseq,
                         q_heads, max_len);
    return NMOE_HIP_OK;
}

extern "C" size_t nmoe_attn_decode_workspace(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *cache, int q_heads, int nseq,
                                             int max_len) {
    if (ctx == NULL || nmoe_dec_check(ctx, cache, q_heads, nseq, max_len) != NMOE_HIP_OK || nseq == 0) return 0;
    return nmoe_dec_ws_bytes(ctx, cache, q_heads, nseq, max_len);
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
    if (max_pages < 1 || !nmoe_scale_ok(scale))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: max_pages >= 1 and a scale below 2^127 are required");
    if (cache->token_stride >= NMOE_DEC_STRIDE)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: the cache's token stride is below %d elements", NMOE_DEC_STRIDE);
    if (nseq == 0) return NMOE_HIP_OK;
    const nmoe_dec_plan p = nmoe_dec_plan_of(ctx, cache, q_heads, nseq, max_len);
    const size_t need = p.rows != 0 ? nmoe_dec_ws_bytes(ctx, cache, q_heads, nseq, max_len) : 0; /* one part: none used */
    if (need != 0 && (ws == NULL || !nmoe_aligned(ws, 16) || ws_bytes < need))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: a workspace of %zu bytes (16-byte aligned) is required, %zu given",
                         need, ws == NULL ? (size_t)0 : ws_bytes);
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (cache->dtype == NMOE_HIP_BF16)
        nmoe_dec_launch<nmoe_bf16>(s, p, *cache, q, q_heads, nseq, seq_lens, page_table, max_pages, scale, out, lse, ws);
    else
        nmoe_dec_launch<_Float16>(s, p, *cache, q, q_heads, nseq, seq_lens, page_table, max_pages, scale, out, lse, ws);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
