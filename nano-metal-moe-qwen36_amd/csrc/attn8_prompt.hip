/*
 * attn8_prompt.hip -- attention of prompts, or pieces of them, over a paged
 * cache in 8 bits (nmoe_attn8_prompt).
 *
 * One pass over a query's keys with a running maximum m and sum l:
 *   s = c q.k,  p = 2^(s - m),  l += p,  o += p v;   out = o / l
 * (c = scale * log2(e)).  It is bound by the matrix cores: 4 D flops a pair of
 * query and key against 2 D bytes a key, which a block's 128 query rows share,
 * and next by the vector units, which make bf16 (or f16) of the codes.
 *
 * 3 prompts of 8191 tokens on 32 + 8 heads of 128 (218 GFLOP): 252 us, 0.87
 * PFLOP/s (in f16 280: scales with the scores and the weights), 96 tokens behind
 * 60001 on 16 + 2 of 256 (94 GFLOP): 125, one of 2048: 70, its last rows' keys in
 * turn.  A tile is about 60 % products and 40 %
 * conversions, exponentials and maxima, of two wavefronts a SIMD that overlap;
 * left out in turn, none of these (nor loads, nor page look-up) takes more than
 * 60 us of the 250 with it, and three wavefronts, tiles of 32 keys, sums in four
 * chains or operands read ahead were not faster.
 */
#include <type_traits>

#include "nmoe_attn8.h"

/* Workgroups of four pieces without groups from which on they fill 256 CUs (two on each): over 95 calls that are not
 * cut the choice took 1.2 % longer than the better of forms 0 and 2 with 300 to 340, 1.9 % with 280. */
#define NMOE_PR8_FULL 300
#define NMOE_PR8_SHORT 64 /* keys up to which groups do not share them (562 tokens of 9, up to 90 keys, heads of 256: 15.8 us, 17.2) */
/* The running maximum may lag by 2^8: weights stay below f16's limit (3 of 8191: 244 us, without 259; one of 8000 on
 * heads of 256: 550, 613). */
#define NMOE_PR8_SLACK 8.0f
/* Scales of values up to which bf16's weights are at most 2^8: a sum over 2^30 keys of 448 times that is below 2^126.  A key
 * whose value has a larger one counts for the running maximum as if its score were larger by the scale's power beyond this, so
 * that no weight times value is above that either; what has no weight, or is not seen, raises nothing. */
#define NMOE_PR8_TOP 79
#define NMOE_PR8_CUT 1024 /* keys from which on a sequence may be cut into parts (404 on 8 heads of 64 in two: 9.8 us, whole 8.6) */
#define NMOE_PR8_PART 512 /* least keys of a large workgroup's part */
/* And of a small one's (4000 keys, 17 tokens on 32 + 8 heads of 128; least parts of 128, 192, 256, 512 keys: 19.8, 14.9, 16.9, 19.0). */
#define NMOE_PR8_LEAST 192
#define NMOE_PR8_PARTS 256  /* most parts of a sequence */
#define NMOE_PR8_ROWS 128   /* query rows of a block of four pieces */
#define NMOE_PR8_JOIN 256
#define NMOE_PR8_FEW 8 /* parts that a wavefront joins by itself */
#define NMOE_PR8_ALL (1 << 30) /* rows times heads: a key head's rows are counted in 32 bits */

typedef __attribute__((address_space(3))) void nmoe_pr8_lds;
typedef int nmoe_i2 __attribute__((ext_vector_type(2)));

template <int D>
constexpr int nmoe_pr8_keys = D == 256 ? 32 : 64; /* of a tile */

/* f16 weights are held up to 2^7 times the lag, relative to the largest scale
 * of the values so far: those down to 2^-21 keep their 11 bits. */
#define NMOE_PR8_LIFT 7.0f

/* The 32-byte pairs of chunks of a tile's row are stored at pair ^ f(row), so
 * that neither 8 rows' same 16 bytes (a key operand's read: rows side by side)
 * nor 8 rows' same 32 bytes (a transposing value read: rows 0-3 and 8-11, or
 * 4-7 and 12-15, of 16) meet in a bank.  256 bytes are the banks' width: 1, 2
 * or 4 rows. */
template <int D>
__device__ __forceinline__ int nmoe_pr8_kswizzle(int row) {
    return D == 256 ? row & 7 : D == 128 ? row >> 1 & 3 : row >> 2 & 1;
}
template <int D>
__device__ __forceinline__ int nmoe_pr8_vswizzle(int row) {
    return D == 256 ? (row & 3) | (row >> 1 & 4) : D == 128 ? (row >> 1 & 1) | (row >> 2 & 2) : row >> 3 & 1;
}

/* Codes as operands: bf16 takes their scale on the way; f16 could not hold
 * every value, so it takes the codes. */
template <typename T>
struct nmoe_pr8_codes;

template <>
struct nmoe_pr8_codes<nmoe_bf16> {
    static __device__ __forceinline__ nmoe_u4 operand(uint32_t a, uint32_t b, float scale) {
        return nmoe_u4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))};
    }
};

template <>
struct nmoe_pr8_codes<_Float16> {
    static __device__ __forceinline__ nmoe_u4 operand(uint32_t a, uint32_t b, float) {
        return nmoe_u4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true))};
    }
};

/* The larger of a lane's value and lane + 32's. */
__device__ __forceinline__ float nmoe_pr8_max32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

struct nmoe_pr8_call {
    int q_heads, nseq, ntok, max_pages, causal, parts, per, cut_rows;
    const int32_t *cu_q, *seq_lens, *page_table;
    float c;
    uint32_t q_and, q_xor;
    float *lse, *part_o, *part_ml;
};

/* The first row of a sequence: partial rows are numbered from it. */
__device__ __forceinline__ int nmoe_pr8_first(const nmoe_pr8_call &a) { return min(max(a.cu_q[0], 0), a.ntok); }

/* How a sequence of len keys and the rows q0 .. q0 + nq is cut: `per` keys a
 * part (the call's, or as many as the call's number of parts needs when
 * max_len was too small); not at all where its partial rows would not be among
 * the cut_rows that the workspace has room for (max_q was too small). */
__device__ __forceinline__ int nmoe_pr8_per(const nmoe_pr8_call &a, int q0, int nq, int len) {
    const int first = nmoe_pr8_first(a);
    if (q0 < first || (int64_t)(q0 + nq - first) * a.q_heads > a.cut_rows) return NMOE_LONGEST;
    const int64_t need = ((int64_t)len + a.parts - 1) / a.parts;
    return need <= a.per ? a.per : (int)((need + 63) / 64 * 64);
}

/* A block: SUBS pieces of 32 query rows of one key head, rows numbered (token,
 * head), and KG groups of SUBS wavefronts that take the key tiles in turn (two
 * where there are too few blocks to fill the device; joined at the end); with
 * parts, of one part of the keys.
 *
 * S^T (keys x queries) = K Q^T, 32x32x16: a lane holds one query's scores, so
 * maximum and sum need one exchange with lane + 32, and the weights are the
 * second product's column operand where they are: of 16 keys, which are one
 * block of the cache, a lane has 8 g + 4 (l / 32) + e (g < 2, e < 4), which is
 * the order the product takes them in.  O^T (dimensions x queries) = V^T P^T;
 * V^T comes from V's rows by the LDS's transposing reads.
 *
 * Tiles go from memory to LDS directly as codes, the next while one is
 * multiplied, and its scales and the pages of the one after into registers:
 * lane j those of the tile's block j.  Rows behind the last key repeat it
 * (their weights are 0).  A stage is H tiles; two of them with heads of 256, whose
 * tiles are short, halve the barriers and look-ups (8000 tokens: 550 us, 561). */
template <typename T, int D, int SUBS, int KG, int H>
__global__ void __launch_bounds__(64 * SUBS * KG, 2)
    nmoe_attn8_prompt_kernel(nmoe_hip_kv8_cache cache, nmoe_pr8_call a, const T *q, T *out) {
    typedef nmoe_mat<T> X;
    typedef nmoe_pr8_codes<T> Y;
    constexpr bool F16 = nmoe_elem<T>::dtype == NMOE_HIP_F16;
    constexpr int GT = 64 * SUBS, KT = nmoe_pr8_keys<D>, ST = H * KT, KS = KT / 32, DT = D / 32; /* keys of a tile, of a stage */
    constexpr int CPR = D / 16, RPI = GT / CPR, NI = ST / RPI;
    constexpr int NB = ST / 16, RPW = 64 / CPR; /* blocks of a stage; rows of a wavefront's load */
    constexpr int EVERY = H * KS * (D / 16) / (2 * NI);
    static_assert(EVERY * 2 * NI == H * KS * (D / 16) && 16 % RPW == 0 && NB <= 32, "a load to so many products, of one block");
    constexpr int TILE = ST * D, HELD = KG * 4 * TILE;
    constexpr int ROUND = KG == 1 ? DT : HELD / (SUBS * 4096) < DT ? HELD / (SUBS * 4096) : DT; /* 32 dimensions of every piece */
    /* [group][buffer][K, V]: by name, as the compiler would take a read of one buffer for one of the tile under way */
    __shared__ alignas(16) uint8_t s_kv0[KG][2][TILE], s_kv1[KG][2][TILE];
    __shared__ float s_ml[2][SUBS][KG == 2 ? 64 : 1];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wq = wave % SUBS, kg = wave / SUBS, hh = lane / 32;
    const int pairs = cache.kv_heads * a.nseq, group = a.q_heads / cache.kv_heads;
    const int pair = blockIdx.x % pairs, kh = pair % cache.kv_heads, b = pair / cache.kv_heads;
    const int part = blockIdx.x / pairs % a.parts, lot = blockIdx.x / pairs / a.parts, lots = gridDim.x / pairs / a.parts;
    const int q0 = min(max(a.cu_q[b], 0), a.ntok), nq = min(max(a.cu_q[b + 1], q0), a.ntok) - q0;
    const int len = nmoe_len_of(a.seq_lens[b], a.max_pages, cache.page_size), nk = max(len, 0);
    const int all = nq * group, tiles = (all + 32 * SUBS - 1) / (32 * SUBS);
    const int ahead = nk - nq + 1; /* query i sees keys below i + ahead */
    const int per = nmoe_pr8_per(a, q0, nq, nk);
    const int64_t from = (int64_t)part * per;
    if (part != 0 && from >= nk) return;
    const int k0 = (int)from, k1 = (int)min((int64_t)nk, from + per); /* the part's keys */

    const uint8_t *const kbase = (const uint8_t *)cache.k + kh * cache.head_stride;
    const uint8_t *const vbase = (const uint8_t *)cache.v + kh * cache.head_stride;
    const int32_t *const table = a.page_table + (int64_t)b * a.max_pages;
    const uint32_t step = (uint32_t)cache.token_stride;
    const int bpp = cache.page_size / 16, last_block = nk > 0 ? (nk - 1) / 16 : 0;
    const int hop = KG * NB, hop_pages = hop / bpp, hop_blocks = hop % bpp; /* from a group's stage to its next */
    const int end_page = last_block / bpp, end_block = last_block % bpp;
    const int64_t block_stride = 16 * cache.token_stride;

    /* a lane's places in a K and a V tile; other chunks of the row by the same bits of their numbers */
    const int kplace = lane % 32 * D + nmoe_pr8_kswizzle<D>(lane % 32) * 32 + hh * 16;
    const int vkey = 4 * hh + lane % 16 / 2 + (lane % 16 >= 8 ? 4 : 0); /* of a block's keys 0-3 and 8-11, or 4-7 and 12-15 */
    const int vplace = vkey * D + nmoe_pr8_vswizzle<D>(vkey) * 32 + lane / 16 % 2 * 16 + lane % 2 * 8;

    /* the latest rows, which see the most keys, first */
    for (int tile = tiles - 1 - lot; tile >= 0; tile -= lots) {
        const int row0 = (tile * SUBS + wq) * 32, row = row0 + lane % 32, last = min(all, (tile + 1) * SUBS * 32) - 1;
        const bool active = row0 < all;
        const int i = min(row, all - 1) / group, h = kh * group + (min(row, all - 1) - i * group);
        const int see = a.causal ? min(max(i + ahead, 0), nk) : nk;
        /* every row of the piece sees keys below see_lo, none those of the part from see_hi on */
        const int see_lo = a.causal ? min(row0, all - 1) / group + ahead : nk;
        const int see_hi = active ? min(a.causal ? min(row0 + 31, all - 1) / group + ahead : nk, k1) : 0;
        const int end = min(a.causal ? last / group + ahead : nk, k1);
        const int nt = end > k0 ? (end - k0 + ST - 1) / ST : 0;

        nmoe_u4 qf[D / 16];
        const T *qr = q + ((int64_t)(q0 + i) * a.q_heads + h) * D + 16 * hh;
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
            qf[k] = *(const nmoe_u4 *)(qr + 32 * (k / 2) + 8 * (k % 2));
#pragma unroll
            for (int e = 0; e < 4; e++) qf[k][e] = (qf[k][e] & a.q_and) ^ a.q_xor;
        }
        nmoe_f16v o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
        float m = -3.402823466e38f, l = 0.0f, ref = nmoe_kv8_two_to(NMOE_KV8_LOW);
        bool bad = len < 0;

        /* lane j: block j % NB of the stage that is next to be asked for */
        int at = (k0 + kg * ST) / 16 + lane % NB, at_page = at / bpp, at_block = at % bpp;
        int page = table[min(at_page, end_page)], block = at > last_block ? end_block : at_block;
        float scale = 0.0f;
        int64_t base[NI];
        int top[NI];
        /* the addresses of the stage whose pages have come, its scales, and the pages of the one behind it */
        auto turn = [&](int first) {
            if (__any(first + 16 * (lane % NB) < see_hi && (uint32_t)page >= (uint32_t)cache.num_pages)) bad = true;
            if ((uint32_t)page >= (uint32_t)cache.num_pages) page = 0;
            scale = (hh == 0 ? cache.k_scale : cache.v_scale)[((int64_t)page * bpp + block) * cache.kv_heads + kh];
            /* as a lane's own, then taken from it: 64-bit products of scalars took more */
            const int64_t off = page * cache.page_stride + block * block_stride;
            const int keys = min(nk - 1 - min(at, last_block) * 16, 15);
#pragma unroll
            for (int n = 0; n < NI; n++) {
                const int u = (n * RPI + wq * RPW) / 16;
                base[n] = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), u) << 32 |
                                    (uint32_t)__builtin_amdgcn_readlane((int)off, u));
                top[n] = __builtin_amdgcn_readlane(keys, u);
            }
            at += hop;
            at_page += hop_pages;
            at_block += hop_blocks;
            if (at_block >= bpp) {
                at_block -= bpp;
                at_page++;
            }
            page = table[min(at_page, end_page)];
            block = at > last_block ? end_block : at_block;
        };
        /* load i of a stage's 2 NI: of K, then of V */
        auto load = [&](auto buf, int i) {
            const int n = i % NI, r = n * RPI + wq * RPW + lane / CPR;
            const uint32_t pair2 = 2 * (i < NI ? nmoe_pr8_kswizzle<D>(r) : nmoe_pr8_vswizzle<D>(r));
            const int off = (int)((uint32_t)min(r % 16, top[n]) * step + ((uint32_t)(lane % CPR) ^ pair2) * 16);
            const __amdgpu_buffer_rsrc_t rs = nmoe_buffer((i < NI ? kbase : vbase) + base[n]);
            const int to = (n * GT + wq * 64) * 16;
            if constexpr (decltype(buf)::value == 0)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (nmoe_pr8_lds *)&s_kv0[kg][i < NI ? 0 : 1][to], 16, off, 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (nmoe_pr8_lds *)&s_kv1[kg][i < NI ? 0 : 1][to], 16, off, 0, 0, 0);
        };
        auto of_block = [&](float v, int j) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), j)); };
        auto work = [&](const int t, auto buf) {
            constexpr bool B = decltype(buf)::value != 0;
            const std::integral_constant<int, !B> other;
            const int stage = k0 + t * ST;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const float held = scale;
            turn(stage + KG * ST);
#pragma unroll
            for (int half = 0; half < H; half++) {
                const int key0 = stage + half * KT;
                if (key0 >= see_hi) {
#pragma unroll
                    for (int n = 0; n < 2 * NI / H; n++) load(other, half * (2 * NI / H) + n);
                    continue;
                }
                const uint8_t *sk = (B ? s_kv1[kg][0] : s_kv0[kg][0]) + half * KT * D, *sv = (B ? s_kv1[kg][1] : s_kv0[kg][1]) + half * KT * D;
                int krow = kplace, vrow = vplace;
                asm volatile("" : "+v"(krow), "+v"(vrow)); /* made anew for each tile, not kept each in a register */
                float s[KS][16];
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    nmoe_f16v x;
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = 0.0f;
                    const int b0 = half * (KT / 16) + 2 * k;
                    const float ks = F16 ? 1.0f : lane % 32 < 16 ? of_block(held, b0) : of_block(held, b0 + 1);
                    const uint8_t *p = sk + 32 * k * D;
#pragma unroll
                    for (int d = 0; d < D / 32; d++) {
                        const nmoe_u4 y = *(const nmoe_u4 *)(p + (krow ^ 32 * d));
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const int n = 2 * d + u;
                            x = X::mma32(Y::operand(y[2 * u], y[2 * u + 1], ks), qf[n], x);
                            if (n % EVERY == EVERY - 1) {
                                load(other, ((half * KS + k) * (D / 16) + n) / EVERY);
                                __builtin_amdgcn_sched_barrier(0x106); /* stays between its products; LDS reads, VALU and SALU need not */
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) s[k][e] = F16 ? x[e] * of_block(held, b0 + e / 8) : x[e];
                }
                if (key0 + KT > min(see_lo, k1)) {
                    asm volatile("" ::: "memory"); /* a branch, not selects in every tile */
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (key0 + 32 * k + 8 * (e / 4) + 4 * hh + e % 4 >= min(see, k1)) s[k][e] = -INFINITY;
                }
                float mt = s[0][0];
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 16; e++) mt = fmaxf(mt, s[k][e]);
                float vs[KT / 16];
#pragma unroll
                for (int u = 0; u < KT / 16; u++) vs[u] = of_block(held, 32 + half * (KT / 16) + u);
                mt = nmoe_pr8_max32(mt) * a.c;
                if constexpr (!F16) {
                    float most = vs[0];
#pragma unroll
                    for (int u = 1; u < KT / 16; u++) most = fmaxf(most, vs[u]);
                    if (most > nmoe_kv8_two_to(NMOE_PR8_TOP)) { /* of the wavefront */
                        mt = -INFINITY;
#pragma unroll
                        for (int u = 0; u < KT / 16; u++) {
                            float x = s[u / 2][8 * (u % 2)];
#pragma unroll
                            for (int e = 1; e < 8; e++) x = fmaxf(x, s[u / 2][8 * (u % 2) + e]);
                            mt = fmaxf(mt, fmaf(x, a.c, nmoe_kv8_beyond(vs[u], NMOE_PR8_TOP)));
                        }
                        mt = nmoe_pr8_max32(mt);
                    }
                }
                if (__any(mt > m + NMOE_PR8_SLACK)) {
                    const float mn = fmaxf(m, mt), f = nmoe_exp2(m - mn);
                    m = mn;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) o[d][e] *= f;
                }
                if constexpr (F16) { /* weights relative to the largest scale that the row has seen so far */
                    if (key0 + KT > min(see_lo, k1)) {
#pragma unroll
                        for (int u = 0; u < KT / 16; u++)
                            if (key0 + 16 * u >= min(see, k1)) vs[u] = 0.0f;
                    }
                    float most = vs[0];
#pragma unroll
                    for (int u = 1; u < KT / 16; u++) most = fmaxf(most, vs[u]);
                    if (most > ref) {
                        const float f = ref / most;
                        ref = most;
#pragma unroll
                        for (int d = 0; d < DT; d++)
#pragma unroll
                            for (int e = 0; e < 16; e++) o[d][e] *= f;
                    }
#pragma unroll
                    for (int u = 0; u < KT / 16; u++) vs[u] = vs[u] / ref * exp2f(NMOE_PR8_LIFT);
                }
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        s[k][e] = nmoe_exp2(fmaf(s[k][e], a.c, -m));
                        l += s[k][e];
                        if constexpr (F16) s[k][e] *= vs[2 * k + e / 8];
                    }
#pragma unroll
                for (int u = 0; u < KT / 16; u++) {
                    const nmoe_u4 pf = X::pack(&s[u / 2][8 * (u % 2)]); /* to 16 bits: the products take no more; l has them in fp32 */
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        typedef __attribute__((address_space(3))) nmoe_i2 lds_i2;
                        const nmoe_i2 y = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2 *)(sv + 16 * u * D + (vrow ^ 32 * d)));
                        o[d] = X::mma32(Y::operand((uint32_t)y[0], (uint32_t)y[1], vs[u]), pf, o[d]);
                    }
                }
            }
        };
        __syncthreads();
        if (kg < nt) {
            turn(k0 + kg * ST);
#pragma unroll
            for (int n = 0; n < 2 * NI; n++) load(std::integral_constant<int, 0>(), n);
        }
        for (int t0 = 0; t0 < nt; t0 += 2 * KG) {
            work(t0 + kg, std::integral_constant<int, 0>());
            if (t0 + KG < nt) work(t0 + KG + kg, std::integral_constant<int, 1>());
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); /* the last loads are for no one, but not for the next block's LDS */
        l += __shfl_xor(l, 32, 64);
        if (bad) l = NAN;
        if constexpr (F16) {
            const float f = ref * exp2f(-NMOE_PR8_LIFT);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= f;
        }
        if constexpr (KG == 2) {
            float m1 = 0.0f, l1 = 0.0f, f0 = 1.0f, f1 = 0.0f;
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += ROUND) {
                /* [piece][16 ROUND][64], over both buffers of both groups */
                float *const so0 = (float *)s_kv0, *const so1 = (float *)s_kv1;
                auto place = [&](int x) { /* of s_kv0 the first half */
                    const int w = (wq * 16 * ROUND + x) * 64 + lane;
                    return w < HELD / 8 ? so0 + w : so1 + (w - HELD / 8);
                };
                __syncthreads();
                if (kg == 1) {
                    s_ml[0][wq][lane] = m;
                    s_ml[1][wq][lane] = l;
#pragma unroll
                    for (int d = 0; d < ROUND; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) *place(16 * d + e) = o[d0 + d][e];
                }
                __syncthreads();
                if (kg == 0) {
                    if (d0 == 0) {
                        m1 = s_ml[0][wq][lane];
                        l1 = s_ml[1][wq][lane];
                        const float mn = fmaxf(m, m1);
                        f0 = nmoe_exp2(m - mn);
                        f1 = nmoe_exp2(m1 - mn);
                        m = mn;
                        l = l * f0 + l1 * f1;
                    }
#pragma unroll
                    for (int d = 0; d < ROUND; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) o[d0 + d][e] = o[d0 + d][e] * f0 + *place(16 * d + e) * f1;
                }
            }
        }
        if (kg == 0 && row < all) {
            const int64_t oh = (int64_t)(q0 + i) * a.q_heads + h;
            if (see <= per) { /* all its keys are the first part's */
                if (part == 0) {
                    const float inv = see > 0 ? 1.0f / l : 0.0f;
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float z[4];
#pragma unroll
                            for (int j = 0; j < 4; j++) z[j] = see > 0 ? o[d][4 * e + j] * inv : bad ? NAN : 0.0f;
                            nmoe_store<T, 4>(out + oh * D + 32 * d + 8 * e + 4 * hh, z);
                        }
                    if (a.lse != NULL && hh == 0)
                        a.lse[oh] = see > 0 ? 0.69314718055994531f * (m + log2f(l)) : bad ? NAN : -INFINITY;
                }
            } else if (see > k0) {
                const int64_t po = (oh - (int64_t)nmoe_pr8_first(a) * a.q_heads) * a.parts + part;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        *(nmoe_f4 *)(a.part_o + po * D + 32 * d + 8 * e + 4 * hh) =
                            nmoe_f4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
                if (hh == 0) {
                    a.part_ml[2 * po] = m;
                    a.part_ml[2 * po + 1] = l;
                }
            }
        }
    }
}

/* Parts that token t's results are joined from: 0 where they are not. */
__device__ __forceinline__ int nmoe_pr8_joined(const nmoe_pr8_call &a, int page_size, int t) {
    const int lane = threadIdx.x % 64;
    /* the sequence whose rows hold it */
    int b = 0, n = a.nseq;
    while (n > 1) {
        const int stride = (n + 63) / 64, at = lane * stride;
        const uint64_t below = __ballot(at < n && min(max(a.cu_q[b + min(at, n - 1)], 0), a.ntok) <= t);
        const int last = max((int)__popcll(below) - 1, 0) * stride;
        b += last;
        n = min(stride, n - last);
    }
    const int q0 = min(max(a.cu_q[b], 0), a.ntok), nq = min(max(a.cu_q[b + 1], q0), a.ntok) - q0;
    if (t < q0 || t >= q0 + nq) return 0;
    const int nk = max(nmoe_len_of(a.seq_lens[b], a.max_pages, page_size), 0);
    const int see = a.causal ? min(t - q0 + 1 + nk - nq, nk) : nk, per = nmoe_pr8_per(a, q0, nq, nk);
    return see <= per ? 0 : (int)(((int64_t)see + per - 1) / per); /* written by its one part */
}

/* Joins a row's parts: a wavefront a row and head, D / 64 dimensions a lane. */
template <typename T, int D>
__global__ void __launch_bounds__(NMOE_PR8_JOIN)
    nmoe_attn8_prompt_join_kernel(nmoe_pr8_call a, int page_size, T *out) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x % 64;
    const int64_t at = (int64_t)blockIdx.x * (NMOE_PR8_JOIN / 64) + threadIdx.x / 64; /* partial row and place in out */
    const int64_t oh = at + (int64_t)nmoe_pr8_first(a) * a.q_heads;
    const int t = (int)(oh / a.q_heads);
    if (at >= a.cut_rows || t >= a.ntok) return;
    const int parts = nmoe_pr8_joined(a, page_size, t);
    if (parts == 0) return;
    const float *ml = a.part_ml + 2 * at * a.parts, *po = a.part_o + at * a.parts * D + E * lane;
    float m = -3.402823466e38f, l = 0.0f, o[E] = {};
    for (int p = 0; p < parts; p++) m = fmaxf(m, ml[2 * p]);
#pragma unroll 4
    for (int p = 0; p < parts; p++) {
        const float f = nmoe_exp2(ml[2 * p] - m);
        l += f * ml[2 * p + 1];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] += f * po[(int64_t)p * D + e];
    }
#pragma unroll
    for (int e = 0; e < E; e++) out[oh * D + E * lane + e] = nmoe_elem<T>::put(o[e] / l);
    if (a.lse != NULL && lane == 0) a.lse[oh] = 0.69314718055994531f * (m + log2f(l));
}

/* The same for many parts, a block a row and head: 256 / (D / 4) groups of
 * threads take them in turn, 4 dimensions a thread (2 tokens behind 60000, heads
 * of 256, 118 parts: 34 us instead of 52; 30 behind 4000, of 64, 16 parts: 10.9,
 * 12.2; 31 on 32 + 8 of 128, 16 parts: 17.6, 16.9; 1024 behind 8000, 2 parts:
 * 180 instead of 173). */
template <typename T, int D>
__global__ void __launch_bounds__(NMOE_PR8_JOIN)
    nmoe_attn8_prompt_join_many_kernel(nmoe_pr8_call a, int page_size, T *out) {
    constexpr int LANES = D / 4, GROUPS = NMOE_PR8_JOIN / LANES;
    __shared__ nmoe_f4 s_y[GROUPS][LANES];
    __shared__ float s_m[GROUPS], s_l[GROUPS];
    const int w = threadIdx.x / LANES, d = threadIdx.x % LANES;
    const int64_t at = blockIdx.x, oh = at + (int64_t)nmoe_pr8_first(a) * a.q_heads;
    const int parts = nmoe_pr8_joined(a, page_size, (int)(oh / a.q_heads));
    if (parts == 0) return; /* the whole block */
    const float *ml = a.part_ml + 2 * at * a.parts, *po = a.part_o + at * a.parts * D + 4 * d;
    float m = -INFINITY, l = 0.0f;
    nmoe_f4 y = {0, 0, 0, 0};
#pragma unroll 4
    for (int p = w; p < parts; p += GROUPS) {
        const float mx = ml[2 * p], lx = ml[2 * p + 1], mn = fmaxf(m, mx);
        const float fa = nmoe_exp2(m - mn), fb = nmoe_exp2(mx - mn);
        y = fa * y + fb * *(const nmoe_f4 *)(po + (int64_t)p * D);
        l = fa * l + fb * lx;
        m = mn;
    }
    s_y[w][d] = y;
    if (d == 0) {
        s_m[w] = m;
        s_l[w] = l;
    }
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int i = 1; i < GROUPS; i++) {
        const float mn = fmaxf(m, s_m[i]), fa = nmoe_exp2(m - mn), fb = nmoe_exp2(s_m[i] - mn); /* the first has a part */
        y = fa * y + fb * s_y[i][d];
        l = fa * l + fb * s_l[i];
        m = mn;
    }
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; e++) z[e] = y[e] / l;
    nmoe_store<T, 4>(out + oh * D + 4 * d, z);
    if (a.lse != NULL && d == 0) a.lse[oh] = 0.69314718055994531f * (m + log2f(l));
}

/* How a call is cut.  Form 0 is workgroups of 4 pieces without groups: the
 * most work a byte, but a row's keys are one wavefront's.  Form 2, 2 pieces
 * with two groups, goes over them in half the time and does about a fifth less
 * a second: it is for calls that are as long as their longest rows take (one
 * prompt, causal, 16 on 2 heads of 256: 2048 tokens 106 us in form 0, 73 in 2;
 * 4100: 200, 178; 6000: 302, 324; 8 heads of 64, 8100: 128, 104), not for
 * ragged batches that fill the device (9 prompts of 2214 on heads of 256: 31,
 * 42).  With few rows and many keys a sequence is cut into parts that a second
 * launch joins: by form 1, 4 pieces with two groups (96 tokens behind 60001:
 * 1515 us in form 2 uncut, 125), or, where large workgroups would be half empty
 * or their parts short, by form 2 (heads of 256, 4000 keys, 7 tokens: in parts
 * of form 1, of 512 keys, 37 us, now 23; of 128, 60000 keys, 2 tokens: 48, 33).
 * All sequences of a call are cut alike, as its longest and fullest would be:
 * one piece among many single tokens leaves those uncut (2048 and 63 single
 * tokens behind 512 each, 711 us; the tokens by nmoe_attn8_decode_rows, 89).
 * Form 1 uncut was never better than both by more than 4 %. */
struct nmoe_pr8_plan {
    int form, pieces, parts, per;
    int64_t lots; /* blocks a pair of sequence and key head, and part */
};

static int64_t nmoe_pr8_cus(const nmoe_hip_ctx *ctx) { return ctx->num_cus > 0 ? ctx->num_cus : 256; }

static nmoe_pr8_plan nmoe_pr8_plan_of(const nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *c, int q_heads, int nseq, int ntok,
                                      int64_t max_q, int64_t max_len, bool causal) {
    nmoe_pr8_plan p;
    const int64_t cus = nmoe_pr8_cus(ctx);
    if (max_q < 1) max_q = 1;
    if (max_q > ntok) max_q = ntok;
    const int64_t real = max_q * nseq < ntok ? max_q * nseq : ntok; /* the others are padding */
    const int group = q_heads / c->kv_heads, D = c->head_dim;
    const int64_t pairs = (int64_t)c->kv_heads * nseq, rows = max_q * group;
    /* tiles of so many rows: as many as all rows fill, and at most one more for each pair */
    const auto tiles = [&](int64_t of) {
        const int64_t least = (real * q_heads + of - 1) / of, each = (rows + of - 1) / of * pairs;
        return each < least ? least : each > least + pairs ? least + pairs : each;
    };
    const int64_t blocks = tiles(NMOE_PR8_ROWS), two = tiles(NMOE_PR8_ROWS / 2);
    /* blocks that a long prompt's last rows do not outlast: as many as if all its rows saw as many keys as the last */
    if (max_len > NMOE_LONGEST) max_len = NMOE_LONGEST;
    const int64_t mean = causal ? max_len - (max_q < max_len ? max_q : max_len) / 2 : max_len;
    const bool full = blocks * mean >= max_len * NMOE_PR8_FULL * cus / 256;
    const bool brief = max_len <= (D == 256 ? 2 : 1) * NMOE_PR8_SHORT || (two > 2 * cus && max_len < 8 * NMOE_PR8_SHORT);
    p.form = full || brief ? 0 : 2;
    p.parts = 1;
    p.per = 1 << 30;
    if (max_len >= NMOE_PR8_CUT) {
        /* one block a CU, all at once: a large one, where it has the rows and its part the keys, else a small one */
        int64_t parts = cus / blocks;
        const int form = two == blocks || parts > max_len / NMOE_PR8_PART ? 2 : 1;
        if (form == 2) {
            parts = cus / two;
            if (parts > max_len / NMOE_PR8_LEAST) parts = max_len / NMOE_PR8_LEAST;
        }
        if (parts > NMOE_PR8_PARTS) parts = NMOE_PR8_PARTS;
        if (parts > 1) {
            p.form = form;
            p.per = (int)(((max_len + parts - 1) / parts + 63) / 64 * 64);
            p.parts = (int)((max_len + p.per - 1) / p.per);
        }
    }
    p.pieces = p.form == 2 ? 2 : 4;
    p.lots = (rows + 32 * p.pieces - 1) / (32 * p.pieces);
    if (p.lots * pairs * p.parts > NMOE_MAX_ROWS) p.lots = NMOE_MAX_ROWS / (pairs * p.parts); /* the blocks go on to further tiles */
    if (p.lots < 1) p.lots = 1;
    return p;
}

/* Partial rows that do for every plan on as many tokens or fewer, and lengths
 * up to max_len.  A plan of r real rows (tokens times heads) has at most cus /
 * ceil(r / 128) <= 128 cus / r parts, or fewer, or max_len / NMOE_PR8_LEAST;
 * with more than r rows, fewer sequences are cut (nmoe_pr8_per). */
static int64_t nmoe_pr8_partial(const nmoe_hip_ctx *ctx, int q_heads, int ntok, int64_t max_len) {
    const int64_t most = NMOE_PR8_ROWS * nmoe_pr8_cus(ctx), rows = (int64_t)ntok * q_heads;
    if (max_len < NMOE_PR8_CUT) return 0;
    int64_t parts = max_len / NMOE_PR8_LEAST;
    if (parts > NMOE_PR8_PARTS) parts = NMOE_PR8_PARTS;
    const int64_t each = rows * parts;
    return most < each ? most : each;
}

static size_t nmoe_pr8_ws_bytes(const nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *c, int q_heads, int ntok, int64_t max_len) {
    return (size_t)nmoe_pr8_partial(ctx, q_heads, ntok, max_len) * (c->head_dim + 2) * sizeof(float);
}

template <typename T, int D>
static void nmoe_pr8_launch_as(hipStream_t s, const nmoe_pr8_plan &p, const nmoe_hip_kv8_cache &c, const nmoe_pr8_call &a,
                               const void *q, void *out) {
    const dim3 g((uint32_t)(p.lots * c.kv_heads * a.nseq * p.parts));
    if (p.form == 0)
        hipLaunchKernelGGL((nmoe_attn8_prompt_kernel<T, D, 4, 1, D == 256 ? 2 : 1>), g, dim3(256), 0, s, c, a, (const T *)q, (T *)out);
    else if (p.form == 1)
        hipLaunchKernelGGL((nmoe_attn8_prompt_kernel<T, D, 4, 2, D == 256 ? 2 : 1>), g, dim3(512), 0, s, c, a, (const T *)q, (T *)out);
    else
        hipLaunchKernelGGL((nmoe_attn8_prompt_kernel<T, D, 2, 2, 1>), g, dim3(256), 0, s, c, a, (const T *)q, (T *)out);
    if (p.parts > 1) {
        const int64_t all = (int64_t)a.ntok * a.q_heads, rows = a.cut_rows < all ? a.cut_rows : all;
        if (p.parts > NMOE_PR8_FEW)
            hipLaunchKernelGGL((nmoe_attn8_prompt_join_many_kernel<T, D>), dim3((uint32_t)rows), dim3(NMOE_PR8_JOIN), 0, s, a,
                               c.page_size, (T *)out);
        else
            hipLaunchKernelGGL((nmoe_attn8_prompt_join_kernel<T, D>), dim3((uint32_t)((rows + NMOE_PR8_JOIN / 64 - 1) / (NMOE_PR8_JOIN / 64))),
                               dim3(NMOE_PR8_JOIN), 0, s, a, c.page_size, (T *)out);
    }
}

template <typename T>
static void nmoe_pr8_launch(hipStream_t s, const nmoe_pr8_plan &p, const nmoe_hip_kv8_cache &c, const nmoe_pr8_call &a,
                            const void *q, void *out) {
    if (c.head_dim == 64)
        nmoe_pr8_launch_as<T, 64>(s, p, c, a, q, out);
    else if (c.head_dim == 128)
        nmoe_pr8_launch_as<T, 128>(s, p, c, a, q, out);
    else
        nmoe_pr8_launch_as<T, 256>(s, p, c, a, q, out);
}

static bool nmoe_pr8_counts_ok(int ntok, int q_heads, int max_q, int max_len) {
    return ntok >= 0 && ntok <= NMOE_MAX_ROWS && (int64_t)ntok * q_heads <= NMOE_PR8_ALL && max_q >= 0 && max_len >= 0;
}

extern "C" size_t nmoe_attn8_prompt_workspace(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, int q_heads, int nseq,
                                              int ntok, int max_q, int max_len) {
    if (ctx == NULL || nmoe_attn8_check_heads(ctx, cache, "prompt", q_heads, nseq) != NMOE_HIP_OK || nseq == 0 ||
        !nmoe_pr8_counts_ok(ntok, q_heads, max_q, max_len))
        return 0;
    return nmoe_pr8_ws_bytes(ctx, cache, q_heads, ntok, max_len);
}

extern "C" int nmoe_attn8_prompt(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const void *q, int q_dtype, int q_heads,
                                 int nseq, const int32_t *cu_q, int ntok, const int32_t *seq_lens, const int32_t *page_table,
                                 int max_pages, int max_q, int max_len, int causal, float scale, void *out, float *lse,
                                 void *ws, size_t ws_bytes, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_attn8_check(ctx, cache, "prompt", q, q_dtype, q_heads, nseq, seq_lens, page_table, max_pages, scale, out, lse);
    if (rc != NMOE_HIP_OK) return rc;
    if (cu_q == NULL || !nmoe_aligned(cu_q, 4) || !nmoe_pr8_counts_ok(ntok, q_heads, max_q, max_len))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: cu_q, 0 <= ntok <= 2^22 (times q_heads 2^30), max_q >= 0 and max_len >= 0 "
                                               "are required");
    if (nseq == 0 || ntok == 0) return NMOE_HIP_OK;
    const nmoe_pr8_plan p = nmoe_pr8_plan_of(ctx, cache, q_heads, nseq, ntok, max_q, max_len, causal != 0);
    const size_t need = p.parts > 1 ? nmoe_pr8_ws_bytes(ctx, cache, q_heads, ntok, max_len) : 0;
    if (need != 0 && (ws == NULL || !nmoe_aligned(ws, 16) || ws_bytes < need))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "prompt: a workspace of %zu bytes (16-byte aligned) is required, %zu given", need,
                         ws == NULL ? (size_t)0 : ws_bytes);
    nmoe_pr8_call a = {};
    a.q_heads = q_heads;
    a.nseq = nseq;
    a.ntok = ntok;
    a.max_pages = max_pages;
    a.causal = causal;
    a.parts = p.parts;
    a.per = p.per;
    a.cu_q = cu_q;
    a.seq_lens = seq_lens;
    a.page_table = page_table;
    /* c > 0, so that the largest score is the largest product: the sign goes to q, exactly, and a scale of 0 to q too */
    a.c = scale == 0.0f ? 1.0f : fabsf(scale) * 1.44269504088896341f;
    a.q_and = scale == 0.0f ? 0u : 0xffffffffu;
    a.q_xor = scale < 0.0f ? 0x80008000u : 0u;
    a.lse = lse;
    a.part_o = (float *)ws;
    if (p.parts > 1) {
        const int64_t partial = nmoe_pr8_partial(ctx, q_heads, ntok, max_len);
        a.part_ml = a.part_o + partial * cache->head_dim;
        a.cut_rows = (int)(partial / p.parts);
    }
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (q_dtype == NMOE_HIP_BF16)
        nmoe_pr8_launch<nmoe_bf16>(s, p, *cache, a, q, out);
    else
        nmoe_pr8_launch<_Float16>(s, p, *cache, a, q, out);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
