/*
 * attn8_decode.hip -- attention of one new token a sequence over a paged
 * cache in 8 bits (nmoe_attn8_decode, nmoe_attn8_decode_rows).
 *
 * One pass over keys and values with a running maximum and sum, a sequence cut
 * into parts that are joined afterwards, as over the cache in 16 bits
 * (attn_decode.hip), and bound by the cache's bytes as there, of which there
 * are half as many: 2 D a key for 4 D flops a query head.
 *
 * A code times its scale is a bf16 exactly, so codes are made bf16 in registers
 * (two an instruction, which takes the scale along) and the products are those
 * of bf16.
 *
 * 64 sequences of about 4096 on 16 + 2 heads of 256 (275 MB): 57 us, 4.9 TB/s,
 * as a copy; one of 131071 on 32 + 8 of 128 (268 MB): 49.  One of 777: 9.4, two
 * launches and a chain of length, page, key, product.
 */
#include <type_traits>

#include "nmoe_attn8.h"
#include "nmoe_decode.h"

#define NMOE_DEC8_NT 2      /* cache policy: read once (nt) */
/* Steps up to which one of many sequences is not cut (255 of 512 and one of 131071: 60 us, with 4 58, with 64 117): of many
 * that are evenly long a share is three quarters of one, and none is to be cut for that. */
#define NMOE_DEC8_WHOLE 16
#define NMOE_DEC8_JOINED 32 /* most pieces that a group of the join's threads goes over */
/* Scales of values up to which weights are at most 1: a sum over 2^30 keys of 448 times that is below 2^127.  A key whose
 * value has a larger one counts for the running maximum as if its score were larger by the scale's power beyond this, so that no
 * weight times value is above that either; what has no weight, or is not seen, raises nothing. */
#define NMOE_DEC8_TOP 88
#define NMOE_DEC8_SEQS 4096 /* sequences whose lengths every block looks through: 16 a thread */

/* Dies that pieces are dealt over, so that all heads of a piece are on one: with
 * heads of 64 two lie in a line of 128 bytes, which two dies would fetch each (64
 * sequences of 8000 on 8 + 8 heads: 193 us, now 162; on 8 + 2: 52, 40).  Longer
 * heads are as they come, neighbouring ones on different dies (64 of 4096 on 32 +
 * 8 of 128: 114 us, together 117).  A cache laid out head by head within a page
 * is read faster than either: 104 us, 97. */
template <int D>
constexpr int nmoe_dec8_dies = D == 64 ? 8 : 1;

/* The 16-byte chunks of a key's row are stored at chunk ^ f(row), so that 8
 * rows' same chunk lies in 8 different places of the banks (256 bytes wide: 1,
 * 2 or 4 rows). */
template <int D>
__device__ __forceinline__ int nmoe_dec8_swizzle(int row) {
    return D == 64 ? (row >> 2) & 3 : row & 7;
}

/* What codes 0, 1 (HI: 2, 3) of a word stand for, as two bf16. */
template <bool HI>
__device__ __forceinline__ uint32_t nmoe_kv8_pair(uint32_t c, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, HI));
}

/* 8 codes as a matrix operand. */
__device__ __forceinline__ nmoe_u4 nmoe_kv8_operand(uint32_t c0, uint32_t c1, float scale) {
    return nmoe_u4{nmoe_kv8_pair<false>(c0, scale), nmoe_kv8_pair<true>(c0, scale), nmoe_kv8_pair<false>(c1, scale),
                   nmoe_kv8_pair<true>(c1, scale)};
}

/* How sequences are cut, by their lengths: into pieces of at most `cap` steps
 * of 128 keys, the same for all, numbered one sequence behind the other; block
 * x of a key head's tile has piece x.  With G blocks running at once and T
 * steps: for one sequence cap is T / G, whatever max_len says (8000 keys under
 * a max_len of 2^20: 11.5 us, in pieces by that 96.8); for up to G / 2 sequences cap is T / (G - nseq / 2) if that makes no
 * more than G pieces, and T / (G - nseq), which never makes more, if not; for
 * more, sequences are pieces by themselves and only those longer than 16 steps
 * and than one and a half shares are cut: G + nseq blocks do for any lengths.
 * One number of parts for all, from the longest's length, leaves a long
 * sequence among short ones to a few blocks; dealt out to the step, with the
 * end of one sequence and the beginning of the next in one block, evenly long
 * ones were slower (256 of 512 tokens 45 us instead of 29). */
struct nmoe_dec8_piece {
    int b, i, n, first; /* the sequence, which piece of it, how many it has, its first one's number */
    int cap;
};

/* Sequence b's row of q and out: b, or with offsets the last of its rows; -1: it has none. */
struct nmoe_dec8_rows {
    const int32_t *cu;
    int ntok;
    __device__ __forceinline__ int of(int b) const {
        if (cu == NULL) return b;
        const int end = min(max(cu[b + 1], 0), ntok);
        return min(max(cu[b], 0), ntok) < end ? end - 1 : -1;
    }
};

__device__ __forceinline__ int nmoe_dec8_steps(const int32_t *lens, const nmoe_dec8_rows &rows, int b, int max_pages, int page_size) {
    if (rows.of(b) < 0) return 1;
    const int len = nmoe_len_of(lens[b], max_pages, page_size);
    return len <= 0 ? 1 : (len + NMOE_DEC_STEP - 1) / NMOE_DEC_STEP; /* one of none is a piece too */
}

__device__ __forceinline__ int64_t nmoe_dec8_scan(int64_t v, int64_t *scratch, int64_t &total) {
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t u = __shfl_up(v, d, 64);
        if (lane >= d) v += u;
    }
    if (lane == 63) scratch[threadIdx.x / 64] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < NMOE_DEC_WAVES; w++) {
        if (w < (int)threadIdx.x / 64) v += scratch[w];
        total += scratch[w];
    }
    return v;
}

/* Piece x; n = 0: there are not so many. */
__device__ __forceinline__ nmoe_dec8_piece nmoe_dec8_find(const int32_t *lens, const nmoe_dec8_rows &rows, int nseq, int max_pages, int page_size,
                                                           int x, int at_once) {
    constexpr int THREADS = 64 * NMOE_DEC_WAVES;
    __shared__ int64_t s_steps[NMOE_DEC_WAVES], s_pieces[NMOE_DEC_WAVES];
    __shared__ int s_found[4];
    if (nseq == 1) {
        const int steps = nmoe_dec8_steps(lens, rows, 0, max_pages, page_size), cap = (steps + at_once - 1) / at_once;
        const int n = (steps + cap - 1) / cap;
        return {0, x, x < n ? n : 0, 0, cap};
    }
    const int each = (nseq + THREADS - 1) / THREADS, b0 = min((int)threadIdx.x * each, nseq), b1 = min(b0 + each, nseq);
    int64_t steps = 0, all;
    for (int b = b0; b < b1; b++) steps += nmoe_dec8_steps(lens, rows, b, max_pages, page_size);
    nmoe_dec8_scan(steps, s_steps, all);
    const auto share = [&](int blocks) { return (int)min((all + blocks - 1) / blocks, (int64_t)NMOE_LONGEST / NMOE_DEC_STEP); };
    const bool few = 2 * nseq <= at_once;
    const int cap0 = few ? share(at_once - nseq / 2) : max(share(2 * at_once / 3), NMOE_DEC8_WHOLE), cap1 = few ? share(at_once - nseq) : cap0;
    int64_t pieces = 0, total; /* with cap0, and with cap1 in the upper half */
    for (int b = b0; b < b1; b++) {
        const int n = nmoe_dec8_steps(lens, rows, b, max_pages, page_size);
        pieces += (n + cap0 - 1) / cap0 + ((int64_t)((n + cap1 - 1) / cap1) << 32);
    }
    if (threadIdx.x == 0) s_found[2] = 0;
    const int64_t sum = nmoe_dec8_scan(pieces, s_pieces, total);
    const bool fits = !few || (int)(uint32_t)total <= at_once;
    const int cap = fits ? cap0 : cap1, mine = (int)(fits ? (uint32_t)pieces : pieces >> 32), upto = (int)(fits ? (uint32_t)sum : sum >> 32);
    if (x >= upto - mine && x < upto) {
        int at = upto - mine, b = b0, n = (nmoe_dec8_steps(lens, rows, b, max_pages, page_size) + cap - 1) / cap;
        while (at + n <= x) {
            at += n;
            b++;
            n = (nmoe_dec8_steps(lens, rows, b, max_pages, page_size) + cap - 1) / cap;
        }
        s_found[0] = b;
        s_found[1] = x - at;
        s_found[2] = n;
        s_found[3] = at;
    }
    __syncthreads();
    return {s_found[0], s_found[1], s_found[2], s_found[3], cap};
}

/* One block a piece, a key head and up to 16 of its query heads, which are the
 * columns of the matrix instructions (16x16x32); its wavefronts take tiles of
 * 32 keys, two blocks of the cache, in turn.
 *
 * Scores: S^T (keys x heads) = K Q^T.  K's rows go to LDS directly, into a
 * buffer of the wavefront's own: the next tile's when this one's have been
 * read.  Lane (r, c) = (l % 16, l / 16) reads 16 bytes of key r at a time, the
 * operands of two products: of dimensions 64 k + 16 c .. + 16, the same as of q.
 * A lane then holds, of its head r, the scores of keys 16 a + 4 c + i (a < 2,
 * i < 4), which is the order the second product takes its 32 keys in.  O^T
 * (dimensions x heads) = V^T P^T needs 8 keys of one dimension in a lane: lane
 * (r, c) reads D / 16 bytes, dimensions D / 16 r .., of its 8 keys and pairs
 * the bytes of neighbouring keys; product dd has the dimensions D / 16 r + dd
 * as its rows.
 * With f16, q and the weights have 11 bits: two terms of 8, two products.
 * Keys behind the end: their addresses are the last key's, their scores
 * -inf, their values zero. */
template <typename T, int D>
__global__ void __launch_bounds__(64 * NMOE_DEC_WAVES, 2)
    nmoe_attn8_decode_kernel(nmoe_hip_kv8_cache cache, const T *q, int q_heads, int tiles, nmoe_dec8_rows rows,
                             const int32_t *seq_lens, int nseq, const int32_t *page_table, int max_pages, int at_once, int likely, float scale2,
                             T *out, float *lse, float *part_o, float *part_ml, int2 *cuts) {
    typedef nmoe_mat<nmoe_bf16> X;
    constexpr int TERMS = nmoe_elem<T>::dtype == NMOE_HIP_F16 ? 2 : 1;
    constexpr int KS = D / 32, DD = D / 16, VW = D / 64; /* products of the scores, of the output; words of a value's lane */
    constexpr int CH = D / 16, RPI = 64 / CH, NI = NMOE_DEC_TILE / RPI; /* chunks of a row, rows and loads of a tile of K */
    /* the wavefronts' tiles of K, in the end their outputs */
    __shared__ alignas(16) char s_kv[NMOE_DEC_WAVES * NMOE_DEC_HEADS * D * 4];
    static_assert(NMOE_DEC_TILE * D <= NMOE_DEC_HEADS * D * 4, "tiles fit");
    __shared__ float s_m[NMOE_DEC_WAVES][NMOE_DEC_HEADS], s_l[NMOE_DEC_WAVES][NMOE_DEC_HEADS];
    __shared__ int s_bad;
    float(*s_o)[NMOE_DEC_HEADS][D] = (float(*)[NMOE_DEC_HEADS][D])s_kv;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, c = lane / 16;
    constexpr int DIES = nmoe_dec8_dies<D>;
    const int units = tiles * cache.kv_heads, unit = blockIdx.x / DIES % units, tile = unit % tiles, kh = unit / tiles;
    const int x = blockIdx.x / (DIES * units) * DIES + blockIdx.x % DIES;
    if (at_once == 0 && x >= nseq) return;
    const int group = q_heads / cache.kv_heads, h0 = kh * group + tile * NMOE_DEC_HEADS;
    const int heads = min(group - tile * NMOE_DEC_HEADS, NMOE_DEC_HEADS);
    /* one sequence: the first tile's page numbers beside its length, where the piece begins if max_len is that; else they
     * are looked up once more */
    const int guess = (int)min((int64_t)x * likely * NMOE_DEC_STEP, (int64_t)NMOE_LONGEST) + w * NMOE_DEC_TILE;
    int early[2] = {0, 0};
    if (nseq == 1) {
#pragma unroll
        for (int a = 0; a < 2; a++) early[a] = page_table[min((uint32_t)(guess + 16 * a) / (uint32_t)cache.page_size, (uint32_t)max_pages - 1)];
    }
    /* at_once 0: a block a sequence */
    const nmoe_dec8_piece piece = at_once == 0 ? nmoe_dec8_piece{x, 0, 1, x, NMOE_LONGEST / NMOE_DEC_STEP}
                                               : nmoe_dec8_find(seq_lens, rows, nseq, max_pages, cache.page_size, x, at_once);
    if (piece.n == 0) return;
    const int b = piece.b, len = nmoe_len_of(seq_lens[b], max_pages, cache.page_size);
    if (at_once != 0 && piece.i == 0 && unit == 0 && tid == 0) cuts[b] = int2{piece.first, piece.n};
    const int qrow = rows.of(b);
    if (qrow < 0) return;
    const int32_t *table = page_table + (int64_t)b * max_pages;
    nmoe_u4 qf[TERMS][KS];
    const T *qr = q + ((int64_t)qrow * q_heads + h0 + min(r, heads - 1)) * D + 16 * c;
#pragma unroll
    for (int k = 0; k < KS; k++) {
        const T *p = qr + 64 * (k / 2) + 8 * (k % 2);
        if constexpr (TERMS == 1)
            qf[0][k] = *(const nmoe_u4 *)p;
        else {
            float x[8], hi[8], lo[8];
            nmoe_load<T, 8>(p, x);
#pragma unroll
            for (int i = 0; i < 8; i++) nmoe_two_terms(x[i], hi[i], lo[i]);
            qf[0][k] = X::pack(hi);
            qf[TERMS - 1][k] = X::pack(lo);
        }
#pragma unroll
        for (int t = 0; t < TERMS; t++)
            if (r >= heads) qf[t][k] = nmoe_u4{0, 0, 0, 0};
    }
    const int64_t first = (int64_t)piece.i * piece.cap * NMOE_DEC_STEP;
    const int begin = (int)first, end = (int)min((int64_t)max(len, 0), first + (int64_t)piece.cap * NMOE_DEC_STEP);
    if (tid == 0) s_bad = len < 0;

    nmoe_f4 o[DD];
#pragma unroll
    for (int i = 0; i < DD; i++) o[i] = nmoe_f4{0, 0, 0, 0};
    float m = -3.402823466e38f, l = 0.0f; /* finite, so that a key whose score is -infinity weighs 0 also where no other is */
    bool bad = false;

    const uint8_t *kb = (const uint8_t *)cache.k + kh * cache.head_stride, *vb = (const uint8_t *)cache.v + kh * cache.head_stride;
    const uint32_t step = (uint32_t)cache.token_stride; /* bytes from a key to the next of its page */
    const int last16 = end > begin ? (end - 1) & ~15 : 0;
    const int t0 = begin + w * NMOE_DEC_TILE;
    /* a tile lies in two halves of 16 keys, each a block of one page */
    auto page_of = [&](int t, int a) { return table[(uint32_t)min(t + 16 * a, last16) / (uint32_t)cache.page_size]; };
    auto row_of = [&](int t, int a, int page, float &ks, float &vs) {
        page = __builtin_amdgcn_readfirstlane(page);
        if ((uint32_t)page >= (uint32_t)cache.num_pages) {
            bad = true;
            page = 0;
        }
        const int token = (int)((uint32_t)min(t + 16 * a, last16) % (uint32_t)cache.page_size);
        const int64_t at = nmoe_kv8_scale_at(cache, page, token, kh);
        ks = cache.k_scale[at];
        vs = cache.v_scale[at];
        return page * cache.page_stride + (int64_t)token * cache.token_stride;
    };
    auto top_of = [&](int t, int a) { return min(end - 1 - min(t + 16 * a, last16), 15); }; /* a half's last key */
    uint8_t *sk = (uint8_t *)s_kv + w * NMOE_DEC_TILE * D;
    const uint32_t chunk = (uint32_t)((lane % CH) ^ nmoe_dec8_swizzle<D>(lane / CH)) * 16;
    auto load_k = [&](int t, const int64_t (&row)[2]) {
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const __amdgpu_buffer_rsrc_t k = nmoe_buffer(kb + row[a]);
            const int top = top_of(t, a);
#pragma unroll
            for (int i = 0; i < NI / 2; i++) {
                const int at = i * RPI + lane / CH;
                /* the swizzle goes by the row's last bits: the same for rows 8 apart (heads of 64: 16) */
                const uint32_t ch = RPI % 8 == 0 ? chunk : (uint32_t)((lane % CH) ^ nmoe_dec8_swizzle<D>(at)) * 16;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(k, (__attribute__((address_space(3))) void *)(sk + (a * 16 + i * RPI) * D),
                                                         16, (int)((uint32_t)min(at, top) * step + ch), 0, 0, NMOE_DEC8_NT);
            }
        }
    };
    int64_t row[2] = {0, 0};
    float ks[2], vs[2];
    auto work = [&](const int t, auto last) {
        constexpr bool LAST = decltype(last)::value;
        int next[2];
        if (!LAST) {
#pragma unroll
            for (int a = 0; a < 2; a++) next[a] = page_of(t + NMOE_DEC_STEP, a);
        }
        asm volatile("" ::: "memory");
        uint32_t vf[8][VW];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const __amdgpu_buffer_rsrc_t v = nmoe_buffer(vb + row[a]);
            const int top = top_of(t, a);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = (int)((uint32_t)min(4 * c + i, top) * step + DD * r);
                if constexpr (D == 256) {
                    const nmoe_u4 y = __builtin_amdgcn_raw_buffer_load_b128(v, at, 0, NMOE_DEC8_NT);
#pragma unroll
                    for (int x = 0; x < 4; x++) vf[4 * a + i][x] = y[x];
                } else if constexpr (D == 128) {
                    const auto y = __builtin_amdgcn_raw_buffer_load_b64(v, at, 0, NMOE_DEC8_NT);
                    vf[4 * a + i][0] = y[0];
                    vf[4 * a + i][1] = y[1];
                } else
                    vf[4 * a + i][0] = __builtin_amdgcn_raw_buffer_load_b32(v, at, 0, NMOE_DEC8_NT);
            }
        }
        nmoe_dec_wait_vm<8>(); /* K has come, these values may be on their way */
        float s[8];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            nmoe_f4 x = {0, 0, 0, 0};
            const uint8_t *p = sk + (16 * a + r) * D;
            const int f = nmoe_dec8_swizzle<D>(r);
#pragma unroll
            for (int k = 0; k < KS / 2; k++) {
                const nmoe_u4 y = *(const nmoe_u4 *)(p + ((4 * k + c) ^ f) * 16);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const nmoe_u4 z = nmoe_kv8_operand(y[2 * u], y[2 * u + 1], ks[a]);
#pragma unroll
                    for (int n = 0; n < TERMS; n++) x = X::mma16(z, qf[n][2 * k + u], x);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * a + i] = x[i] * scale2;
        }
        const float held[2] = {vs[0], vs[1]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (!LAST) {
#pragma unroll
            for (int a = 0; a < 2; a++) row[a] = row_of(t + NMOE_DEC_STEP, a, next[a], ks[a], vs[a]);
            load_k(t + NMOE_DEC_STEP, row);
        } else if (t + NMOE_DEC_TILE > end) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (t + 16 * (j / 4) + 4 * c + j % 4 >= end) {
                    s[j] = -INFINITY;
#pragma unroll
                    for (int v = 0; v < VW; v++) vf[j][v] = 0;
                }
        }
        float mt = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        if (fmaxf(held[0], held[1]) > nmoe_kv8_two_to(NMOE_DEC8_TOP)) { /* of the wavefront */
            mt = -INFINITY;
#pragma unroll
            for (int a = 0; a < 2; a++)
                mt = fmaxf(mt, fmaxf(fmaxf(s[4 * a], s[4 * a + 1]), fmaxf(s[4 * a + 2], s[4 * a + 3])) + nmoe_kv8_beyond(held[a], NMOE_DEC8_TOP));
        }
        mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        if (__any(mt > m)) {
            const float mn = fmaxf(m, mt), a = nmoe_exp2(m - mn);
            m = mn;
            l *= a;
#pragma unroll
            for (int i = 0; i < DD; i++) o[i] *= a;
        }
        float hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            s[j] = nmoe_exp2(s[j] - m);
            l += s[j];
            nmoe_two_terms(s[j], hi[j], lo[j]);
        }
        nmoe_u4 pf[TERMS]; /* bf16: to its 8 bits, as over a cache in 16; l has them in fp32 */
        pf[0] = X::pack(hi);
        if constexpr (TERMS == 2) pf[1] = X::pack(lo);
#pragma unroll
        for (int v = 0; v < VW; v++) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                /* of keys 4 a + 2 x, + 1: bytes 2 u, 2 u + 1 of both, side by side */
                uint32_t y[4];
#pragma unroll
                for (int x = 0; x < 4; x++) y[x] = __builtin_amdgcn_perm(vf[2 * x + 1][v], vf[2 * x][v], u ? 0x07030602 : 0x05010400);
                const nmoe_u4 even = {nmoe_kv8_pair<false>(y[0], held[0]), nmoe_kv8_pair<false>(y[1], held[0]),
                                      nmoe_kv8_pair<false>(y[2], held[1]), nmoe_kv8_pair<false>(y[3], held[1])};
                const nmoe_u4 odd = {nmoe_kv8_pair<true>(y[0], held[0]), nmoe_kv8_pair<true>(y[1], held[0]),
                                     nmoe_kv8_pair<true>(y[2], held[1]), nmoe_kv8_pair<true>(y[3], held[1])};
#pragma unroll
                for (int n = 0; n < TERMS; n++) {
                    o[4 * v + 2 * u] = X::mma16(even, pf[n], o[4 * v + 2 * u]);
                    o[4 * v + 2 * u + 1] = X::mma16(odd, pf[n], o[4 * v + 2 * u + 1]);
                }
            }
        }
    };
    if (t0 < end) {
#pragma unroll
        for (int a = 0; a < 2; a++)
            row[a] = row_of(t0, a, nseq != 1 || t0 != guess ? page_of(t0, a) : t0 + 16 * a <= last16 ? early[a] : early[0], ks[a], vs[a]);
        load_k(t0, row);
        int t = t0;
        /* the last tile on its own: with a path that loads no next one, a wait for values would be one for the next keys */
        for (; (int64_t)t + NMOE_DEC_STEP < end; t += NMOE_DEC_STEP) work(t, std::false_type());
        work(t, std::true_type());
    }
    __syncthreads(); /* the tiles of K are read, s_bad is set */
    if (bad) s_bad = 1;

    /* the wavefronts' parts; a lane's l covers its own keys only */
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (c == 0) {
        s_m[w][r] = m;
        s_l[w][r] = l;
    }
    if (r < heads) {
#pragma unroll
        for (int dd = 0; dd < DD; dd++)
#pragma unroll
            for (int i = 0; i < 4; i++) s_o[w][r][DD * (4 * c + i) + dd] = o[dd][i];
    }
    __syncthreads();
    const bool whole = piece.n == 1;
    for (int y4 = tid; y4 < heads * D / 4; y4 += 64 * NMOE_DEC_WAVES) {
        const int h = y4 / (D / 4), d = y4 % (D / 4) * 4;
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
        const int64_t oh = (int64_t)qrow * q_heads + h0 + h;
        if (s_bad) lj = NAN;
        if (whole) {
            float z[4];
#pragma unroll
            for (int i = 0; i < 4; i++) z[i] = len == 0 ? 0.0f : y[i] / lj;
            nmoe_store<T, 4>(out + oh * D + d, z);
            if (lse != NULL && d == 0) lse[oh] = len == 0 ? -INFINITY : 0.69314718055994531f * (mj + log2f(lj));
        } else {
            const int64_t at = (int64_t)x * q_heads + h0 + h;
            *(nmoe_f4 *)(part_o + at * D + d) = y;
            if (d == 0) {
                part_ml[2 * at] = mj;
                part_ml[2 * at + 1] = lj;
            }
        }
    }
}

/* Joins a head's pieces: 256 / (D / 4) groups of threads take them in turn,
 * 4 dimensions a thread. */
template <typename T, int D>
__global__ void __launch_bounds__(NMOE_DEC_JOIN)
    nmoe_attn8_decode_join_kernel(int q_heads, nmoe_dec8_rows rows, const float *part_o, const float *part_ml, const int2 *cuts, T *out, float *lse) {
    constexpr int LANES = D / 4, GROUPS = NMOE_DEC_JOIN / LANES;
    __shared__ nmoe_f4 s_y[GROUPS][LANES];
    __shared__ float s_m[GROUPS], s_l[GROUPS];
    const int tid = threadIdx.x, h = blockIdx.x % q_heads, b = blockIdx.x / q_heads, w = tid / LANES, d = tid % LANES;
    const int2 cut = cuts[b];
    if (cut.y < 2) return; /* written by its one piece, or without a row */
    float m = -INFINITY, l = 0.0f;
    nmoe_f4 y = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = w; i < cut.y; i += GROUPS) {
        const int64_t at = (int64_t)(cut.x + i) * q_heads + h;
        const float mx = part_ml[2 * at], lx = part_ml[2 * at + 1], mn = fmaxf(m, mx);
        const float fa = nmoe_exp2(m - mn), fb = nmoe_exp2(mx - mn);
        y = fa * y + fb * *(const nmoe_f4 *)(part_o + at * D + 4 * d);
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
        const float mn = fmaxf(m, s_m[i]), fa = nmoe_exp2(m - mn), fb = nmoe_exp2(s_m[i] - mn); /* the first has a piece */
        y = fa * y + fb * s_y[i][d];
        l = fa * l + fb * s_l[i];
        m = mn;
    }
    const int64_t oh = (int64_t)rows.of(b) * q_heads + h;
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; i++) z[i] = y[i] / l;
    nmoe_store<T, 4>(out + oh * D + 4 * d, z);
    if (lse != NULL && d == 0) lse[oh] = 0.69314718055994531f * (m + log2f(l));
}

static int nmoe_dec8_tiles(int kv_heads, int q_heads) { return (q_heads / kv_heads + NMOE_DEC_HEADS - 1) / NMOE_DEC_HEADS; }

/* Blocks a key head's tile of query heads: `at_once` of them run at once, two a
 * CU with heads of 256, which is as many as there are by LDS and registers (64
 * sequences of about 4096: 56, 63, 65, 62 us with 2, 3, 4, 6), and for up to 4
 * sequences (one of 131071 on 32 + 8 heads of 128: 50 us, with four 54; 4 of about
 * 9000: 17.0, 17.7), four else (64 of 4096: 114, with two 118; 30 of 3000: 42,
 * 45).  No more than the join goes over soon (one of 30000 on 16 + 2 of 256, 235
 * pieces 21 us, 118 16; of 120000 on 8 + 1 of 64: 18.5, 14.4).  From
 * NMOE_DEC8_SEQS sequences on a sequence is a piece. */
struct nmoe_dec8_plan {
    int at_once, likely;
    int64_t blocks;
};

static nmoe_dec8_plan nmoe_dec8_plan_of(const nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *c, int q_heads, int nseq, int max_len) {
    nmoe_dec8_plan p = {0, 0, nseq};
    if (nseq > NMOE_DEC8_SEQS) return p;
    const int64_t units = (int64_t)c->kv_heads * nmoe_dec8_tiles(c->kv_heads, q_heads);
    const int64_t want = (c->head_dim == 256 || nseq <= 4 ? 2 : 4) * (ctx->num_cus > 0 ? ctx->num_cus : 256);
    if (nseq * units >= want && max_len <= NMOE_DEC8_WHOLE * NMOE_DEC_STEP) return p; /* none is worth cutting */
    p.at_once = (int)(want > 2 * units ? want / units : 2);
    const int most = NMOE_DEC8_JOINED * (NMOE_DEC_JOIN / (c->head_dim / 4)); /* pieces of a sequence */
    if (p.at_once > (int64_t)nseq * most) p.at_once = nseq * most;
    p.blocks = 2 * (int64_t)nseq <= p.at_once ? p.at_once : (int64_t)p.at_once + nseq;
    const int64_t steps = max_len > NMOE_DEC_STEP ? ((int64_t)max_len + NMOE_DEC_STEP - 1) / NMOE_DEC_STEP : 1;
    p.likely = nseq == 1 ? (int)((steps + p.at_once - 1) / p.at_once) : 0;
    return p;
}

/* A partial row a head and piece, and where each sequence's are: whatever the
 * lengths are, and never less for more sequences. */
static size_t nmoe_dec8_bytes(const nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *c, int q_heads, int nseq) {
    if (nseq > NMOE_DEC8_SEQS) nseq = NMOE_DEC8_SEQS;
    const nmoe_dec8_plan p = nmoe_dec8_plan_of(ctx, c, q_heads, nseq, NMOE_LONGEST);
    return (size_t)p.blocks * q_heads * (c->head_dim + 2) * sizeof(float) + (size_t)nseq * sizeof(int2);
}

template <typename T, int D>
static void nmoe_dec8_launch_as(hipStream_t s, const nmoe_dec8_plan &p, const nmoe_hip_kv8_cache &c, const void *q, int q_heads,
                                int nseq, const nmoe_dec8_rows &rows, const int32_t *lens, const int32_t *table, int max_pages, float scale, void *out,
                                float *lse, void *ws) {
    constexpr int DIES = nmoe_dec8_dies<D>;
    const int tiles = nmoe_dec8_tiles(c.kv_heads, q_heads);
    float *po = (float *)ws, *pml = po + (size_t)p.blocks * q_heads * D;
    int2 *cuts = (int2 *)(pml + 2 * (size_t)p.blocks * q_heads);
    hipLaunchKernelGGL((nmoe_attn8_decode_kernel<T, D>), dim3((uint32_t)((p.blocks + DIES - 1) / DIES * DIES * c.kv_heads * tiles)),
                       dim3(64 * NMOE_DEC_WAVES), 0, s, c, (const T *)q, q_heads, tiles, rows, lens, nseq, table, max_pages, p.at_once, p.likely,
                       scale * 1.44269504088896341f, (T *)out, lse, po, pml, cuts);
    if (p.at_once != 0)
        hipLaunchKernelGGL((nmoe_attn8_decode_join_kernel<T, D>), dim3((uint32_t)nseq * q_heads), dim3(NMOE_DEC_JOIN), 0, s, q_heads,
                           rows, po, pml, cuts, (T *)out, lse);
}

template <typename T>
static void nmoe_dec8_launch(hipStream_t s, const nmoe_dec8_plan &p, const nmoe_hip_kv8_cache &c, const void *q, int q_heads, int nseq,
                             const nmoe_dec8_rows &rows, const int32_t *lens, const int32_t *table, int max_pages, float scale, void *out, float *lse,
                             void *ws) {
    if (c.head_dim == 64)
        nmoe_dec8_launch_as<T, 64>(s, p, c, q, q_heads, nseq, rows, lens, table, max_pages, scale, out, lse, ws);
    else if (c.head_dim == 128)
        nmoe_dec8_launch_as<T, 128>(s, p, c, q, q_heads, nseq, rows, lens, table, max_pages, scale, out, lse, ws);
    else
        nmoe_dec8_launch_as<T, 256>(s, p, c, q, q_heads, nseq, rows, lens, table, max_pages, scale, out, lse, ws);
}

int nmoe_attn8_check_heads(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const char *what, int q_heads, int nseq) {
    int rc = nmoe_check_cache8(ctx, cache);
    if (rc != NMOE_HIP_OK) return rc;
    if (q_heads < 1 || q_heads > NMOE_MAX_HEADS || q_heads % cache->kv_heads != 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "%s: %d query heads on %d key heads (1..%d, a multiple)", what, q_heads,
                         cache->kv_heads, NMOE_MAX_HEADS);
    if (nseq < 0 || (int64_t)nseq * q_heads > NMOE_MAX_ROWS)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "%s: %d sequences of %d heads outside 0..2^22", what, nseq, q_heads);
    return NMOE_HIP_OK;
}

int nmoe_attn8_check(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const char *what, const void *q, int q_dtype,
                     int q_heads, int nseq, const int32_t *seq_lens, const int32_t *page_table, int max_pages, float scale,
                     const void *out, const float *lse) {
    int rc = nmoe_attn8_check_heads(ctx, cache, what, q_heads, nseq);
    if (rc != NMOE_HIP_OK) return rc;
    if (!nmoe_is_half(q_dtype)) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "%s: q_dtype %d is neither bf16 nor f16", what, q_dtype);
    if (q == NULL || out == NULL || seq_lens == NULL || page_table == NULL || !nmoe_aligned(q, 16) || !nmoe_aligned(out, 16) ||
        !nmoe_aligned(lse, 4) || !nmoe_aligned(seq_lens, 4) || !nmoe_aligned(page_table, 4))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "%s: q and out (16-byte aligned), seq_lens and page_table are required", what);
    if (max_pages < 1 || !nmoe_scale_ok(scale))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "%s: max_pages >= 1 and a scale below 2^127 are required", what);
    if (cache->token_stride >= NMOE_KV8_STRIDE)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "%s: the cache's token stride is below %d bytes", what, NMOE_KV8_STRIDE);
    return NMOE_HIP_OK;
}

extern "C" size_t nmoe_attn8_decode_workspace(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, int q_heads, int nseq,
                                              int max_len) {
    if (ctx == NULL || nmoe_attn8_check_heads(ctx, cache, "decode", q_heads, nseq) != NMOE_HIP_OK || nseq == 0 || max_len < 0)
        return 0;
    return nmoe_dec8_bytes(ctx, cache, q_heads, nseq);
}

static int nmoe_dec8_call(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const void *q, int q_dtype, int q_heads, int nseq,
                          const nmoe_dec8_rows &rows, const int32_t *seq_lens, const int32_t *page_table, int max_pages, int max_len,
                          float scale, void *out, float *lse, void *ws, size_t ws_bytes, void *stream) {
    int rc = nmoe_attn8_check(ctx, cache, "decode", q, q_dtype, q_heads, nseq, seq_lens, page_table, max_pages, scale, out, lse);
    if (rc != NMOE_HIP_OK) return rc;
    if (max_len < 0) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: max_len %d < 0", max_len);
    if (nseq == 0 || (rows.cu != NULL && rows.ntok == 0)) return NMOE_HIP_OK;
    const nmoe_dec8_plan p = nmoe_dec8_plan_of(ctx, cache, q_heads, nseq, max_len);
    const size_t need = p.at_once != 0 ? nmoe_dec8_bytes(ctx, cache, q_heads, nseq) : 0;
    if (need != 0 && (ws == NULL || !nmoe_aligned(ws, 16) || ws_bytes < need))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: a workspace of %zu bytes (16-byte aligned) is required, %zu given", need,
                         ws == NULL ? (size_t)0 : ws_bytes);
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (q_dtype == NMOE_HIP_BF16)
        nmoe_dec8_launch<nmoe_bf16>(s, p, *cache, q, q_heads, nseq, rows, seq_lens, page_table, max_pages, scale, out, lse, ws);
    else
        nmoe_dec8_launch<_Float16>(s, p, *cache, q, q_heads, nseq, rows, seq_lens, page_table, max_pages, scale, out, lse, ws);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}

extern "C" int nmoe_attn8_decode(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const void *q, int q_dtype, int q_heads,
                                 int nseq, const int32_t *seq_lens, const int32_t *page_table, int max_pages, int max_len,
                                 float scale, void *out, float *lse, void *ws, size_t ws_bytes, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    return nmoe_dec8_call(ctx, cache, q, q_dtype, q_heads, nseq, nmoe_dec8_rows{NULL, 0}, seq_lens, page_table, max_pages, max_len,
                          scale, out, lse, ws, ws_bytes, stream);
}

extern "C" int nmoe_attn8_decode_rows(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *cache, const void *q, int q_dtype, int q_heads,
                                      int nseq, const int32_t *cu, int ntok, const int32_t *seq_lens, const int32_t *page_table,
                                      int max_pages, int max_len, float scale, void *out, float *lse, void *ws, size_t ws_bytes,
                                      void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    if (cu == NULL || !nmoe_aligned(cu, 4) || ntok < 0 || ntok > NMOE_MAX_ROWS)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "decode: cu (4-byte aligned) and 0 <= ntok <= 2^22 are required");
    return nmoe_dec8_call(ctx, cache, q, q_dtype, q_heads, nseq, nmoe_dec8_rows{cu, ntok}, seq_lens, page_table, max_pages, max_len,
                          scale, out, lse, ws, ws_bytes, stream);
}
