/*
 * delta.hip -- the gated delta rule, one token a sequence (nmoe_delta_step)
 * and over packed prompts (nmoe_delta_prompt).
 */
#include "nmoe_context.h"

#define NMOE_DELTA_MIN_G (-100.0f)
#define NMOE_DELTA_TOKENS (1 << 30)
#define NMOE_DELTA_HEADS (1 << 19) /* sequences x heads: with 8 blocks of 512 threads each a launch's threads stay below 2^32 */

/* The decay's logarithm, held above -100; NaN stays NaN. */
__device__ __forceinline__ float nmoe_delta_g(float g) { return g < NMOE_DELTA_MIN_G ? NMOE_DELTA_MIN_G : g; }

/* ---------------------------------------------------- one token a sequence
 *
 * With a = S^T k and o = S^T q of the old state, both scaled by e^g,
 *   u = beta (v - a),  S <- e^g S + k u^T,  out = scale (o + (q.k) u):
 * one pass, each value of the state read and written once, which is its bound:
 * 200 sequences of 32 heads of 128 x 128 are 844 MB in 156 us, 5.4 TB/s; one,
 * 4.0 us, is the launch.  The stores are marked as not soon read (160 us
 * without); the loads are not, as 20 sequences' states, which the memory-side
 * cache can still hold, then took 17.6 us instead of 14.2 (and 200 152).
 * One block a sequence, head and COLS columns of the state: thread (r, c) has
 * 4 neighbouring columns of the rows r, r + R, ... */
template <typename T, int DK, int DV, int COLS>
__global__ void __launch_bounds__(256)
    nmoe_delta_step_kernel(nmoe_hip_delta_rule d) {
    constexpr int L = COLS / 4, R = 256 / L, N = DK / R;
    __shared__ float s_q[DK], s_k[DK], s_n[3];
    __shared__ nmoe_f4 s_part[2][4][L];
    const int slice = blockIdx.x % (DV / COLS), bh = blockIdx.x / (DV / COLS);
    const int b = bh / d.v_heads, h = bh % d.v_heads, kh = h / (d.v_heads / d.k_heads);
    const int tid = threadIdx.x, c = tid % L, r = tid / L, col = slice * COLS + 4 * c;
    const int state = d.state_index != NULL ? d.state_index[b] : b;
    T *out = (T *)d.out + (int64_t)bh * DV + col;
    if (state < 0 || state >= d.num_states) {
        const float x = state < 0 ? 0.0f : NAN;
        const float z[4] = {x, x, x, x};
        if (r == 0) nmoe_store<T, 4>(out, z);
        return;
    }
    const int64_t at = ((int64_t)state * d.v_heads + h) * DK * DV + col;
    nmoe_f4 S[N];
#pragma unroll
    for (int i = 0; i < N; i++)
        S[i] = d.state_in != NULL ? *(const nmoe_f4 *)(d.state_in + at + (int64_t)(r + R * i) * DV) : nmoe_f4{0, 0, 0, 0};
    float v[4];
    nmoe_load<T, 4>((const T *)d.v + b * d.v_stride + h * DV + col, v);
    const float g = expf(nmoe_delta_g(d.g[bh])), beta = d.beta[bh];
    if (tid < 64) { /* q, k and their three products */
        float q[DK / 64], k[DK / 64], qq = 0.0f, kk = 0.0f, qk = 0.0f;
#pragma unroll
        for (int i = 0; i < DK / 64; i++) {
            q[i] = nmoe_elem<T>::get(((const T *)d.q)[b * d.q_stride + kh * DK + tid + 64 * i]);
            k[i] = nmoe_elem<T>::get(((const T *)d.k)[b * d.k_stride + kh * DK + tid + 64 * i]);
            s_q[tid + 64 * i] = q[i];
            s_k[tid + 64 * i] = k[i];
            qq += q[i] * q[i];
            kk += k[i] * k[i];
            qk += q[i] * k[i];
        }
        qq = nmoe_wave_sum_tree(qq);
        kk = nmoe_wave_sum_tree(kk);
        qk = nmoe_wave_sum_tree(qk);
        if (tid == 0) {
            s_n[0] = d.scale * (d.l2 ? rsqrtf(qq + d.eps) : 1.0f);
            s_n[1] = d.l2 ? rsqrtf(kk + d.eps) : 1.0f;
            s_n[2] = qk;
        }
    }
    __syncthreads();
    nmoe_f4 a = {0, 0, 0, 0}, o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < N; i++) {
        S[i] *= g;
        a += S[i] * s_k[r + R * i];
        o += S[i] * s_q[r + R * i];
    }
    /* over the rows: lanes of a wavefront, then the four wavefronts */
#pragma unroll
    for (int x = L; x < 64; x *= 2)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            a[e] += __shfl_xor(a[e], x, 64);
            o[e] += __shfl_xor(o[e], x, 64);
        }
    if (tid % 64 < L) {
        s_part[0][tid / 64][c] = a;
        s_part[1][tid / 64][c] = o;
    }
    __syncthreads();
    a = (s_part[0][0][c] + s_part[0][1][c]) + (s_part[0][2][c] + s_part[0][3][c]);
    const float nq = s_n[0], nk = s_n[1];
    nmoe_f4 u;
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = beta * nk * (v[e] - nk * a[e]);
#pragma unroll
    for (int i = 0; i < N; i++)
        __builtin_nontemporal_store(S[i] + s_k[r + R * i] * u, (nmoe_f4 *)(d.state_out + at + (int64_t)(r + R * i) * DV));
    if (r == 0) {
        o = (s_part[1][0][c] + s_part[1][1][c]) + (s_part[1][2][c] + s_part[1][3][c]);
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; e++) z[e] = nq * (o[e] + s_n[2] * u[e]);
        nmoe_store<T, 4>(out, z);
    }
}

template <typename T, int DK, int DV>
static void nmoe_delta_step_as(hipStream_t s, const nmoe_hip_delta_rule &d, int nseq) {
    const uint32_t heads = (uint32_t)nseq * d.v_heads;
    hipLaunchKernelGGL((nmoe_delta_step_kernel<T, DK, DV, 32>), dim3(heads * (DV / 32)), dim3(256), 0, s, d);
}

template <typename T>
static void nmoe_delta_launch(hipStream_t s, const nmoe_hip_delta_rule &d, int nseq) {
    if (d.k_dim == 64 && d.v_dim == 64)
        nmoe_delta_step_as<T, 64, 64>(s, d, nseq);
    else if (d.k_dim == 64)
        nmoe_delta_step_as<T, 64, 128>(s, d, nseq);
    else if (d.v_dim == 64)
        nmoe_delta_step_as<T, 128, 64>(s, d, nseq);
    else
        nmoe_delta_step_as<T, 128, 128>(s, d, nseq);
}

/* ------------------------------------------------------- whole prompts
 *
 * In chunks of C = 64 tokens.  With G the running sum of g inside a chunk and
 * S the state before it, the chunk's tokens together are
 *   A_ij = beta_i (k_i.k_j) e^(G_i - G_j)  (j < i),    T = (I + A)^-1
 *   u    = T r,   r_i = beta_i (v_i - e^(G_i) S^T k_i)
 *   out_i = scale (e^(G_i) S^T q_i + sum_{j <= i} (q_i.k_j) e^(G_i - G_j) u_j)
 *   S   <- e^(G_C) S + sum_i e^(G_C - G_i) k_i u_i^T
 * which is matrix products.  T and P = scale (q_i.k_j) e^(G_i - G_j) need no
 * state, so a first launch computes them for all chunks at once; a second
 * goes through a sequence's chunks in order, each block with 16 columns of
 * the state (columns never meet).  Every exponent is a difference of sums in
 * 64 bits and at most 0, so none overflows and a strong decay loses nothing.
 *
 * The state is held and carried in fp32, and the products are as good: on the
 * bf16 matrix instructions (16 times the rate of the fp32 ones), an fp32
 * operand being the sum of three bf16 planes (8 + 8 + 8 bits), a bf16 input
 * one, an f16 input two; of a product's plane pairs (i, j) those with i + j <
 * 3 matter to 2^-24.  What goes to a 16-bit output only (q.S and P u) takes
 * i + j < 2 (2^-16). */

#define NMOE_DELTA_C 64
#define NMOE_DELTA_COLS 16 /* state columns of a block */

template <typename T>
struct nmoe_delta_type;
template <>
struct nmoe_delta_type<float> {
    static constexpr int planes = 3, out_planes = 3, words = 2; /* of k and q, of P and u, 16-byte words of 8 elements */
};
template <>
struct nmoe_delta_type<nmoe_bf16> {
    static constexpr int planes = 1, out_planes = 2, words = 1;
};
template <>
struct nmoe_delta_type<_Float16> {
    static constexpr int planes = 2, out_planes = 2, words = 1;
};

/* M values (M even) as N bf16 planes: the upper half of the word, then of the
 * rest's, and the last rest rounded.  Each taking-off is exact. */
template <int N, int M>
__device__ __forceinline__ void nmoe_split(const float *x, uint32_t (*planes)[M / 2]) {
    float y[M];
#pragma unroll
    for (int e = 0; e < M; e++) y[e] = x[e];
#pragma unroll
    for (int i = 0; i < N - 1; i++) {
#pragma unroll
        for (int e = 0; e < M; e += 2) {
            planes[i][e / 2] = __builtin_amdgcn_perm(__float_as_uint(y[e + 1]), __float_as_uint(y[e]), 0x07060302);
            y[e] -= __uint_as_float(__float_as_uint(y[e]) & 0xffff0000u);
            y[e + 1] -= __uint_as_float(__float_as_uint(y[e + 1]) & 0xffff0000u);
        }
    }
#pragma unroll
    for (int e = 0; e < M; e += 2) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        planes[N - 1][e / 2] = __builtin_bit_cast(uint32_t, b2{(__bf16)y[e], (__bf16)y[e + 1]});
    }
}

/* 8 elements as loaded, as planes. */
template <typename T>
__device__ __forceinline__ void nmoe_planes(const nmoe_u4 *raw, nmoe_u4 (&out)[nmoe_delta_type<T>::planes]) {
    constexpr int N = nmoe_delta_type<T>::planes;
    if constexpr (N == 1)
        out[0] = raw[0];
    else {
        float x[8];
        uint32_t y[N][4];
        nmoe_load<T, 8>((const T *)raw, x);
        nmoe_split<N, 8>(x, y);
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = nmoe_u4{y[i][0], y[i][1], y[i][2], y[i][3]};
    }
}

/* The workspace: for each chunk, the rows of k and q of each head of k, then
 * for each head of v T, P and the factors.  Matrices lie as the 16x16x32
 * operand that the second launch takes them for, a wavefront's 16 bytes a
 * lane side by side (1 KB a block): read as rows, an operand's lanes 0..15
 * are 16 rows, and the memory pipeline takes a lane a cycle instead of four
 * (6300 cycles a chunk in the second launch instead of 4300).
 *   k, q: blocks [16 tokens][32 dimensions][plane]
 *   T, P: blocks [16 tokens w][32 tokens][plane], without the upper half:
 *         (0,0), (1,0), (2,0), (2,1), (3,0), (3,1)
 *         (of 32, the one 16 a + 4 c + i is element 4 a + i of lanes 16 c ..:
 *         the order in which a result has them as its rows)
 *   factors, 64 each, one a token: beta, beta e^G n_k, scale e^G n_q,
 *         e^(G_C - G) n_k, then e^(G_C); n_k and n_q the l2 factors of key
 *         and query (as rows, so that a load of 4 tokens has no unused word:
 *         its register would be taken again while the load is under way,
 *         with a wait for it). */
template <typename T, int DK>
struct nmoe_delta_ws {
    static constexpr int pk = nmoe_delta_type<T>::planes, pp = nmoe_delta_type<T>::out_planes, ks = DK / 32;
    static constexpr size_t block = 1024, q = 4 * ks * pk * block, head_k = 2 * q;
    static constexpr size_t p = 6 * 3 * block, coef = p + 6 * pp * block, head_v = coef + 4 * NMOE_DELTA_C * 4 + 16;
    static __host__ __device__ __forceinline__ size_t chunk(int k_heads, int v_heads) {
        return (size_t)k_heads * head_k + (size_t)v_heads * head_v;
    }
    /* first block of wavefront w in T and P */
    static __device__ __forceinline__ int tri(int w) { return w < 2 ? w : 2 * w - 2; }
};

/* Chunks are numbered through the sequences: chunk n of sequence b is
 * cu[b] / 64 + b + n, so that no two share a number. */
static size_t nmoe_delta_chunks(int nseq, int ntok) { return (size_t)ntok / NMOE_DELTA_C + (size_t)nseq + 1; }

/* 2^x of a 64-bit x, good to fp32: the whole turns by exponent. */
__device__ __forceinline__ float nmoe_delta_pow2(double x) {
    const double n = rint(x);
    return ldexpf(nmoe_exp2((float)(x - n)), (int)n);
}

/* Inclusive sum over the lanes, in 64 bits: within rows of 16 by DPP
 * (row_shr, lanes without a partner add 0), then the rows before. */
template <int N>
__device__ __forceinline__ double nmoe_delta_shr(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, 0x110 | N, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), 0x110 | N, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double nmoe_delta_lane(double x, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double nmoe_delta_scan(double x, int lane) {
    x += nmoe_delta_shr<1>(x);
    x += nmoe_delta_shr<2>(x);
    x += nmoe_delta_shr<4>(x);
    x += nmoe_delta_shr<8>(x);
    const double a = nmoe_delta_lane(x, 15), b = a + nmoe_delta_lane(x, 31), c = b + nmoe_delta_lane(x, 47);
    return x + (lane < 16 ? 0.0 : lane < 32 ? a : lane < 48 ? b : c);
}

/* A lane's 8 of 32 neighbouring elements, at 4 c and 16 + 4 c, as they are
 * and as numbers (p: the first's place). */
template <typename T>
__device__ __forceinline__ void nmoe_delta_row(const T *p, nmoe_u4 (&raw)[nmoe_delta_type<T>::words], float (&x)[8]) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    if constexpr (nmoe_delta_type<T>::words == 2) {
        raw[0] = *(const nmoe_u4 *)p;
        raw[1] = *(const nmoe_u4 *)(p + 16);
    } else {
        const u2 a = *(const u2 *)p, b = *(const u2 *)(p + 16);
        raw[0] = nmoe_u4{a.x, a.y, b.x, b.y};
    }
    nmoe_load<T, 8>((const T *)raw, x);
}

/* Everything of a chunk that needs no state: one block a chunk and head of k,
 * for the v heads on it.  Wavefront w has the tokens 16 w .. as columns:
 *   k.k^T and k.q^T (rows: earlier tokens, columns: its own), of which
 *   A^T goes to LDS and P^T, a lane's rows of a column, is the second
 *   launch's operand as it is;
 *   T^T = (I + A^T)^-1 by blocks of 16: its diagonal block by substitution
 *   (lane j column j), then upwards
 *     T^T[c][w] = -T^T[c][c] sum_{m = c+1}^{w} A^T[c][m] T^T[m][w]
 *   on the fp32 matrix instructions (16x16x4), whose result is their next
 *   column operand, and in the end again the operand wanted, as it is.
 * Its time is latency (a block with two heads takes 18 us, with one 13), so as many blocks as fit
 * share a CU: four with bf16 rows, held to 128 registers; f16 and fp32 ones
 * need more for their planes and would spill.  (All keep 67 to 83 scalars in
 * vector registers' lanes.)  Where the blocks fit the device at once all the
 * same, each takes one head of v only (alone). */
template <typename T, int DK>
__global__ void __launch_bounds__(256, nmoe_elem<T>::dtype == NMOE_HIP_BF16 ? 4 : 1)
    nmoe_delta_prep_kernel(nmoe_hip_delta_rule d, const int32_t *cu, int nseq, int ntok, int alone, char *ws) {
    typedef nmoe_delta_type<T> Y;
    typedef nmoe_delta_ws<T, DK> L;
    constexpr int C = NMOE_DELTA_C, LD = C + 4, PK = Y::planes, PP = Y::out_planes, W = Y::words, KS = DK / 32;
    constexpr int LR = DK + 16 / sizeof(T), CH = DK * sizeof(T) / 16, RPI = 256 / CH; /* a row's stride, its 16-byte chunks */
    __shared__ alignas(16) char s_kx[C * LR * sizeof(T)];
    __shared__ alignas(16) char s_qa[C * LR * sizeof(T) > C * LD * 4 ? C * LR * sizeof(T) : C * LD * 4];
    __shared__ double s_g[4][C];
    __shared__ float s_nk[C], s_nq[C];
    T(*s_k)[LR] = (T(*)[LR])s_kx, (*s_q)[LR] = (T(*)[LR])s_qa;
    /* once k and q have been used: the diagonal blocks, and [j][i] = A_ij */
    float(*s_x)[16][20] = (float(*)[16][20])s_kx, (*s_at)[LD] = (float(*)[LD])s_qa;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, c = lane / 16;
    const int group = d.v_heads / d.k_heads, parts = alone ? group : 1; /* blocks a chunk and head of k */
    const int pairs = nseq * d.k_heads * parts, kh = blockIdx.x / parts % d.k_heads, b = blockIdx.x % pairs / (d.k_heads * parts);
    const int hg0 = blockIdx.x % parts;
    const int state = d.state_index != NULL ? d.state_index[b] : b;
    if (state < 0 || state >= d.num_states) return;
    const int t0 = min(max(cu[b], 0), ntok), len = min(max(cu[b + 1], t0), ntok) - t0;
    for (int64_t n64 = blockIdx.x / pairs; n64 * C < len; n64 += gridDim.x / pairs) {
        const int n = (int)n64, first = t0 + n * C, cnt = min(len - n * C, C);
        char *chunk = ws + (size_t)(t0 / C + b + n) * L::chunk(d.k_heads, d.v_heads);
        char *kq = chunk + (size_t)kh * L::head_k + (size_t)w * KS * PK * L::block + 16 * lane;
        /* g and beta of the lane's token, a head ahead */
        const int64_t gat = (int64_t)(first + min(lane, cnt - 1)) * d.v_heads + kh * group;
#pragma unroll
        for (int i = 0; i < C / RPI; i++) {
            const int row = i * RPI + tid / CH, at = tid % CH * (16 / (int)sizeof(T));
            const int64_t src = first + min(row, cnt - 1);
            *(nmoe_u4 *)&s_k[row][at] = *(const nmoe_u4 *)((const T *)d.k + src * d.k_stride + kh * DK + at);
            *(nmoe_u4 *)&s_q[row][at] = *(const nmoe_u4 *)((const T *)d.q + src * d.q_stride + kh * DK + at);
        }
        nmoe_lds_sync();
        nmoe_f4 kk[4], qk[4];
        float sk = 0.0f, sq = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++) kk[t] = qk[t] = nmoe_f4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KS; k++) {
            nmoe_u4 rk[W], rq[W], pk[PK], pq[PK];
            float xk[8], xq[8];
            nmoe_delta_row<T>(&s_k[16 * w + r][32 * k + 4 * c], rk, xk);
            nmoe_delta_row<T>(&s_q[16 * w + r][32 * k + 4 * c], rq, xq);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                sk += xk[e] * xk[e];
                sq += xq[e] * xq[e];
            }
            nmoe_planes<T>(rk, pk);
            nmoe_planes<T>(rq, pq);
            if (hg0 == 0) {
#pragma unroll
                for (int i = 0; i < PK; i++) {
                    *(nmoe_u4 *)(kq + (k * PK + i) * L::block) = pk[i];
                    *(nmoe_u4 *)(kq + L::q + (k * PK + i) * L::block) = pq[i];
                }
            }
#pragma unroll
            for (int t = 0; t < 4; t++)
                if (t <= w) {
                    nmoe_u4 rt[W];
                    float xt[8];
                    nmoe_delta_row<T>(&s_k[16 * t + r][32 * k + 4 * c], rt, xt);
                    if constexpr (W == 2) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            kk[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(xt[e], xk[e], kk[t], 0, 0, 0);
                            qk[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(xt[e], xq[e], qk[t], 0, 0, 0);
                        }
                    } else {
                        kk[t] = nmoe_mat<T>::mma16(rt[0], rk[0], kk[t]);
                        qk[t] = nmoe_mat<T>::mma16(rt[0], rq[0], qk[t]);
                    }
                }
        }
        sk += __shfl_xor(sk, 16, 64);
        sk += __shfl_xor(sk, 32, 64);
        sq += __shfl_xor(sq, 16, 64);
        sq += __shfl_xor(sq, 32, 64);
        const float nk = d.l2 ? rsqrtf(sk + d.eps) : 1.0f, nq = d.scale * (d.l2 ? rsqrtf(sq + d.eps) : 1.0f);
        if (c == 0) {
            s_nk[16 * w + r] = nk;
            s_nq[16 * w + r] = nq;
        }
        nmoe_lds_sync();
        for (int hg = hg0; hg < group; hg += parts) {
            const int h = kh * group + hg, i = 16 * w + r; /* the lane's column */
            char *head = chunk + (size_t)d.k_heads * L::head_k + (size_t)h * L::head_v;
            /* every wavefront sums for itself (in units of log2) */
            const float gn = d.g[gat + hg], bn0 = d.beta[gat + hg];
            const double G = nmoe_delta_scan(lane < cnt ? (double)nmoe_delta_g(gn) : 0.0, lane) * 1.4426950408889634074;
            const float b0 = lane < cnt ? bn0 : 0.0f, beta = __shfl(b0, i, 64);
            s_g[w][lane] = G;
            if (w == 0) {
                const float eg = lane < cnt ? nmoe_delta_pow2(G) : 0.0f;
                const double all = nmoe_delta_lane(G, 63);
                float *coef = (float *)(head + L::coef);
                coef[lane] = b0;
                coef[C + lane] = b0 * eg * s_nk[lane];
                coef[2 * C + lane] = eg * s_nq[lane];
                coef[3 * C + lane] = lane < cnt ? nmoe_delta_pow2(all - G) * s_nk[lane] : 0.0f;
                if (lane == 0) coef[4 * C] = nmoe_delta_pow2(all);
            }
            const double Gi = s_g[w][i];
            const float bn = beta * nk;
            float pv[4][4];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    pv[t][e] = 0.0f;
                    if (t <= w) {
                        const int j = 16 * t + 4 * c + e;
                        const float dec = j <= i ? nmoe_delta_pow2(Gi - s_g[w][j]) * s_nk[j] : 0.0f;
                        s_at[j][i] = j < i ? bn * kk[t][e] * dec : 0.0f;
                        pv[t][e] = nq * qk[t][e] * dec;
                    }
                }
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (k == 0 || w >= 2) {
                    uint32_t z[PP][4];
                    nmoe_split<PP, 8>(&pv[2 * k][0], z);
#pragma unroll
                    for (int x = 0; x < PP; x++)
                        *(nmoe_u4 *)(head + L::p + ((L::tri(w) + k) * PP + x) * L::block + 16 * lane) =
                            nmoe_u4{z[x][0], z[x][1], z[x][2], z[x][3]};
                }
            /* the diagonal block: column r of (I + A^T)^-1, from below */
            float x[16];
#pragma unroll
            for (int j = 15; j >= 0; j--) {
                float y = j == r ? 1.0f : 0.0f;
#pragma unroll
                for (int m = 12; m >= 0; m -= 4)
                    if (m + 3 > j) {
                        const nmoe_f4 a = *(const nmoe_f4 *)&s_at[16 * w + j][16 * w + m];
#pragma unroll
                        for (int e = 3; e >= 0; e--)
                            if (m + e > j) y -= a[e] * x[m + e];
                    }
                x[j] = y;
            }
            if (c == 0) {
#pragma unroll
                for (int j = 0; j < 16; j++) s_x[w][j][r] = x[j];
            }
            nmoe_lds_sync();
            nmoe_f4 tt[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                tt[t] = nmoe_f4{0, 0, 0, 0};
                if (t == w) {
#pragma unroll
                    for (int e = 0; e < 4; e++) tt[t][e] = s_x[t][4 * c + e][r];
                }
            }
#pragma unroll
            for (int t = 2; t >= 0; t--)
                if (t < w) {
                    nmoe_f4 y = {0, 0, 0, 0}, z = {0, 0, 0, 0};
#pragma unroll
                    for (int m = t + 1; m < 4; m++)
                        if (m <= w) {
                            const nmoe_f4 a = *(const nmoe_f4 *)&s_at[16 * t + r][16 * m + 4 * c];
#pragma unroll
                            for (int e = 0; e < 4; e++) y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], tt[m][e], y, 0, 0, 0);
                        }
                    const nmoe_f4 a = *(const nmoe_f4 *)&s_x[t][r][4 * c];
#pragma unroll
                    for (int e = 0; e < 4; e++) z = __builtin_amdgcn_mfma_f32_16x16x4f32(-a[e], y[e], z, 0, 0, 0);
                    tt[t] = z;
                }
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (k == 0 || w >= 2) {
                    float y[8];
                    uint32_t z[3][4];
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = tt[2 * k + e / 4][e % 4];
                    nmoe_split<3, 8>(y, z);
#pragma unroll
                    for (int m = 0; m < 3; m++)
                        *(nmoe_u4 *)(head + ((L::tri(w) + k) * 3 + m) * L::block + 16 * lane) =
                            nmoe_u4{z[m][0], z[m][1], z[m][2], z[m][3]};
                }
            nmoe_lds_sync(); /* A^T and the diagonal blocks are done with */
        }
    }
}

/* The products of the plane pairs (i, j), i + j < N, by their size. */
template <int NA, int NB, int N>
__device__ __forceinline__ void nmoe_delta_mma(const nmoe_u4 (&a)[NA], const nmoe_u4 (&b)[NB], nmoe_f4 (&acc)[3]) {
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
            if (i + j < N) acc[i + j] = nmoe_mat<nmoe_bf16>::mma16(a[i], b[j], acc[i + j]);
}

__device__ __forceinline__ nmoe_f4 nmoe_delta_sum(const nmoe_f4 (&acc)[3]) { return acc[0] + (acc[1] + acc[2]); }

/* 4 neighbouring rows of a result column as planes, at p + plane * step. */
template <int N>
__device__ __forceinline__ void nmoe_delta_put(nmoe_f4 x, uint16_t *p, int step) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const float y[4] = {x[0], x[1], x[2], x[3]};
    uint32_t z[N][2];
    nmoe_split<N, 4>(y, z);
#pragma unroll
    for (int i = 0; i < N; i++) *(u2 *)(p + i * step) = u2{z[i][0], z[i][1]};
}

#define NMOE_DELTA_ZERO {nmoe_f4{0, 0, 0, 0}, nmoe_f4{0, 0, 0, 0}, nmoe_f4{0, 0, 0, 0}}

/* The chunks of a sequence in order: one block a head and 16 columns of its
 * state, 8 wavefronts.  A chunk is a chain of products,
 *   k.S -> r | T r -> u | k^T (weighted u) -> S
 * and its time is that chain's latency.  So the first four wavefronts do
 * little else, and the fewest exchanges are made on it: each of them holds 32
 * rows of S, which as planes are the operand of k.S where they are; it takes
 * that product over its rows for all 64 tokens, and the parts are added up
 * in LDS.  k's columns for its rows are its own too (through LDS, for the
 * transposing reads, but with no one else).  r and the weighted u have to
 * reach all four: three barriers a chunk.  The other four wavefronts have
 * what is not on the chain: q.S, P u and out, and bringing v and the factors
 * into LDS.
 * The memory pipeline is the second limit (16 cycles for each load of a
 * wavefront, however narrow, 84 of them a chunk): loads are spread over the
 * phases, a chunk ahead.  They are never conditional (the last chunk's again
 * instead): with a path that has none, every wait would be a wait for all of
 * them.
 * The blocks of a head run on one die (blocks are dealt to 8 dies in turn)
 * and share its k, q, T and P in that die's L2.  With bf16 a block stays
 * below 128 registers and 80 KB, so where there are more than one a CU, two
 * share it and fill each other's waits.
 * 1.8 us a chunk with one block a CU: 117 us for 4096 tokens of 32 heads of
 * 128. */
template <typename T, int DK>
__global__ void __launch_bounds__(512)
    nmoe_delta_scan_kernel(nmoe_hip_delta_rule d, const int32_t *cu, int nseq, int ntok, const char *ws) {
    typedef nmoe_delta_type<T> Y;
    typedef nmoe_delta_ws<T, DK> L;
    constexpr int C = NMOE_DELTA_C, PK = Y::planes, PP = Y::out_planes, KS = DK / 32;
    constexpr int LC = C + 8, LK = 48, NC = NMOE_DELTA_COLS, VN = 16 / sizeof(T);
    __shared__ nmoe_f4 s_ks[KS][4][64];
    __shared__ nmoe_u4 s_sp[KS][PP][64]; /* S as q.S takes it */
    __shared__ alignas(16) uint16_t s_r[3][NC][LC], s_u[PP][NC][LC], s_w[3][NC][LC], s_k[KS][PK][C][LK];
    __shared__ alignas(16) T s_v[2][C][NC];
    __shared__ alignas(16) float s_c[2][4 * C + 4];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, c = lane / 16;
    const int w = wave % 4; /* its tokens are 16 w .. of the chunk, its state rows 32 w .. */
    const int slices = d.v_dim / NC, slice = blockIdx.x / 8 % slices;
    const int pair = blockIdx.x / (8 * slices) * 8 + blockIdx.x % 8;
    if (pair >= nseq * d.v_heads) return;
    const int b = pair / d.v_heads, h = pair % d.v_heads, kh = h / (d.v_heads / d.k_heads), col = slice * NC + r;
    const int state = d.state_index != NULL ? d.state_index[b] : b;
    const int t0 = min(max(cu[b], 0), ntok), len = min(max(cu[b + 1], t0), ntok) - t0;
    const int64_t ostep = (int64_t)d.v_heads * d.v_dim;
    T *out = (T *)d.out + (int64_t)t0 * ostep + h * d.v_dim + col;
    if (state < 0 || state >= d.num_states) {
        for (int t = tid / 16; t < len; t += 32) out[t * ostep] = nmoe_elem<T>::put(state < 0 ? 0.0f : NAN);
        return;
    }
    const size_t chunk_bytes = L::chunk(d.k_heads, d.v_heads);
    const char *base_k = ws + (size_t)(t0 / C + b) * chunk_bytes + (size_t)kh * L::head_k;
    const char *base_v = ws + (size_t)(t0 / C + b) * chunk_bytes + (size_t)d.k_heads * L::head_k + (size_t)h * L::head_v;
    const int chunks = (len + C - 1) / C;
    /* the upper half of T's and P's first 32 rows is not there: their first columns again, not used */
    const size_t tri = L::tri(w), second = w >= 2 ? 1 : 0;
    /* token 16 w + 4 c + e of r and u, in T's and P's order */
    const int slot = 32 * (w / 2) + 8 * c + 4 * (w % 2);

    if (wave < 4) {
        /* the state's rows of this wavefront: 16 a + 4 c + e of its 32 */
        const bool has = w < KS;
        const int64_t sat = ((int64_t)state * d.v_heads + h) * DK * d.v_dim + (int64_t)(32 * w + 4 * c) * d.v_dim + col;
        float S[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            S[e] = has && d.state_in != NULL ? d.state_in[sat + (int64_t)(16 * (e / 4) + e % 4) * d.v_dim] : 0.0f;
        nmoe_u4 xa[4][PK], xb[4][PK], xt[2][3];
        const int own = has ? w : 0; /* a wavefront without rows loads the first's */
        auto load_k = [&](int n, nmoe_u4 (&x)[4][PK]) {
            const char *p = base_k + n * chunk_bytes + (size_t)own * PK * L::block + 16 * lane;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < PK; i++) x[t][i] = *(const nmoe_u4 *)(p + (t * KS * PK + i) * L::block);
        };
        auto load_t = [&](int n) {
            const char *p = base_v + n * chunk_bytes + tri * 3 * L::block + 16 * lane;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < 3; i++) xt[k][i] = *(const nmoe_u4 *)(p + (k * second * 3 + i) * L::block);
        };
        auto work = [&](int n, const nmoe_u4 (&xk)[4][PK], nmoe_u4 (&xn)[4][PK]) {
            const int next = min(n + 1, chunks - 1);
            const float all = s_c[n % 2][4 * C];
            if (has) {
                typedef uint32_t u2 __attribute__((ext_vector_type(2)));
                uint32_t z[3][4];
                nmoe_u4 sp[3];
                nmoe_split<3, 8>(S, z);
#pragma unroll
                for (int i = 0; i < 3; i++) sp[i] = nmoe_u4{z[i][0], z[i][1], z[i][2], z[i][3]};
                /* one sum a token tile, the smallest pairs first: four chains are enough to hide each other */
                nmoe_f4 acc[4];
#pragma unroll
                for (int t = 0; t < 4; t++) acc[t] = nmoe_f4{0, 0, 0, 0};
#pragma unroll
                for (int o = 2; o >= 0; o--)
#pragma unroll
                    for (int i = 0; i < PK && i <= o; i++)
#pragma unroll
                        for (int t = 0; t < 4; t++) acc[t] = nmoe_mat<nmoe_bf16>::mma16(xk[t][i], sp[o - i], acc[t]);
#pragma unroll
                for (int t = 0; t < 4; t++) s_ks[own][t][lane] = acc[t];
                /* S for q.S, k's rows to where they are read transposed */
#pragma unroll
                for (int i = 0; i < PP; i++) s_sp[own][i][lane] = sp[i];
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < PK; i++) {
                        uint16_t *p = &s_k[own][i][16 * t + r][4 * c];
                        *(u2 *)p = u2{xk[t][i].x, xk[t][i].y};
                        *(u2 *)(p + 16) = u2{xk[t][i].z, xk[t][i].w};
                    }
            }
            const float *fc = &s_c[n % 2][16 * w + 4 * c];
            const nmoe_f4 beta = *(const nmoe_f4 *)fc, bk = *(const nmoe_f4 *)(fc + C), wk = *(const nmoe_f4 *)(fc + 3 * C);
            nmoe_f4 bv;
#pragma unroll
            for (int e = 0; e < 4; e++) bv[e] = beta[e] * nmoe_elem<T>::get(s_v[n % 2][16 * w + 4 * c + e][r]);
            nmoe_lds_sync();
            nmoe_f4 y = s_ks[0][w][lane];
#pragma unroll
            for (int i = 1; i < KS; i++) y += s_ks[i][w][lane];
            nmoe_delta_put<3>(bv - bk * y, &s_r[0][r][slot], NC * LC);
            load_k(next, xn);
            nmoe_lds_sync();
            nmoe_f4 ua[3] = NMOE_DELTA_ZERO;
            nmoe_u4 rp[2][3];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < 3; i++) rp[k][i] = *(const nmoe_u4 *)&s_r[i][r][32 * k + 8 * c];
            nmoe_delta_mma<3, 3, 3>(xt[0], rp[0], ua);
            if (w >= 2) nmoe_delta_mma<3, 3, 3>(xt[1], rp[1], ua);
            const nmoe_f4 u = nmoe_delta_sum(ua);
            nmoe_delta_put<3>(u * wk, &s_w[0][r][16 * w + 4 * c], NC * LC);
            nmoe_delta_put<PP>(u, &s_u[0][r][slot], NC * LC);
            load_t(next);
            nmoe_lds_sync();
            if (has) {
                nmoe_u4 wp[2][3];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int i = 0; i < 3; i++) wp[k][i] = *(const nmoe_u4 *)&s_w[i][r][32 * k + 8 * c];
                nmoe_u4 kt[2][2][PK];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int a = 0; a < 2; a++)
#pragma unroll
                        for (int i = 0; i < PK; i++) {
                            typedef short s4 __attribute__((ext_vector_type(4)));
                            typedef __attribute__((address_space(3))) s4 lds_s4;
                            union {
                                s4 h[2];
                                nmoe_u4 v;
                            } z;
#pragma unroll
                            for (int g = 0; g < 2; g++)
                                z.h[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (lds_s4 *)&s_k[own][i][32 * k + 8 * c + 4 * g + r / 4][16 * a + r % 4 * 4]);
                            kt[k][a][i] = z.v;
                        }
                nmoe_f4 acc[2][2];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int a = 0; a < 2; a++) acc[k][a] = nmoe_f4{0, 0, 0, 0};
#pragma unroll
                for (int o = 2; o >= 0; o--)
#pragma unroll
                    for (int i = 0; i < PK && i <= o; i++)
#pragma unroll
                        for (int k = 0; k < 2; k++)
#pragma unroll
                            for (int a = 0; a < 2; a++)
                                acc[k][a] = nmoe_mat<nmoe_bf16>::mma16(kt[k][a][i], wp[k][o - i], acc[k][a]);
#pragma unroll
                for (int a = 0; a < 2; a++)
#pragma unroll
                    for (int e = 0; e < 4; e++) S[4 * a + e] = fmaf(S[4 * a + e], all, acc[0][a][e] + acc[1][a][e]);
            }
        };
        if (chunks > 0) {
            load_k(0, xa);
            load_t(0);
        }
        nmoe_lds_sync(); /* v and the factors of the first chunk */
        for (int n = 0; n < chunks; n += 2) {
            work(n, xa, xb);
            if (n + 1 >= chunks) break;
            work(n + 1, xb, xa);
        }
        if (has) {
#pragma unroll
            for (int e = 0; e < 8; e++) d.state_out[sat + (int64_t)(16 * (e / 4) + e % 4) * d.v_dim] = S[e];
        }
    } else {
        nmoe_u4 xp[2][PP], xq[KS][PK], xv, xc;
        float all;
        const int vchunk = tid - 256, vrow = vchunk * VN / NC; /* 16 bytes of v a thread, as many as there are */
        auto load_p = [&](int n) {
            const char *p = base_v + n * chunk_bytes + L::p + tri * PP * L::block + 16 * lane;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < PP; i++) xp[k][i] = *(const nmoe_u4 *)(p + (k * second * PP + i) * L::block);
        };
        auto load_q = [&](int n) {
            const char *p = base_k + n * chunk_bytes + L::q + (size_t)w * KS * PK * L::block + 16 * lane;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < PK; i++) xq[k][i] = *(const nmoe_u4 *)(p + (k * PK + i) * L::block);
        };
        auto load_v = [&](int n) {
            xv = *(const nmoe_u4 *)((const T *)d.v + (int64_t)(t0 + n * C + min(vrow % C, len - n * C - 1)) * d.v_stride +
                                    h * d.v_dim + slice * NC + vchunk * VN % NC);
            const char *p = base_v + n * chunk_bytes + L::coef;
            xc = *(const nmoe_u4 *)(p + 16 * lane);
            all = ((const float *)p)[4 * C];
        };
        auto put_v = [&](int n) {
            if (vrow < C) *(nmoe_u4 *)&s_v[n % 2][vrow][vchunk * VN % NC] = xv;
            if (w == 0) {
                *(nmoe_u4 *)&s_c[n % 2][4 * lane] = xc;
                if (lane == 0) s_c[n % 2][4 * C] = all;
            }
        };
        if (chunks > 0) {
            load_v(0);
            put_v(0);
            load_v(min(1, chunks - 1));
            put_v(1);
            load_q(0);
            load_p(0);
            load_v(min(2, chunks - 1));
        }
        nmoe_lds_sync();
        for (int n = 0; n < chunks; n++) {
            nmoe_lds_sync();
            nmoe_u4 sp[KS][PP];
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < PP; i++) sp[k][i] = s_sp[k][i][lane];
            const nmoe_f4 z = *(const nmoe_f4 *)&s_c[n % 2][2 * C + 16 * w + 4 * c];
            nmoe_lds_sync();
            nmoe_f4 qs[3] = NMOE_DELTA_ZERO, acc[3] = NMOE_DELTA_ZERO;
#pragma unroll
            for (int k = 0; k < KS; k++) nmoe_delta_mma<PK, PP, PP>(xq[k], sp[k], qs);
            nmoe_lds_sync();
            nmoe_u4 up[2][PP];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < PP; i++) up[k][i] = *(const nmoe_u4 *)&s_u[i][r][32 * k + 8 * c];
            nmoe_delta_mma<PP, PP, PP>(xp[0], up[0], acc);
            if (w >= 2) nmoe_delta_mma<PP, PP, PP>(xp[1], up[1], acc);
            const nmoe_f4 o = z * nmoe_delta_sum(qs) + nmoe_delta_sum(acc);
            put_v(n + 2); /* where this chunk's were: the first wavefronts took them before they met these */
            load_q(min(n + 1, chunks - 1));
            load_p(min(n + 1, chunks - 1));
            load_v(min(n + 3, chunks - 1));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int t = n * C + 16 * w + 4 * c + e;
                if (t < len) out[t * ostep] = nmoe_elem<T>::put(o[e]);
            }
        }
    }
}

template <typename T, int DK>
static void nmoe_delta_prompt_as(hipStream_t s, const nmoe_hip_delta_rule &d, int nseq, const int32_t *cu, int ntok,
                                 int max_len, int num_cus, char *ws) {
    const int64_t pairs = (int64_t)nseq * d.k_heads;
    int64_t chunks = (max_len + NMOE_DELTA_C - 1) / NMOE_DELTA_C;
    if (chunks < 1) chunks = 1;
    if (chunks * pairs > NMOE_MAX_ROWS) chunks = NMOE_MAX_ROWS / pairs; /* the blocks go on to further chunks */
    /* Where the blocks of all heads of v run at once (four a CU of bf16, two of the others), one each: for 32 heads on
     * 16, a prompt of 64 takes 17 us (all of it) instead of 22, of 1024 44 instead of 48.  Counted as if all sequences
     * were max_len long: with one long among short ones the blocks may fit and a block take all heads all the same. */
    const int64_t parts = d.v_heads / d.k_heads;
    const bool alone = parts > 1 && chunks * pairs * parts <= (nmoe_elem<T>::dtype == NMOE_HIP_BF16 ? 4 : 2) * (int64_t)num_cus;
    hipLaunchKernelGGL((nmoe_delta_prep_kernel<T, DK>), dim3((uint32_t)(chunks * pairs * (alone ? parts : 1))), dim3(256), 0,
                       s, d, cu, nseq, ntok, (int)alone, ws);
    const int64_t heads = ((int64_t)nseq * d.v_heads + 7) / 8 * 8;
    hipLaunchKernelGGL((nmoe_delta_scan_kernel<T, DK>), dim3((uint32_t)(heads * (d.v_dim / NMOE_DELTA_COLS))), dim3(512),
                       0, s, d, cu, nseq, ntok, ws);
}

template <typename T>
static void nmoe_delta_prompt_launch(hipStream_t s, const nmoe_hip_delta_rule &d, int nseq, const int32_t *cu, int ntok,
                                     int max_len, int num_cus, void *ws) {
    if (d.k_dim == 64)
        nmoe_delta_prompt_as<T, 64>(s, d, nseq, cu, ntok, max_len, num_cus, (char *)ws);
    else
        nmoe_delta_prompt_as<T, 128>(s, d, nseq, cu, ntok, max_len, num_cus, (char *)ws);
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
    if (nseq < 0 || (int64_t)nseq * d->v_heads > NMOE_DELTA_HEADS || ntok < 0 || ntok > NMOE_DELTA_TOKENS)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: %d sequences of %d heads outside 0..2^19, or ntok %d outside 0..2^30",
                         nseq, d->v_heads, ntok);
    return NMOE_HIP_OK;
}

extern "C" int nmoe_delta_step(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_delta_check(ctx, d, nseq, nseq);
    if (rc != NMOE_HIP_OK || nseq == 0) return rc;
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (d->dtype == NMOE_HIP_F32)
        nmoe_delta_launch<float>(s, *d, nseq);
    else if (d->dtype == NMOE_HIP_BF16)
        nmoe_delta_launch<nmoe_bf16>(s, *d, nseq);
    else
        nmoe_delta_launch<_Float16>(s, *d, nseq);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}

template <typename T>
static size_t nmoe_delta_chunk_bytes(const nmoe_hip_delta_rule *d) {
    return d->k_dim == 64 ? nmoe_delta_ws<T, 64>::chunk(d->k_heads, d->v_heads)
                          : nmoe_delta_ws<T, 128>::chunk(d->k_heads, d->v_heads);
}

static size_t nmoe_delta_ws_bytes(const nmoe_hip_delta_rule *d, int nseq, int ntok) {
    return nmoe_delta_chunks(nseq, ntok) * (d->dtype == NMOE_HIP_F32    ? nmoe_delta_chunk_bytes<float>(d)
                                            : d->dtype == NMOE_HIP_BF16 ? nmoe_delta_chunk_bytes<nmoe_bf16>(d)
                                                                        : nmoe_delta_chunk_bytes<_Float16>(d));
}

extern "C" size_t nmoe_delta_prompt_workspace(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, int ntok) {
    if (ctx == NULL || nmoe_delta_check(ctx, d, nseq, ntok) != NMOE_HIP_OK || nseq == 0) return 0;
    return nmoe_delta_ws_bytes(d, nseq, ntok);
}

extern "C" int nmoe_delta_prompt(nmoe_hip_ctx *ctx, const nmoe_hip_delta_rule *d, int nseq, const int32_t *cu, int ntok,
                                 int max_len, void *ws, size_t ws_bytes, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    int rc = nmoe_delta_check(ctx, d, nseq, ntok);
    if (rc != NMOE_HIP_OK) return rc;
    if (cu == NULL || !nmoe_aligned(cu, 4) || max_len < 0)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: cu and max_len >= 0 are required");
    if (nseq == 0) return NMOE_HIP_OK;
    const size_t need = nmoe_delta_ws_bytes(d, nseq, ntok);
    if (ws == NULL || !nmoe_aligned(ws, 16) || ws_bytes < need)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: a workspace of %zu bytes (16-byte aligned) is required, %zu given",
                         need, ws == NULL ? (size_t)0 : ws_bytes);
    if (max_len > ntok) max_len = ntok;
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    if (d->dtype == NMOE_HIP_F32)
        nmoe_delta_prompt_launch<float>(s, *d, nseq, cu, ntok, max_len, ctx->num_cus, ws);
    else if (d->dtype == NMOE_HIP_BF16)
        nmoe_delta_prompt_launch<nmoe_bf16>(s, *d, nseq, cu, ntok, max_len, ctx->num_cus, ws);
    else
        nmoe_delta_prompt_launch<_Float16>(s, *d, nseq, cu, ntok, max_len, ctx->num_cus, ws);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
