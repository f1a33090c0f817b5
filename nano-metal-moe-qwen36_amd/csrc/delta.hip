/*
 * delta.hip -- the gated delta rule, one token a sequence (nmoe_delta_step)
 * and over packed prompts (nmoe_delta_prompt).
 */
#include "nmoe_context.h"

#define NMOE_DELTA_MIN_G (-100.0f)
#define NMOE_DELTA_TOKENS (1 << 30)
#define NMOE_DELTA_HEADS (1 << 20) /* sequences x heads: with 8 blocks each a launch's threads stay below 2^32 */

/* The decay's logarithm, held above -100; NaN stays NaN. */
__device__ __forceinline__ float nmoe_delta_g(float g) { return g < NMOE_DELTA_MIN_G ? NMOE_DELTA_MIN_G : g; }

/* ---------------------------------------------------- one token a sequence
 *
 * With a = S^T k and o = S^T q of the old state, both scaled by e^g,
 *   u = beta (v - a),  S <- e^g S + k u^T,  out = scale (o + (q.k) u):
 * one pass, each value of the state read and written once.  One block a
 * sequence, head and COLS columns of the state: thread (r, c) has 4
 * neighbouring columns of the rows r, r + R, ... */
template <typename T, int DK, int DV, int COLS>
__global__ void __launch_bounds__(256)
    nmoe_delta_step_kernel(nmoe_hip_delta_rule d) {
    constexpr int L = COLS / 4, R = 256 / L, N = DK / R > 0 ? DK / R : 1;
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
    for (int i = 0; i < N; i++) *(nmoe_f4 *)(d.state_out + at + (int64_t)(r + R * i) * DV) = S[i] + s_k[r + R * i] * u;
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

/* x as N bf16 planes, each the rounded rest of those before. */
template <int N>
__device__ __forceinline__ void nmoe_split(float x, __bf16 (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        p[i] = (__bf16)x;
        x -= (float)p[i];
    }
}

/* 8 elements as loaded, as planes. */
template <typename T>
__device__ __forceinline__ void nmoe_planes(const nmoe_u4 *raw, nmoe_u4 (&out)[nmoe_delta_type<T>::planes]) {
    constexpr int N = nmoe_delta_type<T>::planes;
    if constexpr (N == 1)
        out[0] = raw[0];
    else {
        const nmoe_pack<T, 8> x = *(const nmoe_pack<T, 8> *)raw;
        nmoe_b8 y[N];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            __bf16 p[N];
            nmoe_split<N>(nmoe_elem<T>::get(x.v[e]), p);
#pragma unroll
            for (int i = 0; i < N; i++) y[i][e] = p[i];
        }
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = __builtin_bit_cast(nmoe_u4, y[i]);
    }
}

/* A chunk and head in the workspace: T and P as planes [64][64], then for
 * each token (beta, beta e^G n_k, scale e^G n_q, e^(G_C - G) n_k) and, last,
 * e^(G_C); n_k and n_q are the l2 factors of its key and query. */
template <typename T>
struct nmoe_delta_ws {
    static constexpr size_t plane = NMOE_DELTA_C * NMOE_DELTA_C * 2;
    static constexpr size_t p = 3 * plane, coef = p + nmoe_delta_type<T>::out_planes * plane;
    static constexpr size_t bytes = coef + (NMOE_DELTA_C + 1) * 16;
};

/* Chunks are numbered through the sequences: chunk n of sequence b is
 * cu[b] / 64 + b + n, so that no two share a number. */
static size_t nmoe_delta_chunks(int nseq, int ntok) { return (size_t)ntok / NMOE_DELTA_C + (size_t)nseq + 1; }

/* T, P and the factors of a chunk: one block a chunk and head of k, for the
 * v heads on it.  Wavefront w has rows 16 w .. of k.k^T and q.k^T.  T by
 * blocks of 16: the diagonal ones by substitution (lane j column j), then
 * wavefront c the blocks below in its block column,
 *   T[r][c] = -T[r][r] sum_{m = c}^{r-1} A[r][m] T[m][c],
 * on the fp32 matrix instructions (16x16x4), whose result is their next
 * column operand where it is. */
template <typename T, int DK>
__global__ void __launch_bounds__(256)
    nmoe_delta_prep_kernel(nmoe_hip_delta_rule d, const int32_t *cu, int nseq, int ntok, char *ws) {
    typedef nmoe_delta_type<T> Y;
    constexpr int C = NMOE_DELTA_C, LD = C + 4, PP = Y::out_planes;
    __shared__ alignas(16) float s_a[C][LD], s_t[C][LD], s_p[C][LD];
    __shared__ double s_g[C];
    __shared__ float s_beta[C], s_nk[C], s_nq[C];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, c = lane / 16;
    const int pairs = nseq * d.k_heads, kh = blockIdx.x % pairs % d.k_heads, b = blockIdx.x % pairs / d.k_heads;
    const int state = d.state_index != NULL ? d.state_index[b] : b;
    if (state < 0 || state >= d.num_states) return;
    const int t0 = min(max(cu[b], 0), ntok), len = min(max(cu[b + 1], t0), ntok) - t0;
    const int group = d.v_heads / d.k_heads;
    for (int64_t n64 = blockIdx.x / pairs; n64 * C < len; n64 += gridDim.x / pairs) {
        const int n = (int)n64, first = t0 + n * C, cnt = min(len - n * C, C);
        const T *kb = (const T *)d.k + first * d.k_stride + kh * DK, *qb = (const T *)d.q + first * d.q_stride + kh * DK;
        nmoe_f4 kk[4], qk[4];
        float sk = 0.0f, sq = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++) kk[t] = qk[t] = nmoe_f4{0, 0, 0, 0};
        const int64_t krow = min(16 * w + r, cnt - 1) * d.k_stride, qrow = min(16 * w + r, cnt - 1) * d.q_stride;
        if constexpr (Y::words == 2) {
            for (int x = 0; x < DK; x += 16) {
                const nmoe_f4 a = *(const nmoe_f4 *)(kb + krow + x + 4 * c), q = *(const nmoe_f4 *)(qb + qrow + x + 4 * c);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    sk += a[e] * a[e];
                    sq += q[e] * q[e];
                }
#pragma unroll
                for (int t = 0; t < 4; t++)
                    if (t <= w) {
                        const nmoe_f4 y = *(const nmoe_f4 *)(kb + min(16 * t + r, cnt - 1) * d.k_stride + x + 4 * c);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            kk[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], y[e], kk[t], 0, 0, 0);
                            qk[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[e], y[e], qk[t], 0, 0, 0);
                        }
                    }
            }
        } else {
            for (int x = 0; x < DK; x += 32) {
                const nmoe_u4 a = *(const nmoe_u4 *)(kb + krow + x + 8 * c), q = *(const nmoe_u4 *)(qb + qrow + x + 8 * c);
                float ea[8], eq[8];
                nmoe_load<T, 8>((const T *)&a, ea);
                nmoe_load<T, 8>((const T *)&q, eq);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    sk += ea[e] * ea[e];
                    sq += eq[e] * eq[e];
                }
#pragma unroll
                for (int t = 0; t < 4; t++)
                    if (t <= w) {
                        const nmoe_u4 y = *(const nmoe_u4 *)(kb + min(16 * t + r, cnt - 1) * d.k_stride + x + 8 * c);
                        kk[t] = nmoe_mat<T>::mma16(a, y, kk[t]);
                        qk[t] = nmoe_mat<T>::mma16(q, y, qk[t]);
                    }
            }
        }
        sk += __shfl_xor(sk, 16, 64);
        sk += __shfl_xor(sk, 32, 64);
        sq += __shfl_xor(sq, 16, 64);
        sq += __shfl_xor(sq, 32, 64);
        __syncthreads();
        if (c == 0) {
            s_nk[16 * w + r] = d.l2 ? rsqrtf(sk + d.eps) : 1.0f;
            s_nq[16 * w + r] = d.scale * (d.l2 ? rsqrtf(sq + d.eps) : 1.0f);
        }
        for (int hg = 0; hg < group; hg++) {
            const int h = kh * group + hg;
            char *base = ws + ((size_t)(t0 / C + b + n) * d.v_heads + h) * nmoe_delta_ws<T>::bytes;
            if (w == 0) {
                const int64_t at = (int64_t)(first + min(lane, cnt - 1)) * d.v_heads + h;
                double g = lane < cnt ? (double)nmoe_delta_g(d.g[at]) : 0.0;
#pragma unroll
                for (int i = 1; i < 64; i *= 2) {
                    const double y = __shfl_up(g, i, 64);
                    if (lane >= i) g += y;
                }
                s_g[lane] = g;
                s_beta[lane] = lane < cnt ? d.beta[at] : 0.0f;
            }
            __syncthreads();
            if (w == 0) {
                const float beta = s_beta[lane], eg = lane < cnt ? expf((float)s_g[lane]) : 0.0f;
                const float left = lane < cnt ? expf((float)(s_g[63] - s_g[lane])) : 0.0f;
                nmoe_f4 *coef = (nmoe_f4 *)(base + nmoe_delta_ws<T>::coef);
                coef[lane] = nmoe_f4{beta, beta * eg * s_nk[lane], eg * s_nq[lane], left * s_nk[lane]};
                if (lane == 0) {
                    const float all = expf((float)s_g[63]);
                    coef[C] = nmoe_f4{all, all, all, all};
                }
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int j = 16 * t + r;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = 16 * w + 4 * c + e;
                    const float dec = j <= i ? expf((float)(s_g[i] - s_g[j])) * s_nk[j] : 0.0f;
                    s_a[i][j] = j < i ? s_beta[i] * s_nk[i] * kk[t][e] * dec : 0.0f;
                    s_p[i][j] = j <= i ? s_nq[i] * qk[t][e] * dec : 0.0f;
                    if (t > w) s_t[i][j] = 0.0f;
                }
            }
            __syncthreads();
            float x[16]; /* column r of the diagonal block's inverse */
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float y = i == r ? 1.0f : 0.0f;
#pragma unroll
                for (int m = 0; m < i; m++) y -= s_a[16 * w + i][16 * w + m] * x[m];
                x[i] = y;
            }
            if (c == 0) {
#pragma unroll
                for (int i = 0; i < 16; i++) s_t[16 * w + i][16 * w + r] = x[i];
            }
            __syncthreads();
            nmoe_f4 col[4];
#pragma unroll
            for (int e = 0; e < 4; e++) col[0][e] = s_t[16 * w + 4 * c + e][16 * w + r];
            for (int br = w + 1; br < 4; br++) {
                nmoe_f4 y = {0, 0, 0, 0}, z = {0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < 3; m++)
                    if (m < br - w) {
                        const nmoe_f4 a = *(const nmoe_f4 *)&s_a[16 * br + r][16 * (w + m) + 4 * c];
#pragma unroll
                        for (int e = 0; e < 4; e++) y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], col[m][e], y, 0, 0, 0);
                    }
                const nmoe_f4 a = *(const nmoe_f4 *)&s_t[16 * br + r][16 * br + 4 * c];
#pragma unroll
                for (int e = 0; e < 4; e++) z = __builtin_amdgcn_mfma_f32_16x16x4f32(-a[e], y[e], z, 0, 0, 0);
#pragma unroll
                for (int m = 1; m < 4; m++)
                    if (m == br - w) col[m] = z;
#pragma unroll
                for (int e = 0; e < 4; e++) s_t[16 * br + 4 * c + e][16 * w + r] = z[e];
            }
            __syncthreads();
            /* thread: 8 neighbouring values of a row, twice */
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int row = tid / 8 + 32 * i, at = tid % 8 * 8;
                nmoe_b8 tp[3], pp[PP];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    __bf16 y[3], z[PP];
                    nmoe_split<3>(s_t[row][at + e], y);
                    nmoe_split<PP>(s_p[row][at + e], z);
#pragma unroll
                    for (int j = 0; j < 3; j++) tp[j][e] = y[j];
#pragma unroll
                    for (int j = 0; j < PP; j++) pp[j][e] = z[j];
                }
#pragma unroll
                for (int j = 0; j < 3; j++)
                    *(nmoe_b8 *)(base + j * nmoe_delta_ws<T>::plane + (row * C + at) * 2) = tp[j];
#pragma unroll
                for (int j = 0; j < PP; j++)
                    *(nmoe_b8 *)(base + nmoe_delta_ws<T>::p + j * nmoe_delta_ws<T>::plane + (row * C + at) * 2) = pp[j];
            }
            __syncthreads();
        }
    }
}

/* What a wavefront reads of a chunk. */
template <typename T, int DK>
struct nmoe_delta_in {
    nmoe_u4 k[DK / 32 * nmoe_delta_type<T>::words], q[DK / 32 * nmoe_delta_type<T>::words];
    nmoe_u4 t[2][3], p[2][nmoe_delta_type<T>::out_planes];
    nmoe_f4 coef[4], all;
    T v[4];
};

/* The products of the plane pairs (i, j), i + j < N: the largest apart from
 * the rest. */
template <int NA, int NB, int N>
__device__ __forceinline__ void nmoe_delta_mma(const nmoe_u4 (&a)[NA], const nmoe_u4 (&b)[NB], nmoe_f4 &hi, nmoe_f4 &lo) {
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
        for (int j = 0; j < NB; j++) {
            if (i + j == 0)
                hi = nmoe_mat<nmoe_bf16>::mma16(a[i], b[j], hi);
            else if (i + j < N)
                lo = nmoe_mat<nmoe_bf16>::mma16(a[i], b[j], lo);
        }
}

/* 4 neighbouring rows of a result column as planes, at p + plane * step. */
template <int N>
__device__ __forceinline__ void nmoe_delta_put(nmoe_f4 x, uint16_t *p, int step) {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    b4 y[N];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        __bf16 z[N];
        nmoe_split<N>(x[e], z);
#pragma unroll
        for (int i = 0; i < N; i++) y[i][e] = z[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++) *(b4 *)(p + i * step) = y[i];
}

/* The chunks of a sequence in order: one block a head and 16 columns of its
 * state.  Wavefront w has the chunk's tokens 16 w .. (k.S, q.S, u, out) and
 * rows DK / 4 w .. of the state; S, r, u and the weighted u go round through
 * LDS as planes, column by column (a lane's 8 rows of a column operand side
 * by side, columns 16 bytes further than a multiple of the banks), k's rows
 * too, for the transposing reads.  The next chunk's inputs are on their way
 * while one is worked on.  The blocks of a head run on one die (blocks are
 * dealt to 8 dies in turn) and share its k, q, T and P in that die's L2. */
template <typename T, int DK>
__global__ void __launch_bounds__(256)
    nmoe_delta_scan_kernel(nmoe_hip_delta_rule d, const int32_t *cu, int nseq, int ntok, const char *ws) {
    typedef nmoe_delta_type<T> Y;
    constexpr int C = NMOE_DELTA_C, PK = Y::planes, PP = Y::out_planes, W = Y::words, KS = DK / 32, RT = DK / 64;
    constexpr int LS = DK + 8, LC = C + 8, LK = DK + 16, NC = NMOE_DELTA_COLS;
    __shared__ alignas(16) uint16_t s_s[3][NC][LS], s_r[3][NC][LC], s_u[PP][NC][LC], s_w[3][NC][LC], s_k[PK][C][LK];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64, r = lane % 16, c = lane / 16;
    const int slices = d.v_dim / NC, slice = blockIdx.x / 8 % slices;
    const int pair = blockIdx.x / (8 * slices) * 8 + blockIdx.x % 8;
    if (pair >= nseq * d.v_heads) return;
    const int b = pair / d.v_heads, h = pair % d.v_heads, kh = h / (d.v_heads / d.k_heads), col = slice * NC + r;
    const int state = d.state_index != NULL ? d.state_index[b] : b;
    const int t0 = min(max(cu[b], 0), ntok), len = min(max(cu[b + 1], t0), ntok) - t0;
    T *out = (T *)d.out + (int64_t)t0 * d.v_heads * d.v_dim + h * d.v_dim + col;
    if (state < 0 || state >= d.num_states) {
        for (int t = tid / 16; t < len; t += 16)
            out[(int64_t)t * d.v_heads * d.v_dim] = nmoe_elem<T>::put(state < 0 ? 0.0f : NAN);
        return;
    }
    /* the state's rows of this wavefront: 4 c + e of each tile of 16 */
    const int64_t sat = ((int64_t)state * d.v_heads + h) * DK * d.v_dim + (int64_t)(16 * RT * w + 4 * c) * d.v_dim + col;
    nmoe_f4 S[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
        for (int e = 0; e < 4; e++) S[t][e] = d.state_in != NULL ? d.state_in[sat + (int64_t)(16 * t + e) * d.v_dim] : 0.0f;
        nmoe_delta_put<3>(S[t], &s_s[0][r][16 * (RT * w + t) + 4 * c], NC * LS);
    }
    const char *base = ws + ((size_t)(t0 / C + b) * d.v_heads + h) * nmoe_delta_ws<T>::bytes;
    const size_t chunk_bytes = (size_t)d.v_heads * nmoe_delta_ws<T>::bytes;
    const int chunks = (len + C - 1) / C;

    auto load = [&](int n, nmoe_delta_in<T, DK> &x) {
        const char *p = base + n * chunk_bytes;
        const int first = t0 + n * C, cnt = min(len - n * C, C), row = first + min(16 * w + r, cnt - 1);
        const T *kr = (const T *)d.k + row * d.k_stride + kh * DK + 8 * c;
        const T *qr = (const T *)d.q + row * d.q_stride + kh * DK + 8 * c;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int i = 0; i < W; i++) {
                x.k[k * W + i] = ((const nmoe_u4 *)(kr + 32 * k))[i];
                x.q[k * W + i] = ((const nmoe_u4 *)(qr + 32 * k))[i];
            }
        const char *pt = p + ((16 * w + r) * C + 8 * c) * 2;
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k == 0 || w >= 2) {
#pragma unroll
                for (int i = 0; i < 3; i++) x.t[k][i] = *(const nmoe_u4 *)(pt + i * nmoe_delta_ws<T>::plane + 64 * k);
#pragma unroll
                for (int i = 0; i < PP; i++)
                    x.p[k][i] = *(const nmoe_u4 *)(pt + nmoe_delta_ws<T>::p + i * nmoe_delta_ws<T>::plane + 64 * k);
            }
        const nmoe_f4 *coef = (const nmoe_f4 *)(p + nmoe_delta_ws<T>::coef);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x.coef[e] = coef[16 * w + 4 * c + e];
            x.v[e] = ((const T *)d.v)[(int64_t)(first + min(16 * w + 4 * c + e, cnt - 1)) * d.v_stride + h * d.v_dim + col];
        }
        x.all = coef[C];
    };

    auto work = [&](int n, const nmoe_delta_in<T, DK> &x) {
        nmoe_f4 khi = {0, 0, 0, 0}, klo = khi, qhi = khi, qlo = khi;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            nmoe_u4 sp[3], kp[PK], qp[PK];
#pragma unroll
            for (int i = 0; i < 3; i++) sp[i] = *(const nmoe_u4 *)&s_s[i][r][32 * k + 8 * c];
            nmoe_planes<T>(&x.k[k * W], kp);
            nmoe_planes<T>(&x.q[k * W], qp);
            nmoe_delta_mma<PK, 3, 3>(kp, sp, khi, klo);
            nmoe_delta_mma<PK, 3, PP>(qp, sp, qhi, qlo);
#pragma unroll
            for (int i = 0; i < PK; i++) *(nmoe_u4 *)&s_k[i][16 * w + r][32 * k + 8 * c] = kp[i];
        }
        nmoe_f4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = x.coef[e].x * nmoe_elem<T>::get(x.v[e]) - x.coef[e].y * (khi[e] + klo[e]);
        nmoe_delta_put<3>(y, &s_r[0][r][16 * w + 4 * c], NC * LC);
        __syncthreads();
        nmoe_f4 uhi = {0, 0, 0, 0}, ulo = uhi;
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k == 0 || w >= 2) {
                nmoe_u4 rp[3];
#pragma unroll
                for (int i = 0; i < 3; i++) rp[i] = *(const nmoe_u4 *)&s_r[i][r][32 * k + 8 * c];
                nmoe_delta_mma<3, 3, 3>(x.t[k], rp, uhi, ulo);
            }
        nmoe_f4 u;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            u[e] = uhi[e] + ulo[e];
            y[e] = u[e] * x.coef[e].w;
        }
        nmoe_delta_put<PP>(u, &s_u[0][r][16 * w + 4 * c], NC * LC);
        nmoe_delta_put<3>(y, &s_w[0][r][16 * w + 4 * c], NC * LC);
        __syncthreads();
        /* the state first: the next chunk waits for it */
        nmoe_u4 wp[2][3];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int i = 0; i < 3; i++) wp[k][i] = *(const nmoe_u4 *)&s_w[i][r][32 * k + 8 * c];
#pragma unroll
        for (int t = 0; t < RT; t++) {
            nmoe_f4 hi = {0, 0, 0, 0}, lo = hi;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                typedef short s4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s4 lds_s4;
                nmoe_u4 kt[PK];
#pragma unroll
                for (int i = 0; i < PK; i++) {
                    union {
                        s4 h[2];
                        nmoe_u4 v;
                    } z;
#pragma unroll
                    for (int g = 0; g < 2; g++)
                        z.h[g] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s4 *)&s_k[i][32 * k + 8 * c + 4 * g + r / 4][16 * (RT * w + t) + r % 4 * 4]);
                    kt[i] = z.v;
                }
                nmoe_delta_mma<PK, 3, 3>(kt, wp[k], hi, lo);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) S[t][e] = fmaf(S[t][e], x.all.x, hi[e] + lo[e]);
            nmoe_delta_put<3>(S[t], &s_s[0][r][16 * (RT * w + t) + 4 * c], NC * LS);
        }
        nmoe_f4 hi = {0, 0, 0, 0}, lo = hi;
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (k == 0 || w >= 2) {
                nmoe_u4 up[PP];
#pragma unroll
                for (int i = 0; i < PP; i++) up[i] = *(const nmoe_u4 *)&s_u[i][r][32 * k + 8 * c];
                nmoe_delta_mma<PP, PP, PP>(x.p[k], up, hi, lo);
            }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int t = n * C + 16 * w + 4 * c + e;
            if (t < len)
                out[(int64_t)t * d.v_heads * d.v_dim] =
                    nmoe_elem<T>::put(x.coef[e].z * (qhi[e] + qlo[e]) + (hi[e] + lo[e]));
        }
        __syncthreads();
    };

    nmoe_delta_in<T, DK> x0, x1;
    if (chunks > 0) load(0, x0);
    __syncthreads();
    for (int n = 0; n < chunks; n += 2) {
        if (n + 1 < chunks) load(n + 1, x1);
        work(n, x0);
        if (n + 1 >= chunks) break;
        if (n + 2 < chunks) load(n + 2, x0);
        work(n + 1, x1);
    }
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) d.state_out[sat + (int64_t)(16 * t + e) * d.v_dim] = S[t][e];
}

template <typename T, int DK>
static void nmoe_delta_prompt_as(hipStream_t s, const nmoe_hip_delta_rule &d, int nseq, const int32_t *cu, int ntok,
                                 int max_len, char *ws) {
    const int64_t pairs = (int64_t)nseq * d.k_heads;
    int64_t chunks = (max_len + NMOE_DELTA_C - 1) / NMOE_DELTA_C;
    if (chunks < 1) chunks = 1;
    if (chunks * pairs > NMOE_MAX_ROWS) chunks = NMOE_MAX_ROWS / pairs; /* the blocks go on to further chunks */
    hipLaunchKernelGGL((nmoe_delta_prep_kernel<T, DK>), dim3((uint32_t)(chunks * pairs)), dim3(256), 0, s, d, cu, nseq,
                       ntok, ws);
    const int64_t heads = ((int64_t)nseq * d.v_heads + 7) / 8 * 8;
    hipLaunchKernelGGL((nmoe_delta_scan_kernel<T, DK>), dim3((uint32_t)(heads * (d.v_dim / NMOE_DELTA_COLS))), dim3(256),
                       0, s, d, cu, nseq, ntok, ws);
}

template <typename T>
static void nmoe_delta_prompt_launch(hipStream_t s, const nmoe_hip_delta_rule &d, int nseq, const int32_t *cu, int ntok,
                                     int max_len, void *ws) {
    if (d.k_dim == 64)
        nmoe_delta_prompt_as<T, 64>(s, d, nseq, cu, ntok, max_len, (char *)ws);
    else
        nmoe_delta_prompt_as<T, 128>(s, d, nseq, cu, ntok, max_len, (char *)ws);
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
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "delta: %d sequences of %d heads outside 0..2^20, or ntok %d outside 0..2^30",
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

static size_t nmoe_delta_ws_bytes(const nmoe_hip_delta_rule *d, int nseq, int ntok) {
    return nmoe_delta_chunks(nseq, ntok) * (size_t)d->v_heads *
           (d->dtype == NMOE_HIP_F32 ? nmoe_delta_ws<float>::bytes : nmoe_delta_ws<nmoe_bf16>::bytes);
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
        nmoe_delta_prompt_launch<float>(s, *d, nseq, cu, ntok, max_len, ws);
    else if (d->dtype == NMOE_HIP_BF16)
        nmoe_delta_prompt_launch<nmoe_bf16>(s, *d, nseq, cu, ntok, max_len, ws);
    else
        nmoe_delta_prompt_launch<_Float16>(s, *d, nseq, cu, ntok, max_len, ws);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
