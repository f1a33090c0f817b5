/*
 * nmoe_context.h -- what the context operators (kv.hip, attn_decode.hip,
 * attn_prompt.hip, delta.hip; plan.hip, kv8.hip, attn8_decode.hip,
 * attn8_prompt.hip) share: element types, row loads, the device guard and the
 * checks of their descriptors.
 */
#ifndef NMOE_CONTEXT_H
#define NMOE_CONTEXT_H

#include <math.h>

#include "nmoe_device.h"

#define NMOE_MAX_HEADS 1024
#define NMOE_MAX_ROWS (1 << 22) /* sequences x heads of a call: a launch's threads stay below 2^32 */

/* Makes the context's device current for a call's launches, and the caller's
 * again afterwards. */
struct nmoe_on_device {
    int back;
    explicit nmoe_on_device(const nmoe_hip_ctx *ctx) : back(-1) {
        int now = -1;
        if (hipGetDevice(&now) == hipSuccess && now != ctx->device && hipSetDevice(ctx->device) == hipSuccess)
            back = now;
    }
    ~nmoe_on_device() {
        if (back >= 0) (void)hipSetDevice(back);
    }
};

static inline size_t nmoe_elem_size(int dtype) { return dtype == NMOE_HIP_F32 ? 4 : 2; }

static inline int nmoe_is_half(int dtype) { return dtype == NMOE_HIP_BF16 || dtype == NMOE_HIP_F16; }

/* A stride in elements: not negative, whole 16-byte pieces, and below 2^limit:
 * 2^30 rows 2^30 elements apart, or 2^27 pages 2^34, are 2^62 bytes or less. */
#define NMOE_ROW_STRIDE 30
#define NMOE_PAGE_STRIDE 34
static inline int nmoe_stride_ok(int64_t stride, int dtype, int limit) {
    return stride >= 0 && stride < ((int64_t)1 << limit) && stride % (int64_t)(16 / nmoe_elem_size(dtype)) == 0;
}

static inline int nmoe_rows_ok(const void *p, int64_t token_stride, int64_t head_stride, int dtype) {
    return p != NULL && nmoe_aligned(p, 16) && nmoe_stride_ok(token_stride, dtype, NMOE_ROW_STRIDE) &&
           nmoe_stride_ok(head_stride, dtype, NMOE_ROW_STRIDE);
}

/* Attention takes its scores in powers of two: scale * log2(e) is finite too. */
static inline int nmoe_scale_ok(float scale) { return fabsf(scale) < 0x1p127f; }

/* kv.hip: the checks of a cache and of q/k/v rows (with_q: rows->q too) that
 * every call on them makes. */
int nmoe_check_cache(nmoe_hip_ctx *ctx, const nmoe_hip_kv_cache *c);
int nmoe_check_rows(nmoe_hip_ctx *ctx, const nmoe_hip_qkv *r, int with_q);

/* kv.hip: the checks of the norm and rotation (prep may be NULL: neither). */
int nmoe_check_prep(nmoe_hip_ctx *ctx, const nmoe_hip_qk_prep *prep, int head_dim, nmoe_hip_qk_prep *out);

/* kv8.hip: the checks of a cache in 8 bits that every call on it makes. */
int nmoe_check_cache8(nmoe_hip_ctx *ctx, const nmoe_hip_kv8_cache *c);

/* ---------------------------------------------------------------- device */

struct nmoe_bf16 {
    uint16_t bits;
};

template <typename T>
struct nmoe_elem;

template <>
struct nmoe_elem<float> {
    static constexpr int dtype = NMOE_HIP_F32;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};

template <>
struct nmoe_elem<nmoe_bf16> {
    static constexpr int dtype = NMOE_HIP_BF16;
    static __device__ __forceinline__ float get(nmoe_bf16 v) { return nmoe_bf16f(v.bits); }
    /* to nearest, ties to even; NaN stays NaN (the compiler's conversion) */
    static __device__ __forceinline__ nmoe_bf16 put(float v) {
        return nmoe_bf16{__builtin_bit_cast(uint16_t, (__bf16)v)};
    }
};

template <>
struct nmoe_elem<_Float16> {
    static constexpr int dtype = NMOE_HIP_F16;
    static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};

/* N neighbouring elements (N * sizeof(T) a multiple of 16 bytes, or 8), in
 * 16-byte loads. */
template <typename T, int N>
struct alignas(sizeof(T) * N >= 16 ? 16 : sizeof(T) * N) nmoe_pack {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void nmoe_load(const T *p, float (&out)[N]) {
    const nmoe_pack<T, N> r = *(const nmoe_pack<T, N> *)p;
#pragma unroll
    for (int i = 0; i < N; i++) out[i] = nmoe_elem<T>::get(r.v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void nmoe_store(T *p, const float (&in)[N]) {
    nmoe_pack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; i++) r.v[i] = nmoe_elem<T>::put(in[i]);
    *(nmoe_pack<T, N> *)p = r;
}

/* ------------------------------------------------------ matrix operands */

typedef float nmoe_f4 __attribute__((ext_vector_type(4)));
typedef float nmoe_f16v __attribute__((ext_vector_type(16)));
typedef __bf16 nmoe_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 nmoe_h8 __attribute__((ext_vector_type(8)));
typedef uint32_t nmoe_u4 __attribute__((ext_vector_type(4)));

/* 8 neighbouring 16-bit elements as a matrix operand.  16x16x32: the lane's
 * row (or column) is l % 16, its elements 8 (l / 16) ..; the result's column
 * is l % 16, its rows 4 (l / 16) ...  32x32x16: l % 32, 8 (l / 32) ..; the
 * result's column l % 32, row 8 (i / 4) + 4 (l / 32) + i % 4 in element i. */
template <typename T>
struct nmoe_mat;

template <>
struct nmoe_mat<nmoe_bf16> {
    static __device__ __forceinline__ nmoe_f4 mma16(nmoe_u4 a, nmoe_u4 b, nmoe_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(nmoe_b8, a), __builtin_bit_cast(nmoe_b8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ nmoe_f16v mma32(nmoe_u4 a, nmoe_u4 b, nmoe_f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(nmoe_b8, a), __builtin_bit_cast(nmoe_b8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ nmoe_u4 pack(const float *p) {
        nmoe_b8 r;
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = (__bf16)p[i];
        return __builtin_bit_cast(nmoe_u4, r);
    }
};

template <>
struct nmoe_mat<_Float16> {
    static __device__ __forceinline__ nmoe_f4 mma16(nmoe_u4 a, nmoe_u4 b, nmoe_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(nmoe_h8, a), __builtin_bit_cast(nmoe_h8, b), c,
                                                      0, 0, 0);
    }
    static __device__ __forceinline__ nmoe_f16v mma32(nmoe_u4 a, nmoe_u4 b, nmoe_f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(nmoe_h8, a), __builtin_bit_cast(nmoe_h8, b), c,
                                                      0, 0, 0);
    }
    static __device__ __forceinline__ nmoe_u4 pack(const float *p) {
        nmoe_h8 r;
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = (_Float16)p[i];
        return __builtin_bit_cast(nmoe_u4, r);
    }
};

/* Two terms of 8 bits each that make up v to 2^-17 of it. */
__device__ __forceinline__ void nmoe_two_terms(float v, float &hi, float &lo) {
    hi = (float)(__bf16)v;
    lo = v - hi;
}

#define NMOE_LONGEST (1 << 30) /* keys of a sequence: leaves room in 32 bits for a step past the end */

/* A length that the table's row can hold, else -1. */
__device__ __forceinline__ int nmoe_len_of(int len, int max_pages, int page_size) {
    len = max(len, 0);
    return (int64_t)len > (int64_t)max_pages * page_size || len > NMOE_LONGEST ? -1 : len;
}

/* Workgroup barrier over LDS only: waits for this wavefront's LDS accesses
 * (lgkmcnt 0), not for its loads and stores of device memory in flight,
 * which __syncthreads() does. */
__device__ __forceinline__ void nmoe_lds_sync() {
    __builtin_amdgcn_s_waitcnt(0xC07F); /* vmcnt 63, expcnt 7, lgkmcnt 0 */
    asm volatile("s_barrier" ::: "memory");
}

/* cos and sin of position * inv_freq, reduced to a turn in 64 bits: a
 * position of 2^31 times a frequency of 24 bits has 55, so the product is
 * off by at most 2^-22 turns there and exact below 2^29. */
__device__ __forceinline__ void nmoe_turn(int position, float inv_freq, float &c, float &s) {
    const double turns = (double)position * (double)inv_freq * 0.15915494309189533577;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
}

/* 2^x by the unit alone: results below 2^-126 are 0. */
__device__ __forceinline__ float nmoe_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

#endif
