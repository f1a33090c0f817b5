/*
 * nmoe_kv8.h -- what the operators on a cache in 8 bits (kv8.hip,
 * attn8_decode.hip, attn8_prompt.hip) share: codes and their scales.
 */
#ifndef NMOE_KV8_H
#define NMOE_KV8_H

#include "nmoe_context.h"

#define NMOE_KV8_LOW (-117) /* a scale's least power of two: a value's last bit, 2^-9 of it, is still a normal bf16 */
#define NMOE_KV8_HIGH 118   /* and its greatest: 448 of it are below 2^127 */
#define NMOE_KV8_STRIDE (1 << 24) /* 16 tokens' offsets stay below 2^31 bytes */

/* Where a token's block has its scale. */
__device__ __forceinline__ int64_t nmoe_kv8_scale_at(const nmoe_hip_kv8_cache &c, int page, int token, int head) {
    return ((int64_t)page * (c.page_size / NMOE_HIP_KV8_BLOCK) + token / NMOE_HIP_KV8_BLOCK) * c.kv_heads + head;
}

/* The power of two of a block whose largest magnitude is amax: the least e
 * with amax <= 448 * 2^e = 1.75 * 2^(e + 8). */
__device__ __forceinline__ int nmoe_kv8_power(float amax) {
    const uint32_t b = __float_as_uint(amax);
    return min(max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u), NMOE_KV8_LOW), NMOE_KV8_HIGH);
}

/* A scale's power beyond `top`, or 0. */
__device__ __forceinline__ float nmoe_kv8_beyond(float scale, int top) {
    return (float)max((int)(__float_as_uint(scale) >> 23) - (127 + top), 0);
}

__device__ __forceinline__ float nmoe_kv8_two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

/* Four codes for x[0..3] * inv, of a magnitude of at most 448, or NaN. */
__device__ __forceinline__ uint32_t nmoe_kv8_codes(const float *x, float inv) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, r, true);
    return (uint32_t)r;
}

/* Of any magnitude: beyond the largest, that; infinities and NaN: NaN. */
__device__ __forceinline__ uint32_t nmoe_kv8_codes_of_any(const float *x, float inv) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = fabsf(x[i]) < INFINITY ? fminf(fmaxf(x[i] * inv, -448.0f), 448.0f) : NAN;
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
    return (uint32_t)r;
}

/* Four codes rounded again for a scale 1 / f times as large. */
__device__ __forceinline__ uint32_t nmoe_kv8_again(uint32_t c, float f) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(b[0] * f, b[1] * f, r, true);
    return (uint32_t)r;
}

#endif
