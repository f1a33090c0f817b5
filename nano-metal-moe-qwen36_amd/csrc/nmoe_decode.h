/*
 * nmoe_decode.h -- what decode attention has alike over a cache in 16 bits
 * (attn_decode.hip) and in 8 (attn8_decode.hip): its workgroups' shape.
 */
#ifndef NMOE_DECODE_H
#define NMOE_DECODE_H

#include "nmoe_context.h"

#define NMOE_DEC_WAVES 4
#define NMOE_DEC_TILE 32                              /* keys of a wavefront's step */
#define NMOE_DEC_STEP (NMOE_DEC_WAVES * NMOE_DEC_TILE) /* keys of a block's step; parts are multiples of it */
#define NMOE_DEC_HEADS 16                             /* query heads of a block */
#define NMOE_DEC_JOIN 256

template <int N>
__device__ __forceinline__ void nmoe_dec_wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

#endif
