/* exl3b200_dense.h -- the argument records the C host side (exl3b200_dense.c) hands the kernels of the dense and MXFP4
 * expert operators. Plain C, passed by value as kernel parameters. */
#ifndef EXL3B200_DENSE_H
#define EXL3B200_DENSE_H

#include <stdint.h>

#include "exl3b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* n / d for n < 2^31 as (umulhi(n, mul) + n) >> shift, with 2^shift the least power of two from d on and
 * mul = floor(2^32 (2^shift - d) / d) + 1 (Granlund and Montgomery, "Division by Invariant Integers using
 * Multiplication", 1994). */
typedef struct Exl3bDiv {
    uint32_t d, mul, shift;
} Exl3bDiv;
static inline Exl3bDiv exl3b_div(uint32_t d) {
    Exl3bDiv v = { d, 0, 0 };
    while (((uint64_t)1 << v.shift) < d) ++v.shift;
    v.mul = (uint32_t)(((((uint64_t)1 << v.shift) - d) << 32) / d + 1);
    return v;
}
#ifdef __CUDACC__
static __device__ __forceinline__ uint32_t exl3b_div_of(uint32_t n, const Exl3bDiv& v) {
    return (__umulhi(n, v.mul) + n) >> v.shift;
}
#endif

/* block_norm (exl3b200_norm.cu); pitches in elements, q_pitch and qs_pitch in bytes. */
typedef struct Exl3bNormOp {
    int64_t     rows, cols;
    const void* branch;
    int64_t     branch_pitch;
    const void* post_w;
    const void* gate;
    int64_t     gate_pitch;
    const void* res;
    int64_t     res_pitch;
    void*       out;
    int64_t     out_pitch;
    const void* pre_w;
    void*       y;
    int64_t     y_pitch;
    uint8_t*    q;
    int64_t     q_pitch;
    uint8_t*    q_scales;
    int64_t     qs_pitch;
    int32_t     gate_kind;
    float       post_eps, pre_eps, res_scale;
} Exl3bNormOp;

/* grouped_mm (exl3b200_gmm.cu). */
typedef struct Exl3bGmmOp {
    int64_t        n_rows, n_out, n_in;
    int64_t        w_rows;               /* the weight's rows: n_out, or twice that with silu_mul */
    int64_t        x_rows;
    int32_t        n_expert, top_k;      /* top_k 0: sorted row i reads x row i */
    Exl3bDiv       slots;                /* of a token: top_k (0: 1) */
    int32_t        act, y_dtype;
    const void*    x;                    /* elements, or MXFP4 codes */
    int64_t        x_pitch_bytes;
    const void*    w;
    int64_t        w_pitch_bytes, w_expert_bytes;
    const int32_t* sorted_tok;           /* NULL: every row live */
    const int32_t* expert_offset;        /* NULL: one group of all rows */
    void*          y;
    int64_t        y_pitch;              /* elements; bytes for MXFP4 */
    uint8_t*       y_scales;
    int64_t        ys_pitch;
    const uint8_t* x_scales;
    int64_t        xs_pitch;
    const uint8_t* w_scales;             /* the tiled form */
    int64_t        ws_expert_bytes, ws_blk_bytes;
    int32_t        mx4, bf16;
    int32_t*       err;                  /* device word: set nonzero when a bounded wait gives up */
} Exl3bGmmOp;

#ifdef __cplusplus
}
#endif

#endif /* EXL3B200_DENSE_H */
