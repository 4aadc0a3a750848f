/*
 * akv_rotary.h — C ABI of the rotary positions: rotating the heads of tokens
 * with one or several position axes (text; images: height and width; video:
 * time, height and width), and the table that an append to the 4-bit cache
 * rotates keys and queries with (akv_q4.h).
 *
 * Conventions of akv_cuda.h: caller-owned buffers, int status, stream order,
 * no allocation, no synchronisation. No call needs akv_cuda_init.
 * The reference project has no counterpart to these calls.
 */
#ifndef AKV_ROTARY_H
#define AKV_ROTARY_H

#include "akv_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define AKV_ROTARY_MAX_AXES 8

/*
 * Positions. table[p][i] = cos and sin of pair i at position p, fp32: made once
 * (in 64 bits, so that far positions have exact angles), with any frequencies
 * and any scaling. Pair i of a token takes the row of its position on axis
 * axis[i]. The pairs are channels (i, i + rotary_dim / 2), or (2i, 2i + 1)
 * when interleaved; channels from rotary_dim on stay as they are.
 */
typedef struct AkvRotary {
    const float* table_dev;         /* [positions][rotary_dim / 2][2], 16-byte aligned */
    int32_t positions, rotary_dim;  /* rotary_dim even, at most 256 */
    int32_t axes, interleaved;      /* axes 1 to AKV_ROTARY_MAX_AXES */
    uint8_t axis[128];              /* of each pair, below axes */
} AkvRotary;

/*
 * Rotate: y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin in fp32 (each product and
 * each sum rounded), rounded once to `dtype`; `inverse` takes -sin, which gives
 * the gradient of x from that of y. x and out are [batch][tokens][heads]
 * [head_dim] with element strides batch / token / head; out may be x, with x's
 * strides, and must not overlap it otherwise. A token with a position outside
 * [0, positions) on an axis that a pair uses has NaN in all rotated channels
 * and reports AKV_ERR_INVALID_ARGUMENT in status_dev.
 */
typedef struct AkvRotateDesc {
    AkvRotary rotary;
    int32_t batch, tokens, heads, head_dim; /* head_dim at most 256 */
    int32_t dtype;                  /* AKV_Q_*, of x and out */
    int32_t inverse;
    const void* x_dev;
    void* out_dev;
    int64_t x_stride[3], out_stride[3];
    const int32_t* positions_dev;   /* [axes][batch][tokens] */
    int32_t* status_dev;            /* optional */
} AkvRotateDesc;

int akv_rotate(const AkvRotateDesc* desc, void* stream);

/* Host-only: sizeof of AkvRotary (0), AkvRotateDesc (1); 0 otherwise. */
size_t akv_rotary_struct_size(int which);

#ifdef __cplusplus
}
#endif

#endif /* AKV_ROTARY_H */
