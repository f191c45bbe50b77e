/*
 * rk_npu_heads.h -- what stands between an attention layer's QKV projection and its attention: the norm of every query and key head and
 * their rotation by position, in one pass over the rows.  MI355X only; no counterpart in the reference.
 *
 * For each row (token) t and head, with D = head_dim and R = rotary_dim:
 *     z = x / sqrt(mean(x^2) + eps) * weight            (norm != 0; otherwise z = x)
 *     pairs i = 0 .. R / 2 - 1 of z:  (a, b) = (z[i], z[i + R / 2]), or (z[2 i], z[2 i + 1]) with neighbours != 0
 *         phi = positions[axis of i][t] * inv_freq[i]
 *         a' = rotation_scale * (a cos phi - b sin phi),   b' = rotation_scale * (b cos phi + a sin phi)
 *     z[R] .. z[D - 1] as they are
 * computed in fp32 and rounded once.  The angle is made and reduced in fp64 and then rounded to fp32: off by less than 2^-23 near zero, and by less than 2^-20 for
 * positions of all 32 bits, where inv_freq is 1 or less (products beyond 2^31 lose bits of the angle as fp64 does).
 * Squares are added in fp32, without scaling; a NaN makes its head NaN where there is a norm, and otherwise the pair.
 *
 * Positions have up to four axes (time, height, width, ..), and a table says by which one a pair is turned: sections of pairs one behind
 * the other, or interleaved ones, or whatever a model was trained with.
 *
 * All pointers are device pointers but pair_axis; the call enqueues on the context's stream and returns, under the rules for *_device
 * calls in rk_npu_hip.h.  Element types are those of rk_npu_mx4.h, one for all four tensors.  Element (t, h, d) of a tensor lies at
 * t * row + h * head + d, in values: either rows hold their heads (head >= D, row >= (heads - 1) * head + D) or heads their rows
 * (row >= D, head >= (rows - 1) * row + D); strides of a single row or head do not matter.  Queries, keys and values of one buffer are such tensors.
 * An output may be its input's own buffer (the same address and strides); otherwise no output may share a byte with an input or the
 * other output (RK_NPU_ERR_PARAM).  Tensors of one pitch may lie between each other's rows; others are told apart by their ranges,
 * first byte to last.  No rows, or no heads: nothing to do.
 */
#ifndef RK_NPU_HEADS_H
#define RK_NPU_HEADS_H

#include "rk_npu_mx4.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    uint32_t struct_size;    /* sizeof(rk_npu_heads_args) */
    int rows, head_dim;      /* head_dim: 1 .. 512 */
    int q_heads, k_heads;    /* 0: there are none, and their pointers do not matter */
    int type;
    int norm;
    float eps;
    const float* q_weight;   /* [head_dim], or NULL: 1 */
    const float* k_weight;
    const void* q;
    const void* k;
    void* q_out;
    void* k_out;
    int64_t q_row, q_head, k_row, k_head, q_out_row, q_out_head, k_out_row, k_out_head;
    int rotary_dim;          /* even, 0 .. head_dim; 0: no rotation */
    int neighbours;
    int axes;                /* 1 .. 4 */
    const int32_t* positions; /* [axes][rows], an axis position_axis values from the next */
    int64_t position_axis;
    const uint8_t* pair_axis; /* HOST array [rotary_dim / 2], read during the call, or NULL: axis 0 */
    const float* inv_freq;   /* [rotary_dim / 2] */
    float rotation_scale;
} rk_npu_heads_args;
/* One axis, eps 1e-6, rotation_scale 1, norm on, rotary_dim = head_dim; everything else zero. */
void rk_npu_heads_args_init(rk_npu_heads_args* args, int rows, int head_dim);
int rk_npu_heads_norm_rotate_device(rk_npu_ctx* ctx, const rk_npu_heads_args* args);

#ifdef __cplusplus
}
#endif
#endif /* RK_NPU_HEADS_H */
