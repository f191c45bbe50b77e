/*
 * rk_heads_shim.h -- the C ABI between the host layer of the heads' norm and rotation (rk_heads.cpp) and its kernel (rk_kernels_heads.hip).
 * Conventions as in rk_hip_shim.h.
 */
#ifndef RK_HEADS_SHIM_H
#define RK_HEADS_SHIM_H

#include "rk_mx4_shim.h" /* element types */

#ifdef __cplusplus
extern "C" {
#endif

enum { RKH_HEADS_MOST_DIM = 512 };

typedef struct rkh_heads_args {
    int rows, D, R;
    int q_heads, k_heads;
    int type, norm, neighbours;
    float eps, rotation_scale;
    const float *q_weight, *k_weight, *inv_freq;
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_row, q_head, k_row, k_head, q_out_row, q_out_head, k_out_row, k_out_head;
    const int32_t* positions;
    int64_t position_axis;
    uint32_t axis_of[RKH_HEADS_MOST_DIM / 2 / 16]; /* two bits a pair */
    int first;                                     /* (a launch's first row; the launcher's own) */
} rkh_heads_args;
int rkh_heads(void* stream, const rkh_heads_args* args);

#ifdef __cplusplus
}
#endif
#endif /* RK_HEADS_SHIM_H */
