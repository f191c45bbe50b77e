/*
 * rk_npu_g4.h -- linear layers on group-scaled 4-bit (G4) weights with 16-bit activations, MI355X only.
 *
 * None of these entry points has a counterpart in the reference.  They stand beside the W4A8 layers (one scale per column, int8 activations)
 * and the MX4 layers (scales that are powers of two, 4-bit activations) for models whose weights are 4-bit integers with a scale, and
 * perhaps a zero point, per group of consecutive values of K, and whose activations stay fp16 or bf16.
 *
 *     w[n, k] = (code[n, k] - zero[n, k / group]) * scale[n, k / group],    C[m, n] = sum over k of A[m, k] w[n, k]
 *
 * No weight is rounded: products are of small integers and exact, sums have 32 bits, each group's sum is scaled in fp32, and the result is rounded
 * once.  What is multiplied:
 *   fp16 rows: code - zero, with A as it is.
 *   bf16 rows, more than 16 of them: code - zero, with the row as fp16 times a power of two.  A is as it is down to 2^-31 of its row's largest
 *     magnitude; what is smaller is off by up to 2^-39 of that magnitude.
 *   bf16 rows, up to 16: the code, and zero times the group's sum of A is taken off the group's sum in fp32, whose roundings are those of terms
 *     (code + zero) |A|, also where the weight is zero; or as more rows.
 * So fp16 rows have results that differ by the order of fp32 sums alone, however many there are, and bf16 rows ones that differ by the above, too.
 * Rows are independent of each other; a row that holds an infinity or a NaN has infinities and NaN as its results, and so may one
 * whose sums ahead of the scale are beyond fp32: up to 128 terms of up to 255 |A|, bf16 values from 2^113 on.  Scales are finite numbers.
 *
 * All pointers are device pointers unless said otherwise; the calls enqueue on the context's stream and return, under the rules
 * for *_device calls in rk_npu_hip.h (rk_npu_hip_sync() waits, stream capture records them, a workspace is BUSY only while a
 * call enqueues).  Rows lie `ld` values apart (ld >= the row's length, any alignment of the element's size).  Calls of zero
 * rows do nothing.  The output may not share a byte with the input (RK_NPU_ERR_PARAM); rows of one pitch in bytes may lie between each
 * other's, as column slices of one buffer do.  Element types are those of rk_npu_mx4.h.
 */
#ifndef RK_NPU_G4_H
#define RK_NPU_G4_H

#include "rk_npu_mx4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Weights [N, K], one row per output column:
 *   codes   [N][ceil(K / 2)] bytes, value 2 i of a row in the low half of byte i, value 2 i + 1 in the high half; 0..15
 *   scales  [N][ceil(K / group)] of scale_type (RK_NPU_MX4_F16 or RK_NPU_MX4_BF16)
 *   zeros   [N][ceil(K / group)] bytes, 0..255, or NULL: 8
 * group: a multiple of 32; the last group of a row may be shorter, and K or more is one scale per row.
 * gate_up != 0: N = 2 F rows, the gate's F and then the up projection's F, for rk_npu_g4_run_swiglu_device; others go with
 * rk_npu_g4_run_device.  The codes are laid out for the kernels once; the arrays given are not needed afterwards.
 * NULL: an argument is out of range, or memory ran out. */
typedef struct {
    int K, N;
    int group;
    int gate_up;
    int scale_type;
} rk_npu_g4_weight_config;
typedef struct rk_npu_g4_weights rk_npu_g4_weights;
/* ... from host arrays (blocking) */
rk_npu_g4_weights* rk_npu_g4_weights_create(rk_npu_iommu_domain* domain, const rk_npu_g4_weight_config* config, const uint8_t* codes,
                                            const void* scales, const uint8_t* zeros);
/* ... from device arrays (waits for the context's stream) */
rk_npu_g4_weights* rk_npu_g4_weights_create_device(rk_npu_iommu_domain* domain, const rk_npu_g4_weight_config* config, const uint8_t* codes,
                                                   const void* scales, const uint8_t* zeros);
void rk_npu_g4_weights_free(rk_npu_g4_weights* weights);
/* Either result may be NULL. */
int rk_npu_g4_weights_query(const rk_npu_g4_weights* weights, rk_npu_g4_weight_config* config, uint64_t* device_bytes);

/* Workspace: staged rows and scratch of products of up to `max_rows` rows of K values with weights of K x N (N: 2 F for gate / up
 * weights).  Results do not depend on its sizes. */
typedef struct rk_npu_g4_workspace rk_npu_g4_workspace;
rk_npu_g4_workspace* rk_npu_g4_workspace_create(rk_npu_iommu_domain* domain, int max_rows, int K, int N);
void rk_npu_g4_workspace_free(rk_npu_g4_workspace* workspace);

/* C[rows, N] = A[rows, K] times the weights.  a_type: RK_NPU_MX4_F16 or RK_NPU_MX4_BF16; c_type: any. */
int rk_npu_g4_run_device(rk_npu_g4_workspace* workspace, const rk_npu_g4_weights* weights, int rows, int a_type, const void* A, int64_t lda,
                         int c_type, void* C, int64_t ldc);
/* C[rows, F] = silu(A * gate) * (A * up), silu(x) = x / (1 + exp(-x)) in fp32: zero below -88.7, where exp leaves it. */
int rk_npu_g4_run_swiglu_device(rk_npu_g4_workspace* workspace, const rk_npu_g4_weights* gate_up, int rows, int a_type, const void* A, int64_t lda,
                                int c_type, void* C, int64_t ldc);

#ifdef __cplusplus
}
#endif
#endif /* RK_NPU_G4_H */
