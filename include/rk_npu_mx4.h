/*
 * rk_npu_mx4.h -- microscaled 4-bit (MX4) linear layers and the norms around them, MI355X only.
 *
 * None of these entry points has a counterpart in the reference.  They stand beside the W8A8 and W4A8 layers for models
 * whose weights are held as MX4: weights AND activations are e2m1 codes in blocks of 32 along K that share a power of two,
 * which the matrix cores multiply as stored, with fp32 sums.
 *
 * All pointers are device pointers unless said otherwise; the calls enqueue on the context's stream and return, under the rules
 * for *_device calls in rk_npu_hip.h (rk_npu_hip_sync() waits, stream capture records them, a workspace is BUSY only while a
 * call enqueues).  Rows lie `ld` values apart (ld >= the row's length, any alignment of the element's size).  Calls of zero
 * rows do nothing.  An output may not share a byte with an input or another output (RK_NPU_ERR_PARAM), except where it is said
 * below.  Rows of one pitch in bytes may lie between each other's, as column slices of one buffer do; rows of different pitches
 * are told apart by their ranges alone, first byte to last.
 *
 * MX4 rows
 *   code    bits 3 sign, 2..0 one of 0, 0.5, 1, 1.5, 2, 3, 4, 6
 *   block   32 consecutive values of a row: 16 bytes, value 2 i in the low half of byte i, value 2 i + 1 in the high half;
 *           the last block of a row is filled up with zeros
 *   scale   one byte e per block: the codes count 2^(e - 127); 255: the block is NaN
 *   A matrix of `rows` x K is codes[rows][ceil(K / 32)][16] and scales[rows][ceil(K / 32)], without gaps.
 * Quantization: e - 127 = floor(log2(largest |value| of the block)) - 2, not below -127 (which blocks of zeros take, too);
 * codes are the nearest ones to value / 2^(e - 127), ties to the even code, values beyond 6 become 6.  A block that holds an
 * infinity or a NaN becomes NaN as a whole (e = 255, codes 0).  Nothing is rejected: products with a NaN block are NaN in
 * that row (activations) or column (weights).
 */
#ifndef RK_NPU_MX4_H
#define RK_NPU_MX4_H

#include "rk_npu_common.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations and results. */
#define RK_NPU_MX4_F32  0
#define RK_NPU_MX4_F16  1
#define RK_NPU_MX4_BF16 2

/* Values [rows, K] to MX4 rows, and MX4 rows to values (rounded once, to nearest). */
int rk_npu_mx4_quantize_device(rk_npu_ctx* ctx, int type, int64_t rows, int K, const void* x, int64_t ldx, uint8_t* codes,
                               uint8_t* scales);
int rk_npu_mx4_dequantize_device(rk_npu_ctx* ctx, int type, int64_t rows, int K, const uint8_t* codes, const uint8_t* scales,
                                 void* y, int64_t ldy);

/* Weights: MX4 rows of a matrix [N, K], one row per output column.  gate_up != 0: N = 2 F rows, the gate's F and then the up
 * projection's F, for rk_npu_mx4_run_swiglu_device and the FFN calls; others go with rk_npu_mx4_run(_staged)_device.  The codes are laid
 * out for the kernels once; the arrays given are not needed afterwards.  NULL: an argument is out of range, or memory ran out. */
typedef struct {
    int K, N;
    int gate_up;
} rk_npu_mx4_weight_config;
typedef struct rk_npu_mx4_weights rk_npu_mx4_weights;
/* ... from host arrays (blocking) */
rk_npu_mx4_weights* rk_npu_mx4_weights_create(rk_npu_iommu_domain* domain, const rk_npu_mx4_weight_config* config,
                                              const uint8_t* codes, const uint8_t* scales);
/* ... from device arrays, such as rk_npu_mx4_quantize_device writes (waits for the context's stream) */
rk_npu_mx4_weights* rk_npu_mx4_weights_create_device(rk_npu_iommu_domain* domain, const rk_npu_mx4_weight_config* config,
                                                     const uint8_t* codes, const uint8_t* scales);
void rk_npu_mx4_weights_free(rk_npu_mx4_weights* weights);
/* Either result may be NULL. */
int rk_npu_mx4_weights_query(const rk_npu_mx4_weights* weights, rk_npu_mx4_weight_config* config, uint64_t* device_bytes);

/* Workspace: the MX4 rows that products read and their scratch, for up to `max_rows` rows of K values and weights of K x N (N: 2 F
 * for gate / up weights). */
typedef struct rk_npu_mx4_workspace rk_npu_mx4_workspace;
rk_npu_mx4_workspace* rk_npu_mx4_workspace_create(rk_npu_iommu_domain* domain, int max_rows, int K, int N);
void rk_npu_mx4_workspace_free(rk_npu_mx4_workspace* workspace);

/* C[rows, N] = A[rows, K] as MX4 times the weights. */
int rk_npu_mx4_run_device(rk_npu_mx4_workspace* workspace, const rk_npu_mx4_weights* weights, int rows, int a_type, const void* A,
                          int64_t lda, int c_type, void* C, int64_t ldc);
/* The same in two calls, for rows that several weights of one shape multiply (or of a smaller N; gate / up weights give what
 * run_swiglu gives): stage quantizes A into the workspace, where the rows stay until the next call but run_staged that uses the
 * workspace.  run_staged multiplies as many rows as the last call staged; where that is none, because nothing was staged or a call
 * of zero rows was the last, it returns RK_NPU_ERR_PARAM and writes nothing: a program whose batches may be empty leaves it out for
 * those.  A captured stage counts as a call when it is captured, and its replays put their own rows into the workspace: the
 * products of those rows belong into the same graph. */
int rk_npu_mx4_stage_device(rk_npu_mx4_workspace* workspace, int rows, int a_type, const void* A, int64_t lda);
int rk_npu_mx4_run_staged_device(rk_npu_mx4_workspace* workspace, const rk_npu_mx4_weights* weights, int c_type, void* C, int64_t ldc);
/* C[rows, F] = silu(A * gate) * (A * up), silu(x) = x / (1 + exp(-x)) in fp32: zero below -88.7, where exp leaves it. */
int rk_npu_mx4_run_swiglu_device(rk_npu_mx4_workspace* workspace, const rk_npu_mx4_weights* gate_up, int rows, int a_type,
                                 const void* A, int64_t lda, int c_type, void* C, int64_t ldc);
/* Gate / up product, SwiGLU and down product; the middle goes from the fp32 sums to MX4 rows in down_workspace and is not written
 * as values.  Both workspaces take `rows` rows; down's K is F. */
int rk_npu_mx4_run_ffn_device(rk_npu_mx4_workspace* workspace, const rk_npu_mx4_weights* gate_up, rk_npu_mx4_workspace* down_workspace,
                              const rk_npu_mx4_weights* down, int rows, int a_type, const void* A, int64_t lda, int c_type, void* C,
                              int64_t ldc);

/*
 * The norms after a block and before the next one, with the block's gate and the residual's scale, in one pass over the rows:
 *     z = branch                                          (branch_weight NULL)
 *         branch / sqrt(mean(branch^2) + eps) * branch_weight   (norm after the block)
 *     r = residual_scale * residual + branch_scale * gate * z
 *     y = r / sqrt(mean(r^2) + eps) * weight              (norm before the next block)
 * computed in fp32 and rounded once per output; y is computed from r before its rounding.  Every part may be left out: branch NULL: r = residual
 * as it is (no scale, no gate); gate NULL: 1; weight NULL: 1; outputs NULL: not wanted, but one has to be.  residual_out may
 * be the residual's own buffer (same stride): the stream is then updated in place.  Rows of the gate lie gate_ld values
 * apart, 0: one row for all.  A NaN makes its row of y NaN.  Squares are added in fp32, without scaling: where the sum of a row's
 * is beyond fp32 (a root mean square of 1.8e19 / sqrt(D)), its normed values are zero (NaN where the row is infinite).
 * staged: a workspace of K = D that takes the normed rows as MX4, quantized from fp32, for rk_npu_mx4_run_staged_device.
 */
typedef struct {
    uint32_t struct_size; /* sizeof(rk_npu_block_norm_args) */
    int rows, D;
    int residual_type, branch_type, gate_type, y_type;
    float eps, residual_scale, branch_scale;
    const void* residual;
    const void* branch;
    const void* gate;
    const float* branch_weight; /* [D] */
    const float* weight;        /* [D] */
    void* residual_out;         /* residual_type */
    void* y;
    rk_npu_mx4_workspace* staged;
    int64_t residual_ld, branch_ld, gate_ld, residual_out_ld, y_ld;
} rk_npu_block_norm_args;
/* Scales 1, eps 1e-6, everything else zero. */
void rk_npu_block_norm_args_init(rk_npu_block_norm_args* args, int rows, int D);
int rk_npu_block_norm_device(rk_npu_ctx* ctx, const rk_npu_block_norm_args* args);

/*
 * A gated FFN block on the residual stream:
 *     h = residual / sqrt(mean(residual^2) + eps) * weight,   branch = FFN(h),   residual_out = r as above,   y = the next norm of r
 * norm->residual, rows, D, types, gate, scales, branch_weight, outputs and strides as above; norm->weight is the norm BEFORE
 * the FFN and next_weight the one of y (NULL: 1; y NULL: not wanted).  branch is a buffer of rows of D values of branch_type, branch_ld
 * apart, that receives the FFN's output; norm->branch and norm->staged have to be NULL.  D is K of gate_up and N of down.
 */
int rk_npu_mx4_run_ffn_block_device(rk_npu_mx4_workspace* workspace, const rk_npu_mx4_weights* gate_up,
                                    rk_npu_mx4_workspace* down_workspace, const rk_npu_mx4_weights* down,
                                    const rk_npu_block_norm_args* norm, void* branch, const float* next_weight);

#ifdef __cplusplus
}
#endif
#endif /* RK_NPU_MX4_H */
