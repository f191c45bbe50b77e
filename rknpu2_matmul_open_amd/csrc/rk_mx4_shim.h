/*
 * rk_mx4_shim.h -- the C ABI between the host layer of the microscaled 4-bit (MX4) operators and of the block norm
 * (rk_mx4.cpp) and their kernels (rk_kernels_mx4.hip, rk_kernels_norm.hip; rk_kernels_mx4_gemm.h, in two units: rk_kernels_mx4_gemm.hip and
 * rk_kernels_mx4_swiglu.hip).  Conventions as in rk_hip_shim.h.
 *
 * Device data layouts
 * -------------------
 * "MX4 rows" (what callers see): row-major blocks of 32 values along K; block b of a row is 16 bytes of codes at
 * b * 16 (value 2 i in the low half of byte i, value 2 i + 1 in the high one) and one scale byte.
 *
 * "Operand blocks" (activations in a workspace, weights): 1 KiB pieces of 16 rows x 128 k.  Piece (rb, ks) starts at
 * (4 K4 rb + ks) * 1024, K4 = ceil(K / 512); inside it lane l = r + 16 q owns the 16 bytes at l * 16, the codes of block
 * 4 ks + q of row 16 rb + r.  One 16-byte load per lane is an operand of v_mfma_scale_f32_16x16x128_f8f6f4, whose lane
 * (r, q) holds 32 consecutive k of one row: an MX block exactly, with its one scale.  The scales of four consecutive
 * pieces share a dword: (rb, ks, l) is byte ks % 4 of the dword ((rb * K4 + ks / 4) * 64 + l), and the
 * product takes the byte by its operand select.  Blocks beyond K hold zeros.
 *
 * Weights: the rows of the operand blocks are output columns, in an order that leaves each lane of an accumulator eight
 * consecutive ones: place 16 h + 4 q + e of 32 holds column 8 q + 4 h + e of the 32.  Gate / up matrices [2F, K] alternate
 * 32 columns of the gate and the same 32 of the up half, each half padded to a multiple of 32 with zeros.
 */
#ifndef RK_MX4_SHIM_H
#define RK_MX4_SHIM_H

#include "rk_hip_shim.h"

#ifdef __cplusplus
extern "C" {
#endif

enum rkh_mx4_type { RKH_MX4_F32 = 0, RKH_MX4_F16 = 1, RKH_MX4_BF16 = 2, RKH_MX4_ROWS = 3 /* SwiGLU only: operand blocks */ };

static inline RKH_HD int64_t rkh_mx4_ks(int64_t K) { return (K + 127) / 128; }
static inline RKH_HD int64_t rkh_mx4_k4(int64_t K) { return (K + 511) / 512; }
/* Bytes of the operand blocks of `rows` rows, and of their scales. */
static inline size_t rkh_mx4_code_bytes(int64_t rows, int64_t K) { return (size_t)((rows + 15) / 16 * rkh_mx4_k4(K)) * 4096; }
static inline size_t rkh_mx4_scale_bytes(int64_t rows, int64_t K) { return (size_t)((rows + 15) / 16 * rkh_mx4_k4(K)) * 256; }
/* Columns that the operand blocks of a weight matrix hold: N, or 2 * align32(F) for gate / up pairs. */
static inline RKH_HD int64_t rkh_mx4_columns(int64_t N, int gate_up) { return gate_up ? 2 * rkh_align_up(N / 2, 32) : rkh_align_up(N, 32); }

/* Rows of values to MX4 rows and back; ldx / ldy in values. */
int rkh_mx4_quantize(void* stream, int type, int64_t rows, int K, const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales);
int rkh_mx4_dequantize(void* stream, int type, int64_t rows, int K, const uint8_t* codes, const uint8_t* scales, void* y, int64_t ldy);
/* Rows of values to operand blocks. */
int rkh_mx4_stage(void* stream, int type, int rows, int K, const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales);
/* MX4 rows of a weight matrix [N, K] to operand blocks. */
int rkh_mx4_pack(void* stream, const uint8_t* codes, const uint8_t* scales, int K, int N, int gate_up, uint8_t* dst, uint8_t* dst_scales);

typedef struct rkh_mx4_gemm_args {
    const uint8_t* A;      /* activations: operand blocks, or NULL: x holds the rows             */
    const uint8_t* a_scale;
    const uint8_t* W;      /* weights                                                             */
    const uint8_t* w_scale;
    const void* x;         /* rows of values that the few-row kernel quantizes itself             */
    int64_t ldx;
    int x_type;
    int x_norm;            /* (SwiGLU) normed first: x / sqrt(mean(x^2) + x_eps) * x_weight       */
    const float* x_weight; /* or NULL                                                             */
    float x_eps;
    int M, N, K;           /* N: columns of the result (SwiGLU: F)                                */
    int swiglu;
    int out_type;          /* rkh_mx4_type                                                        */
    void* C;               /* [M, ldc]; RKH_MX4_ROWS: operand blocks of M rows of N values        */
    int64_t ldc;
    uint8_t* c_scale;      /* RKH_MX4_ROWS: their scales                                          */
    float* scratch;        /* partial tiles of a K split over workgroups                          */
    size_t scratch_bytes;  /* too few for the split: K is not split                               */
} rkh_mx4_gemm_args;
int rkh_mx4_gemm(void* stream, const rkh_mx4_gemm_args* args);
/* Whether rkh_mx4_gemm takes the rows as they are (x) for this shape. */
int rkh_mx4_takes_rows(int M, int N, int K, int swiglu);
/* What rkh_mx4_gemm does for a shape, by arithmetic alone: the kernel (0: few rows, 1: tiles), rows and columns of a
 * workgroup and the parts that K is split into.  N as in the args. */
void rkh_mx4_route(int M, int N, int K, int swiglu, int* kernel, int* rows, int* columns, int* parts);
size_t rkh_mx4_scratch_bytes(int M, int N, int K, int swiglu);
/* ... and the most that any product of up to max_rows rows of K values needs. */
size_t rkh_mx4_scratch_most(int max_rows, int K);

typedef struct rkh_block_norm_args {
    int rows, D;
    int stream_type, branch_type, gate_type, y_type;
    float eps, residual_scale, branch_scale;
    const void* stream;    /* [rows, ld_stream] the residual stream                               */
    const void* branch;    /* [rows, ld_branch] the block's output, or NULL                       */
    const void* gate;      /* rows gate_row_stride apart (0: one row), or NULL                    */
    const float* branch_weight; /* norm after the block, or NULL                                  */
    const float* weight;   /* norm before the next one, or NULL: no weight                        */
    void* stream_out;      /* or NULL                                                             */
    void* y;               /* or NULL                                                             */
    int64_t ld_stream, ld_branch, gate_row_stride, ld_stream_out, ld_y;
    uint8_t* q;            /* operand blocks of the normed rows, or NULL                          */
    uint8_t* q_scale;
    int first;             /* (a launch's first row; the launcher's own)                           */
} rkh_block_norm_args;
int rkh_block_norm(void* stream, const rkh_block_norm_args* args);

#ifdef __cplusplus
}
#endif
#endif /* RK_MX4_SHIM_H */
