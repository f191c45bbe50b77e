/*
 * rk_g4_shim.h -- the C ABI between the host layer of the group-scaled 4-bit (G4) layers (rk_g4.cpp) and their kernels
 * (rk_kernels_g4.hip: packing, staging, few rows; rk_kernels_g4_tile.h in three units: tiles).  Conventions as in rk_hip_shim.h.
 *
 * Device data layouts
 * -------------------
 * Codes: 1 KiB pieces of 16 places x 128 k.  Piece (pb, kb) starts at (pb * KB + kb) * 1024, KB = ceil(K / 128).  Lane l = c + 16 q of a
 * piece owns the 16 bytes at l * 16; its dword i holds the codes of k = 128 kb + 32 i + 8 q + 0..7 of place 16 pb + c, an even k + t at
 * bits 2 t and an odd one at bits 16 + 2 (t - 1), so that one mask leaves two neighbours in the halves of a dword.  Dword i of all lanes
 * is an operand of a 16x16x32 product; dword i of the lanes with q = h and q = h + 2 are two consecutive ones of 32x32x16, whose
 * lane (c + 16 b, h) holds 8 k of 32 places.  Codes beyond K and N are zero.
 *
 * Scales: a dword for each place and internal group of 128 / gpb (gpb = 1, 2, 4: groups in a piece) k, piece by piece as the codes: [pb][kb][c][gpb], the
 * scale's 16 bits above 0x6400 + zero point (the half 1024 + zero point).  Beyond K and N the scale is zero.
 *
 * Places of columns, in units of 64 (16-place blocks 0..3 of it): place 16 (2 b + j) + c is column 32 b + 2 c + j of the 64, so that lane c
 * + 16 b of two accumulators j of 32 places has two neighbouring columns.  Gate / up matrices: column 16 b + c of 32, j = 0 of the gate and j = 1 of
 * the up half.
 *
 * Staged rows: fp16, row-major, Kp = 128 KB values apart, zeros beyond K; bf16 rows times 2^e(row) (exact for all that is not below 2^-31 of the
 * row's largest), the exponents in an array of their own.
 */
#ifndef RK_G4_SHIM_H
#define RK_G4_SHIM_H

#include "rk_mx4_shim.h" /* element types */

#ifdef __cplusplus
extern "C" {
#endif

static inline RKH_HD int64_t rkh_g4_kb(int64_t K) { return (K + 127) / 128; }
/* Places of a matrix of N columns (2F: gate / up pairs). */
static inline RKH_HD int64_t rkh_g4_places(int64_t N, int gate_up) { return gate_up ? 2 * rkh_align_up(N / 2, 32) : rkh_align_up(N, 64); }
/* Internal groups in a piece for groups of `group` values: the longest of 128, 64 and 32 that divides it. */
static inline RKH_HD int rkh_g4_gpb(int group) { return group % 128 == 0 ? 1 : group % 64 == 0 ? 2 : 4; }
static inline size_t rkh_g4_code_bytes(int64_t places, int64_t K) { return (size_t)(places * rkh_g4_kb(K)) * 64; }
static inline size_t rkh_g4_scale_bytes(int64_t places, int64_t K, int gpb) { return (size_t)(places * rkh_g4_kb(K) * gpb) * 4; }
static inline size_t rkh_g4_staged_bytes(int64_t rows, int64_t K) { return (size_t)(rows * rkh_g4_kb(K)) * 256; }

/* Codes [N][ceil(K / 2)], scales [N][groups] (16 bits each) and zero points [N][groups] (or NULL: 8) to the layouts above. */
int rkh_g4_pack(void* stream, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int K, int N, int group, int gate_up, uint8_t* dst,
                uint32_t* dst_scales);

typedef struct rkh_g4_args {
    const uint8_t* W;
    const uint32_t* w_scale;
    int gpb;
    int scale_type;      /* of the scales' 16 bits: rkh_mx4_type  */
    const void* x;       /* [M, ldx] fp16 or bf16                 */
    int64_t ldx;
    int x_type;
    int M, N, K;         /* N: columns of the result (SwiGLU: F)  */
    int swiglu;
    int out_type;
    void* C;
    int64_t ldc;
    uint16_t* staged;    /* staged rows, where a product needs them */
    int* exponents;      /* of M rows, and room for whole tiles of 256 */
    float* scratch;      /* partial tiles of a K split over workgroups */
    size_t scratch_bytes;
} rkh_g4_args;
int rkh_g4_run(void* stream, const rkh_g4_args* args);
/* What rkh_g4_run does for a shape, by arithmetic alone: the kernel (0: few rows, 1: tiles), rows and columns (SwiGLU: of both halves) of a
 * workgroup and the parts that K is split into.  N as in the args. */
void rkh_g4_route(int M, int N, int K, int gpb, int swiglu, int* kernel, int* rows, int* columns, int* parts);
/* ... and of up to 16 rows which few-row kernel: rows that it is made for (0: it loads operands), columns and waves of a workgroup, and whether a wave loads more than once. */
void rkh_g4_few_route(int M, int N, int K, int gpb, int swiglu, int* rows, int* columns, int* waves, int* again);
size_t rkh_g4_scratch_bytes(int M, int N, int K, int gpb, int swiglu);
/* ... and the most that any product of up to max_rows rows of K values needs. */
size_t rkh_g4_scratch_most(int max_rows, int K);

#ifdef __cplusplus
}
#endif
#endif /* RK_G4_SHIM_H */
