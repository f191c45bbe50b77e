// MX4 products with weights of single columns, and the entry points of all of them; the kernels are in rk_kernels_mx4_gemm.h.
#include "rk_kernels_mx4_gemm.h"

extern "C" {

int rkh_mx4_gemm(void* stream, const rkh_mx4_gemm_args* args) {
    if (!args->M || !args->N) return RKH_OK;
    if (!args->A && !rkh_mx4_takes_rows(args->M, args->N, args->K, args->swiglu)) return RKH_ERR_RUNTIME;
    return args->swiglu ? rkk::launch_mx4_swiglu((hipStream_t)stream, *args) : launch<false>((hipStream_t)stream, *args);
}
int rkh_mx4_takes_rows(int M, int N, int K, int swiglu) {
    // Every workgroup quantizes all rows: up to 16384 values (1 x 14336 -> 4096 7.2 us, with a launch of its own in front 9.1; 4 x 4096 -> 14336
    // 8.8 and 9.7; 4 x 14336 -> 4096 11.5 and 9.1), in whole pieces of eight.
    (void)N, (void)swiglu;
    return M <= MX_ROWS && K % 8 == 0 && (int64_t)M * K <= 16384;
}
void rkh_mx4_route(int M, int N, int K, int swiglu, int* kernel, int* rows, int* columns, int* parts) {
    const MxRoute r = mx_route(M, N, K, swiglu);
    *kernel = r.few ? 0 : 1;
    *rows = r.few ? 16 * r.rm : 32 * r.rm;
    *columns = r.few ? 16 * r.cn : 32 * r.cn;
    *parts = r.parts;
}
// (mx_route: K in parts of four groups or more, a part for each compute unit at most, tiles of up to 128 x 128)
size_t rkh_mx4_scratch_most(int max_rows, int K) { return max_rows > 16 && rkh_mx4_k4(K) >= 8 ? (size_t)MX_CUS * 128 * 128 * 4 : 0; }
size_t rkh_mx4_scratch_bytes(int M, int N, int K, int swiglu) { return mx_scratch(mx_route(M, N, K, swiglu)); }

} // extern "C"
