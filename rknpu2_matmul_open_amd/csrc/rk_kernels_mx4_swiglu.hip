// MX4 products with gate / up weights: the kernels of rk_kernels_mx4_gemm.h with SwiGLU behind them.
#include "rk_kernels_mx4_gemm.h"

int rkk::launch_mx4_swiglu(hipStream_t st, const rkh_mx4_gemm_args& g) { return launch<true>(st, g); }
