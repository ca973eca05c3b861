// k_fp8.hip -- translation unit for hv_gemm_fp8.h (see hv_kernels.h)
#include "hv_gemm_fp8.h"
#include "hv_kernels.h"

int hvk_gemm_fp8(const hv_gemm_fp8_params& p, hipStream_t s) { return hv_gemm_fp8_launch(p, s); }
void hvk_gemm_fp8_tile(int v) { g_hv_gemm_fp8_tile = v; }
long hvk_gemm_fp8_workspace(const hv_gemm_fp8_params& p) { return hv_gemm_fp8_workspace_of(p); }
int hvk_fp8_quantize(const bf16_t* X, long ldx, int M, int K, int block_rows, unsigned char* Q, long ldq, float* scale, long scale_row,
                     long scale_k, hipStream_t s) {
    HvQuantArgs a{X, Q, scale, ldx, ldq, scale_row, scale_k, M, K, 0};
    return hv_fp8_quantize_launch(a, block_rows, s);
}
