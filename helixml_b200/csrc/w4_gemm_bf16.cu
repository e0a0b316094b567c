// hx_gemm_w4 with bf16 rows of A.
#include "w4_gemm.cuh"

namespace hx {
namespace w4 {

hx_status gemm_bf16(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                    cudaStream_t st) {
    // up to eight rows: 1 x 16384 x 4096 13.3 us, 16.4 with the kernel for more; too long to be staged, 8 x 4096 x 16384, 17.1 with that one
    if (M <= 8 && fits_staged(m, M)) return launch_few(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    if (M <= 16) return launch_rows<__nv_bfloat16, 2>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    if (M <= 32) return launch_rows<__nv_bfloat16, 4>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    return launch_rows<__nv_bfloat16, 8>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
}

}  // namespace w4
}  // namespace hx
