// hx_gemm_w4 with fp32 rows of A.
#include "w4_gemm.cuh"

namespace hx {
namespace w4 {

hx_status gemm_f32(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                   cudaStream_t st) {
    return launch_rows_for<float>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
}

}  // namespace w4
}  // namespace hx
