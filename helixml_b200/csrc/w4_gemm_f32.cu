// hx_gemm_w4 with up to 16 fp32 rows of A.  Cutting a piece of A into its parts costs three times what a block of codes
// does, so it is done once for three tiles of outputs where those still fill the SMs.
#include "w4_gemm.cuh"

namespace hx {
namespace w4 {

hx_status gemm_f32(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                   cudaStream_t st) {
    if (M <= 8) HX_W4_ROWS(float, 1, 1);
    if (M > 16) return gemm_f32_rows(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    if (fills(m, 48)) HX_W4_ROWS(float, 2, 3);
    HX_W4_ROWS(float, 2, 1);
}

}  // namespace w4
}  // namespace hx
