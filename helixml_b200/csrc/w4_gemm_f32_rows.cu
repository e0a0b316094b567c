// hx_gemm_w4 with more than 16 fp32 rows of A (24 x 5001 x 8192: 62 us with three tiles of outputs a piece of A, 123 with one).
#include "w4_gemm.cuh"

namespace hx {
namespace w4 {

hx_status gemm_f32_rows(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                        cudaStream_t st) {
    if (M <= 24 && fills(m, 48)) HX_W4_ROWS(float, 3, 3);
    if (M <= 32) {
        if (fills(m, 48)) HX_W4_ROWS(float, 4, 3);
        HX_W4_ROWS(float, 4, 1);
    }
    HX_W4_ROWS(float, 8, 2);
}

}  // namespace w4
}  // namespace hx
