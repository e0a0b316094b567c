// hx_gemm_w4 with bf16 rows of A.
#include "w4_gemm.cuh"

namespace hx {
namespace w4 {

hx_status gemm_bf16(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                    cudaStream_t st) {
    if (M <= 8) HX_W4_ROWS(__nv_bfloat16, 1, 1);
    if (M <= 16) HX_W4_ROWS(__nv_bfloat16, 2, 1);
    if (M <= 32) {   // a piece of A for two tiles of outputs: 32 x 16384 x 4096 28 us, 34 with one
        if (fills(m, 32)) HX_W4_ROWS(__nv_bfloat16, 4, 2);
        HX_W4_ROWS(__nv_bfloat16, 4, 1);
    }
    HX_W4_ROWS(__nv_bfloat16, 8, 1);   // 64 x 16384 x 4096 58 us, 63 with two
}

}  // namespace w4
}  // namespace hx
