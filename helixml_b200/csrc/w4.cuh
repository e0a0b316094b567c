// The 4-bit matrix: its layout and what the kernels on it share.
#pragma once

#include "gemm.cuh"

namespace hx {
namespace w4 {

constexpr int kBlockCols = 128, kBlockBytes = 64;
constexpr uint32_t kFill = 0x88888888u;  // eight codes of 8: what pads the last block of a row

// The 32-bit word w of a block (in the order of columns: columns 8 w .. 8 w + 7) is at word 4 (w mod 4) + w / 4.
__device__ __forceinline__ int word_at(int w) { return (w & 3) * 4 + (w >> 2); }
// column i of 8 is at nibble i / 2 + 4 (i mod 2)
__device__ __forceinline__ int nibble_of(int i) { return (i >> 1) | ((i & 1) << 2); }
__device__ __forceinline__ int column_of(int p) { return (p & 3) * 2 + (p >> 2); }

// A thread's eight consecutive elements, as fp32.
template <typename T> __device__ __forceinline__ void load8(const T *p, bool vec, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const float4 lo = reinterpret_cast<const float4 *>(p)[0], hi = reinterpret_cast<const float4 *>(p)[1];
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
            v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
            return;
        }
    } else {
        if (vec) {
            const uint4 r = *reinterpret_cast<const uint4 *>(p);
            const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(u[i] << 16);
                v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ld_f32(p + i);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}
// 32 bytes, a whole sector in one instruction where the address allows it
__device__ __forceinline__ void store32(void *p, const uint32_t (&u)[8]) {
    if (((uintptr_t)p & 31) == 0) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
                     "r"(u[6]), "r"(u[7])
                     : "memory");
    } else {
        static_cast<uint4 *>(p)[0] = make_uint4(u[0], u[1], u[2], u[3]);
        static_cast<uint4 *>(p)[1] = make_uint4(u[4], u[5], u[6], u[7]);
    }
}
template <typename T> __device__ __forceinline__ void store16(T *p, bool vec, const float (&v)[16]) {
    if (vec) {
        uint32_t u[8];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(v[half * 8 + i]);
                store32(p + half * 8, u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            store32(p, u);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) st_f32(p + i, v[i]);
}

__device__ __forceinline__ float load_scale(const void *scale, int dtype, int64_t i) {
    return dtype == HX_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(scale)[i]) : static_cast<const float *>(scale)[i];
}

inline int blocks_of(int cols) { return (int)(((int64_t)cols + kBlockCols - 1) / kBlockCols); }
inline bool aligned8(const void *p, int64_t ld, int dtype) {   // rows whose every 8 elements are aligned for 16-byte accesses
    return ((uintptr_t)p & 15) == 0 && (ld * (int64_t)dtype_size(dtype)) % 16 == 0;
}

// C = A W^T (+ bias) (+ activation) on checked arguments, in translation units of their own (w4_gemm_*.cu).
hx_status gemm_bf16(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                    cudaStream_t st);
hx_status gemm_f32(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                   cudaStream_t st);

}  // namespace w4
}  // namespace hx
