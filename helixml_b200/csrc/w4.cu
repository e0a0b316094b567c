// Weights in 4 bits with a scale per group of columns: quantising, laying out given codes, reading back, and the product of a
// few rows with such a matrix.
#include "gemm.cuh"

namespace hx {
namespace w4 {

constexpr int kBlockCols = 128, kBlockBytes = 64;
constexpr uint32_t kFill = 0x88888888u;  // eight codes of 8: what pads the last block of a row

// The 32-bit word w of a block (in the order of columns: columns 8 w .. 8 w + 7) is at word 4 (w mod 4) + w / 4.
__device__ __forceinline__ int word_at(int w) { return (w & 3) * 4 + (w >> 2); }
// column i of 8 is at nibble i / 2 + 4 (i mod 2)
__device__ __forceinline__ int nibble_of(int i) { return (i >> 1) | ((i & 1) << 2); }

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
template <typename T> __device__ __forceinline__ void store8(T *p, bool vec, const float (&v)[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            __nv_bfloat162 r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(r);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) st_f32(p + i, v[i]);
}

__device__ __forceinline__ float load_scale(const void *scale, int dtype, int64_t i) {
    return dtype == HX_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(scale)[i]) : static_cast<const float *>(scale)[i];
}

// round(w / s) to even as exact arithmetic decides it.  The fp32 quotient w * inv is off by less than 2^-20 for the |w / s| < 17
// that matter (larger ones are clamped), so only a fraction within 2^-16 of 1/2 can be decided wrongly; there the division is
// done in double, whose quotient of two fp32 numbers cannot round across a half: the distance of w / s from a half that it does
// not meet is at least 2^-25 relative.
__device__ __forceinline__ float round_quotient(float w, float s, float inv) {
    const float q = w * inv, n = rintf(q);
    if (fabsf(q - n) > 0.5f - 1.52587890625e-5f || !(fabsf(q) < 1e6f)) return (float)rint((double)w / (double)s);
    return n;
}

// One thread per word of 8 columns, 16 threads per block of 128; a group's 4, 8 or 16 threads meet in shuffles.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_kernel(const T *__restrict__ W, int64_t ldw, const hx_w4_matrix m, int blocks, bool vec) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // word of the matrix, in the order of rows and columns
    const int64_t n = i / (blocks * 16);
    const int w = (int)(i % (blocks * 16));
    const bool live = n < m.rows && w * 8 < m.cols;
    float v[8] = {};
    if (live) load8(W + n * ldw + w * 8, vec, v);
    float lo = 0.f, hi = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        bad |= !(fabsf(v[j]) <= 3.402823466e38f);
        lo = fminf(lo, v[j]);
        hi = fmaxf(hi, v[j]);
    }
    for (int o = 1; o < m.group / 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
    }
    if (n >= m.rows) return;
    uint32_t word = kFill;
    if (live) {
        float s = m.zero ? (float)(((double)hi - (double)lo) / 15.0) : (float)((double)fmaxf(hi, -lo) / 7.0);
        if (m.scale_dtype == HX_BF16) s = __bfloat162float(__float2bfloat16_rn(s));
        if (bad) s = __int_as_float(0x7fc00000);
        float zero = 8.f;
        if (s > 0.f) {   // neither zero nor NaN
            const float inv = 1.0f / s;
            if (m.zero) zero = fminf(fmaxf(round_quotient(-lo, s, inv), 0.f), 15.f);
            const float low = m.zero ? 0.f : 1.f;
            word = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float q = fminf(fmaxf(round_quotient(v[j], s, inv) + zero, low), 15.f);
                word |= (uint32_t)q << (4 * nibble_of(j));
            }
        }
        if (w % (m.group / 8) == 0) {
            const int64_t at = n * (m.cols / m.group) + w / (m.group / 8);
            if (m.scale_dtype == HX_BF16) static_cast<__nv_bfloat16 *>(m.scale)[at] = __float2bfloat16_rn(s);
            else static_cast<float *>(m.scale)[at] = s;
            if (m.zero) m.zero[at] = (uint8_t)zero;
        }
    }
    reinterpret_cast<uint32_t *>(m.codes)[(n * blocks + w / 16) * 16 + word_at(w & 15)] = word;
}

__global__ void __launch_bounds__(256)
pack_kernel(const uint8_t *__restrict__ in, int64_t ldc, const hx_w4_matrix m, int blocks) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t n = i / (blocks * 16);
    const int w = (int)(i % (blocks * 16));
    if (n >= m.rows) return;
    uint32_t word = kFill;
    if (w * 8 < m.cols) {
        word = 0;
        const uint8_t *p = in + n * ldc + w * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) word |= (uint32_t)(p[j] & 15) << (4 * nibble_of(j));
    }
    reinterpret_cast<uint32_t *>(m.codes)[(n * blocks + w / 16) * 16 + word_at(w & 15)] = word;
}

template <typename T>
__global__ void __launch_bounds__(256)
dequantize_kernel(const hx_w4_matrix m, T *__restrict__ W, int64_t ldw, int blocks, bool vec) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int words = m.cols / 8;
    const int64_t n = i / words;
    const int w = (int)(i % words);
    if (n >= m.rows) return;
    const uint32_t word = reinterpret_cast<const uint32_t *>(m.codes)[(n * blocks + w / 16) * 16 + word_at(w & 15)];
    const int64_t at = n * (m.cols / m.group) + w / (m.group / 8);
    const float s = load_scale(m.scale, m.scale_dtype, at);
    const int zero = m.zero ? m.zero[at] : 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s * (float)((int)((word >> (4 * nibble_of(j))) & 15) - zero);
    store8(W + n * ldw + w * 8, vec, v);
}

// One warp per output column and 8 rows of A: a lane takes every 32nd word of 8 columns.
template <typename TA, typename TC, int EPI>
__global__ void __launch_bounds__(128)
gemm_w4_kernel(const TA *__restrict__ A, int64_t lda, const hx_w4_matrix m, const float *__restrict__ bias, TC *__restrict__ C,
               int64_t ldc, int M, int blocks) {
    const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, r0 = blockIdx.y * 8;
    if (n >= m.rows) return;
    const uint32_t *row = reinterpret_cast<const uint32_t *>(m.codes) + n * blocks * 16;
    float acc[8] = {};
    for (int w = lane; w < m.cols / 8; w += 32) {
        const uint32_t word = row[(w >> 4) * 16 + word_at(w & 15)];
        const int64_t at = n * (m.cols / m.group) + w / (m.group / 8);
        const float s = load_scale(m.scale, m.scale_dtype, at);
        const int zero = m.zero ? m.zero[at] : 8;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (r0 + r >= M) break;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                sum = fmaf((float)((int)((word >> (4 * nibble_of(j))) & 15) - zero), ld_f32(A + (r0 + r) * lda + w * 8 + j), sum);
            acc[r] = fmaf(s, sum, acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (lane == 0 && r0 + r < M) st_f32(C + (r0 + r) * ldc + n, gemm::apply_epilogue<EPI>(acc[r] + (bias ? bias[n] : 0.f)));
    }
}

static hx_status check_matrix(const char *who, const hx_w4_matrix *m) {
    HX_REQUIRE(m != nullptr, HX_ERR_INVALID_INPUT, "%s: the matrix is NULL", who);
    HX_REQUIRE(m->rows >= 0 && m->cols >= 0, HX_ERR_INVALID_DIMENSION, "%s: a matrix of %d x %d", who, m->rows, m->cols);
    HX_REQUIRE(m->group == 32 || m->group == 64 || m->group == 128, HX_ERR_INVALID_DIMENSION, "%s: group %d is not 32, 64 or 128", who,
               m->group);
    HX_REQUIRE(m->cols % m->group == 0, HX_ERR_SHAPE_MISMATCH, "%s: %d columns are not a multiple of the group %d", who, m->cols, m->group);
    HX_REQUIRE(m->scale_dtype == HX_F32 || m->scale_dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH,
               "%s: scale_dtype %d is neither HX_F32 nor HX_BF16", who, m->scale_dtype);
    if (m->rows == 0 || m->cols == 0) return HX_OK;
    HX_REQUIRE(m->codes && m->scale, HX_ERR_INVALID_INPUT, "%s: codes and scale must not be NULL", who);
    HX_REQUIRE(((uintptr_t)m->codes & 15) == 0, HX_ERR_INVALID_INPUT, "%s: codes must be 16-byte aligned", who);
    return HX_OK;
}
static int blocks_of(int cols) { return (int)(((int64_t)cols + kBlockCols - 1) / kBlockCols); }
// The grid of a kernel with one thread per item, if there is one.
static hx_status grid_of(const char *who, int64_t items, unsigned *grid) {
    const int64_t g = (items + 255) / 256;
    HX_REQUIRE(g <= 0x7fffffff, HX_ERR_INVALID_DIMENSION, "%s: the matrix is too large for one launch", who);
    *grid = (unsigned)g;
    return HX_OK;
}
static bool aligned8(const void *p, int64_t ld, int dtype) {   // rows whose every 8 elements are aligned for 16-byte accesses
    return ((uintptr_t)p & 15) == 0 && (ld * (int64_t)dtype_size(dtype)) % 16 == 0;
}

}  // namespace w4
}  // namespace hx

using namespace hx;
using namespace hx::w4;

extern "C" {

size_t hx_w4_row_bytes(int32_t cols) { return cols <= 0 ? 0 : (size_t)blocks_of(cols) * kBlockBytes; }

hx_status hx_w4_quantize(const void *W, int64_t ldw, int32_t w_dtype, const hx_w4_matrix *m, void *stream) {
    const hx_status s = check_matrix("hx_w4_quantize", m);
    if (s != HX_OK) return s;
    HX_REQUIRE(w_dtype == HX_F32 || w_dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "hx_w4_quantize: w_dtype %d is neither HX_F32 nor HX_BF16", w_dtype);
    if (m->rows == 0 || m->cols == 0) return HX_OK;
    HX_REQUIRE(W != nullptr, HX_ERR_INVALID_INPUT, "hx_w4_quantize: W is NULL");
    HX_REQUIRE(ldw >= 0, HX_ERR_INVALID_INPUT, "hx_w4_quantize: negative stride");
    const int blocks = blocks_of(m->cols);
    unsigned grid;
    const hx_status g = grid_of("hx_w4_quantize", (int64_t)m->rows * blocks * 16, &grid);
    if (g != HX_OK) return g;
    const bool vec = aligned8(W, ldw, w_dtype);
    if (w_dtype == HX_BF16) quantize_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(static_cast<const __nv_bfloat16 *>(W), ldw, *m, blocks, vec);
    else quantize_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(static_cast<const float *>(W), ldw, *m, blocks, vec);
    return check_launch("quantize_kernel");
}

hx_status hx_w4_pack(const uint8_t *in, int64_t ldc, const hx_w4_matrix *m, void *stream) {
    const hx_status s = check_matrix("hx_w4_pack", m);
    if (s != HX_OK) return s;
    if (m->rows == 0 || m->cols == 0) return HX_OK;
    HX_REQUIRE(in != nullptr, HX_ERR_INVALID_INPUT, "hx_w4_pack: the codes are NULL");
    HX_REQUIRE(ldc >= 0, HX_ERR_INVALID_INPUT, "hx_w4_pack: negative stride");
    const int blocks = blocks_of(m->cols);
    unsigned grid;
    const hx_status g = grid_of("hx_w4_pack", (int64_t)m->rows * blocks * 16, &grid);
    if (g != HX_OK) return g;
    pack_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(in, ldc, *m, blocks);
    return check_launch("pack_kernel");
}

hx_status hx_w4_dequantize(const hx_w4_matrix *m, void *W, int64_t ldw, int32_t w_dtype, void *stream) {
    const hx_status s = check_matrix("hx_w4_dequantize", m);
    if (s != HX_OK) return s;
    HX_REQUIRE(w_dtype == HX_F32 || w_dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "hx_w4_dequantize: w_dtype %d is neither HX_F32 nor HX_BF16", w_dtype);
    if (m->rows == 0 || m->cols == 0) return HX_OK;
    HX_REQUIRE(W != nullptr, HX_ERR_INVALID_INPUT, "hx_w4_dequantize: W is NULL");
    HX_REQUIRE(m->rows == 1 || ldw >= m->cols, HX_ERR_SHAPE_MISMATCH, "hx_w4_dequantize: rows of W overlap (stride %lld)", (long long)ldw);
    unsigned grid;
    const hx_status g = grid_of("hx_w4_dequantize", (int64_t)m->rows * (m->cols / 8), &grid);
    if (g != HX_OK) return g;
    const bool vec = aligned8(W, ldw, w_dtype);
    const int blocks = blocks_of(m->cols);
    if (w_dtype == HX_BF16) dequantize_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(*m, static_cast<__nv_bfloat16 *>(W), ldw, blocks, vec);
    else dequantize_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(*m, static_cast<float *>(W), ldw, blocks, vec);
    return check_launch("dequantize_kernel");
}

hx_status hx_gemm_w4(const void *A, int64_t lda, int32_t a_dtype, const hx_w4_matrix *m, const float *bias, void *C, int64_t ldc,
                     int32_t c_dtype, int32_t M, int32_t epilogue, void *stream) {
    const hx_status s = check_matrix("hx_gemm_w4", m);
    if (s != HX_OK) return s;
    HX_REQUIRE(M >= 0, HX_ERR_INVALID_DIMENSION, "hx_gemm_w4: %d rows", M);
    HX_REQUIRE((a_dtype == HX_F32 || a_dtype == HX_BF16) && (c_dtype == HX_F32 || c_dtype == HX_BF16), HX_ERR_DTYPE_MISMATCH,
               "hx_gemm_w4: A and C are HX_F32 or HX_BF16, got %d and %d", a_dtype, c_dtype);
    HX_REQUIRE(epilogue == gemm::kEpiNone || epilogue == gemm::kEpiSilu || epilogue == gemm::kEpiSoftplus, HX_ERR_INVALID_INPUT,
               "hx_gemm_w4: unknown epilogue %d", epilogue);
    if (M == 0 || m->rows == 0) return HX_OK;
    HX_REQUIRE(m->cols > 0, HX_ERR_INVALID_DIMENSION, "hx_gemm_w4: a matrix without columns");
    HX_REQUIRE(A && C, HX_ERR_INVALID_INPUT, "hx_gemm_w4: A and C must not be NULL");
    HX_REQUIRE(lda >= 0, HX_ERR_INVALID_INPUT, "hx_gemm_w4: negative stride");
    HX_REQUIRE(M == 1 || ldc >= m->rows, HX_ERR_SHAPE_MISMATCH, "hx_gemm_w4: rows of C overlap (stride %lld)", (long long)ldc);
    HX_REQUIRE((M + 7) / 8 <= 65535, HX_ERR_INVALID_DIMENSION, "hx_gemm_w4: %d rows", M);
    const dim3 grid((unsigned)((m->rows + 3) / 4), (unsigned)((M + 7) / 8));
    const int blocks = blocks_of(m->cols);
    auto st = (cudaStream_t)stream;
#define HX_W4_EPI(TA, TC, E) gemm_w4_kernel<TA, TC, E><<<grid, 128, 0, st>>>(static_cast<const TA *>(A), lda, *m, bias, static_cast<TC *>(C), ldc, M, blocks)
#define HX_W4_TYPES(TA, TC)                                                   \
    do {                                                                      \
        if (epilogue == gemm::kEpiNone) HX_W4_EPI(TA, TC, gemm::kEpiNone);    \
        else if (epilogue == gemm::kEpiSilu) HX_W4_EPI(TA, TC, gemm::kEpiSilu); \
        else HX_W4_EPI(TA, TC, gemm::kEpiSoftplus);                           \
    } while (0)
    if (a_dtype == HX_BF16) {
        if (c_dtype == HX_BF16) HX_W4_TYPES(__nv_bfloat16, __nv_bfloat16);
        else HX_W4_TYPES(__nv_bfloat16, float);
    } else {
        if (c_dtype == HX_BF16) HX_W4_TYPES(float, __nv_bfloat16);
        else HX_W4_TYPES(float, float);
    }
    return check_launch("gemm_w4_kernel");
}

}  // extern "C"
