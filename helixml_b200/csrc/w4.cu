// Weights in 4 bits with a scale per group of columns: quantising, laying out given codes, reading back, and the
// entry points of the product.
#include <type_traits>

#include "hx_overlap.h"
#include "hx_tma.cuh"
#include "w4.cuh"

namespace hx {
namespace w4 {

// Row and column of item i of a matrix with `across` items a row; nearly always 32 bits do.
__device__ __forceinline__ void split(int64_t i, int across, int64_t &row, int &col) {
    if (i >> 32 == 0) {
        row = (uint32_t)i / (uint32_t)across;
        col = (int)((uint32_t)i - (uint32_t)row * (uint32_t)across);
    } else {
        row = i / across;
        col = (int)(i - row * across);
    }
}

constexpr float kRound = 12582912.f;   // 1.5 * 2^23: adding it rounds to an integer, ties to even, and leaves that in the low bits
constexpr float kNear = 0.5f - 1.52587890625e-5f;   // 1/2 - 2^-16

// w / s rounded as exact arithmetic decides it, given fp32's q = w * (1 / s) and n, that rounded.  The reciprocal and the product round
// once each, so q is off by at most 2^-23 of itself, less than 2^-18 for |w / s| < 17 (larger ones are clamped).  So only a q within
// 2^-16 of a half can have gone to the wrong side, and there the sign of w - half * s, which a fused multiply-add gives exactly, tells.
__device__ __forceinline__ float settle(float w, float s, float q, float n) {
    const float e = q - n;
    if (!(fabsf(e) > kNear)) return n;
    const float step = e > 0.f ? 1.f : -1.f, d = step * fmaf(-(n + 0.5f * step), s, w);
    const bool odd = (int)n & 1;
    return d > 0.f || (d == 0.f && odd) ? n + step : n;
}

constexpr int kEach = 2;   // words of a thread
constexpr float kLargest = 3.402823466e38f;
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A thread takes 16 columns, two words; a group's threads meet in shuffles.  8192 x 8192 fp32 48.5 us in a graph (95 % of a copy's rate);
// 16384 x 4096 bf16 with bf16 scales 44.7 (57 %): half the bytes under the same instructions a thread, two thirds of the issue slots.
template <typename T, bool ZERO>
__global__ void __launch_bounds__(256)
quantize_kernel(const T *__restrict__ W, int64_t ldw, const hx_w4_matrix m, int blocks, int shift, bool vec) {   // group = 2^shift
    constexpr int per = 8 * kEach;
    int64_t n;   // row, and the thread's part of the row
    int part;
    split((int64_t)blockIdx.x * 256 + threadIdx.x, blocks * (kBlockCols / per), n, part);
    const bool live = n < m.rows && part * per < m.cols;
    float v[kEach][8] = {};
    if (live) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) load8(W + n * ldw + part * per + i * 8, vec, v[i]);
    }
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (ZERO) lo = min_nan(lo, v[i][j]), hi = max_nan(hi, v[i][j]);
            else hi = max_nan(hi, fabsf(v[i][j]));
        }
    if (!(hi <= kLargest && lo >= -kLargest)) hi = __int_as_float(0x7f800000);   // an infinity or a NaN travels with the maximum
    for (int o = 1; o * per < m.group; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        if constexpr (ZERO) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (n >= m.rows) return;
    uint32_t word[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) word[i] = kFill;
    if (live) {
        float s, zero = 8.f;
        if constexpr (ZERO) {
            const double d = (double)hi - (double)lo;
            s = (float)d / 15.f;
            if ((double)(float)d != d) s = (float)(d / 15.0);
        } else {
            s = hi / 7.f;
        }
        if (m.scale_dtype == HX_BF16) s = __bfloat162float(__float2bfloat16_rn(s));
        if (hi > kLargest) s = __int_as_float(0x7fc00000);
        if (s > 0.f) {   // neither zero nor NaN
            float t = s;   // the divisor, out of the range where its reciprocal overflows
            float worst = 0.f;
            if (s < 0x1p-100f) {   // also where s is so coarse that quotients may lie beyond their range
                worst = 1.f;
                t *= 0x1p100f;
                lo *= 0x1p100f;
#pragma unroll
                for (int i = 0; i < kEach; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[i][j] *= 0x1p100f;
            }
            const float inv = 1.f / t;
            if constexpr (ZERO) {
                const float q = fminf(-lo * inv, 16.f);
                zero = fminf(fmaxf(settle(-lo, t, q, (q + kRound) - kRound), 0.f), 15.f);
            }
            const float low = (ZERO ? 0.f : 1.f) - zero, high = 15.f - zero;
            // A word is the sum of its codes times powers of 16, and the integer that kRound leaves in the low bits is one term
            // of it, without its zero point and with kRound's own bits on top, both of which `rest` makes good.  Symmetric
            // quotients are within 7 (1 + 2^-8) by themselves.
            const uint32_t rest = ((uint32_t)zero - __float_as_uint(kRound)) * 0x11111111u;
            const float2 inv2 = splat2(inv), round2 = splat2(kRound), back2 = splat2(-kRound), minus2 = splat2(-1.f), minus_t2 = splat2(-t);
            auto words = [&](auto short_operands) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    float u[8];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float2 w = make_float2(v[i][j], v[i][j + 1]);
                        float2 q = mul2(w, inv2);
                        if constexpr (short_operands) q = fma2(fma2(q, minus_t2, w), inv2, q);
                        if constexpr (ZERO) q = make_float2(fminf(fmaxf(q.x, low), high), fminf(fmaxf(q.y, low), high));
                        const float2 r = add2(q, round2);
                        if constexpr (!short_operands) {
                            const float2 off = fma2(add2(r, back2), minus2, q);
                            worst = fmaxf(worst, fmaxf(fabsf(off.x), fabsf(off.y)));
                        }
                        u[j] = r.x, u[j + 1] = r.y;
                    }
                    uint32_t sum = 0;
#pragma unroll
                    for (int p = 7; p >= 0; --p) sum = (sum << 4) + __float_as_uint(u[column_of(p)]);
                    word[i] = sum + rest;
                }
            };
            // Weights and scales of 8 bits: a quotient is a half or at least 2^-9 from one, and one that is a half is common (16384 x
            // 4096: 66 us where every warp settles some).  The remainder w - q t is exact, and with it q is a half where the quotient is.
            if (sizeof(T) == 2 && m.scale_dtype == HX_BF16) words(std::true_type{});
            else words(std::false_type{});
            if (worst > kNear) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    word[i] = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float q = fminf(fmaxf(v[i][j] * inv, low), high);
                        word[i] |= (uint32_t)(settle(v[i][j], t, q, (q + kRound) - kRound) + zero) << (4 * nibble_of(j));
                    }
                }
            }
        }
        if ((part * per & (m.group - 1)) == 0) {
            const int64_t at = n * (m.cols >> shift) + (part * per >> shift);
            if (m.scale_dtype == HX_BF16) static_cast<__nv_bfloat16 *>(m.scale)[at] = __float2bfloat16_rn(s);
            else static_cast<float *>(m.scale)[at] = s;
            if constexpr (ZERO) m.zero[at] = (uint8_t)zero;
        }
    }
    uint32_t *row = reinterpret_cast<uint32_t *>(m.codes) + (n * blocks + part / (16 / kEach)) * 16;
#pragma unroll
    for (int i = 0; i < kEach; ++i) row[word_at(part % (16 / kEach) * kEach + i)] = word[i];
}

// A word of eight codes a thread, read byte by byte at any alignment, once when a model is loaded: 16384 x 4096 34 us (45 % of a copy's
// rate).
__global__ void __launch_bounds__(256)
pack_kernel(const uint8_t *__restrict__ in, int64_t ldc, const hx_w4_matrix m, int blocks) {
    int64_t n;
    int w;
    split((int64_t)blockIdx.x * 256 + threadIdx.x, blocks * 16, n, w);
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

// A thread takes 16 columns, two words of one group; they are 64 or 32 bytes of W, written a sector at a time: 8192 x 8192 fp32 47.3 us
// in a graph (97 % of a copy's rate), 16384 x 4096 bf16 31.8 (80 %).  (As calls of their own, 51 and 37, where 16-byte stores of a word
// a thread took 74 and 49.)
template <typename T>
__global__ void __launch_bounds__(256)
dequantize_kernel(const hx_w4_matrix m, T *__restrict__ W, int64_t ldw, int blocks, int shift, bool vec) {
    int64_t n;
    int part;
    split((int64_t)blockIdx.x * 256 + threadIdx.x, m.cols >> 4, n, part);
    if (n >= m.rows) return;
    const uint32_t *words = reinterpret_cast<const uint32_t *>(m.codes) + (n * blocks + (part >> 3)) * 16;
    const uint32_t word[2] = {words[word_at((part & 7) * 2)], words[word_at((part & 7) * 2 + 1)]};
    const int64_t at = n * (m.cols >> shift) + (part * 16 >> shift);
    const float s = load_scale(m.scale, m.scale_dtype, at);
    const float base = 8388608.f + (float)(m.zero ? m.zero[at] : 8);   // 2^23: a code in its low bits adds itself
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = s * (__uint_as_float(((word[j / 8] >> (4 * nibble_of(j % 8))) & 15u) | 0x4b000000u) - base);
    store16(W + n * ldw + part * 16, vec, v);
}

static hx_status check_matrix(const char *who, const hx_w4_matrix *m) {
    HX_REQUIRE(m != nullptr, HX_ERR_INVALID_INPUT, "%s: the matrix is NULL", who);
    HX_REQUIRE(m->rows >= 0 && m->rows <= 0x7fffff00 && m->cols >= 0, HX_ERR_INVALID_DIMENSION, "%s: a matrix of %d x %d", who, m->rows, m->cols);
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
static int64_t codes_bytes(const hx_w4_matrix &m) { return (int64_t)m.rows * blocks_of(m.cols) * kBlockBytes; }
static int64_t scale_bytes(const hx_w4_matrix &m) { return (int64_t)m.rows * (m.cols / m.group) * (int64_t)dtype_size(m.scale_dtype); }
static int64_t zero_bytes(const hx_w4_matrix &m) { return (int64_t)m.rows * (m.cols / m.group); }
#define HX_W4_PARTS(M) {"codes", dense_of((M).codes, codes_bytes(M))}, {"scale", dense_of((M).scale, scale_bytes(M))}, {"zero", dense_of((M).zero, zero_bytes(M))}

// The grid of a kernel with one thread per item, if there is one.
static hx_status grid_of(const char *who, int64_t items, unsigned *grid) {
    const int64_t g = (items + 255) / 256;
    HX_REQUIRE(g <= 0x7fffffff, HX_ERR_INVALID_DIMENSION, "%s: the matrix is too large for one launch", who);
    *grid = (unsigned)g;
    return HX_OK;
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
    const Operand outs[] = {HX_W4_PARTS(*m)}, ins[] = {{"W", rows_of(W, m->rows, ldw, 1, 0, m->cols, dtype_size(w_dtype))}};
    const char *one, *other;
    HX_REQUIRE(!shared_operands(outs, ins, one, other), HX_ERR_INVALID_INPUT, "hx_w4_quantize: %s and %s share memory", one, other);
    const hx_status g = grid_of("hx_w4_quantize", (int64_t)m->rows * blocks * (16 / kEach), &grid);
    if (g != HX_OK) return g;
    const bool vec = aligned8(W, ldw, w_dtype);
    const int shift = m->group == 32 ? 5 : m->group == 64 ? 6 : 7;
    auto st = (cudaStream_t)stream;
    if (w_dtype == HX_BF16) {
        auto w = static_cast<const __nv_bfloat16 *>(W);
        if (m->zero) quantize_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(w, ldw, *m, blocks, shift, vec);
        else quantize_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(w, ldw, *m, blocks, shift, vec);
    } else {
        auto w = static_cast<const float *>(W);
        if (m->zero) quantize_kernel<float, true><<<grid, 256, 0, st>>>(w, ldw, *m, blocks, shift, vec);
        else quantize_kernel<float, false><<<grid, 256, 0, st>>>(w, ldw, *m, blocks, shift, vec);
    }
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
    const Operand outs[] = {{"codes", dense_of(m->codes, codes_bytes(*m))}}, ins[] = {{"the codes given", rows_of(in, m->rows, ldc, 1, 0, m->cols, 1)}};
    const char *one, *other;
    HX_REQUIRE(!shared_operands(outs, ins, one, other), HX_ERR_INVALID_INPUT, "hx_w4_pack: %s and %s share memory", one, other);
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
    const Operand outs[] = {{"W", rows_of(W, m->rows, ldw, 1, 0, m->cols, dtype_size(w_dtype))}}, ins[] = {HX_W4_PARTS(*m)};
    const char *one, *other;
    HX_REQUIRE(!shared_operands(outs, ins, one, other), HX_ERR_INVALID_INPUT, "hx_w4_dequantize: %s and %s share memory", one, other);
    const hx_status g = grid_of("hx_w4_dequantize", (int64_t)m->rows * (m->cols / 16), &grid);
    if (g != HX_OK) return g;
    const bool vec = aligned8(W, ldw, w_dtype);
    const int shift = m->group == 32 ? 5 : m->group == 64 ? 6 : 7;
    const int blocks = blocks_of(m->cols);
    if (w_dtype == HX_BF16) dequantize_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(*m, static_cast<__nv_bfloat16 *>(W), ldw, blocks, shift, vec);
    else dequantize_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(*m, static_cast<float *>(W), ldw, blocks, shift, vec);
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
    const Operand outs[] = {{"C", rows_of(C, M, ldc, 1, 0, m->rows, dtype_size(c_dtype))}};
    const Operand ins[] = {{"A", rows_of(A, M, lda, 1, 0, m->cols, dtype_size(a_dtype))}, {"the bias", dense_of(bias, (int64_t)m->rows * 4)}, HX_W4_PARTS(*m)};
    const char *one, *other;
    HX_REQUIRE(!shared_operands(outs, ins, one, other), HX_ERR_INVALID_INPUT, "hx_gemm_w4: %s and %s share memory", one, other);
    return a_dtype == HX_BF16 ? gemm_bf16(A, lda, *m, bias, C, ldc, c_dtype, M, epilogue, (cudaStream_t)stream)
                              : gemm_f32(A, lda, *m, bias, C, ldc, c_dtype, M, epilogue, (cudaStream_t)stream);
}

}  // extern "C"
