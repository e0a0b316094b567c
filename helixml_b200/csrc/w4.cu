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

// ---------------------------------------------------------------- C = A W^T for a few rows
// A stream over the codes: HBM gives an SM about 23 bytes = 46 codes a cycle, each of which has to become a tensor-core operand, so
// instructions per code are what the kernel is made of.  W is the left operand (16 outputs x 16 columns), the rows of A the right one
// (8 rows a tile).  Which column a k index of the MMA stands for does not matter as long as both operands agree; the layout of the
// codes is such that lane (g, c) = (lane / 4, lane mod 4) finds in its 16 bytes of row g four words, word j holding the columns
// 32 j + 8 c .. + 7 of the block, as the four k-pairs of two MMAs.  So the MMAs of word j cover columns 32 j .. 32 j + 31 whatever
// the group size, one LDG.128 brings a lane's share of 128 columns, and the matching piece of A is 16 consecutive bytes.
// A pair of codes becomes two bf16 numbers with (w >> 4 p & 0x000f000f) | 0x43004300, which is 128 + code exactly, minus 128 + zero,
// also exact.  Products are exact in fp32, sums fp32; a group's sum is scaled in fp32 and added to the total.  fp32 rows of A are cut
// into three bf16 parts of 8 bits that add up to them exactly, each with its own MMA.
// A CTA owns 16 RT outputs; its warps take the blocks of 128 columns in turn, kAhead of them under way, and their partial sums are
// added in the order of the warps.
constexpr int kWarps = 8, kAhead = 4;

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_codes(const uint8_t *p) {   // read once
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// codes 2 p and 2 p + 1 of a word, less the zero point: two bf16
__device__ __forceinline__ uint32_t two_weights(uint32_t word, int p, __nv_bfloat162 bias) {
    const uint32_t u = ((word >> (4 * p)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&u), bias);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Eight consecutive elements of a row of A as MMA operands: one part (bf16) or three that add up to them (fp32).
template <typename TA> struct Operand;
template <> struct Operand<__nv_bfloat16> {
    static constexpr int kParts = 1;
    uint32_t r[1][4];
    __device__ __forceinline__ void load(const __nv_bfloat16 *p, bool vec) {
        if (vec) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            r[0][0] = v.x, r[0][1] = v.y, r[0][2] = v.z, r[0][3] = v.w;
        } else {
            const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) r[0][i] = (uint32_t)u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
        }
    }
};
template <> struct Operand<float> {
    static constexpr int kParts = 3;
    uint32_t r[3][4];
    // v = high 8 bits + rest; the rest is exact, and zero for an infinity
    static __device__ __forceinline__ float take(float &v) {
        const float high = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
        v = v == high ? 0.f : v - high;
        return high;
    }
    __device__ __forceinline__ void load(const float *p, bool vec) {
        float v[8];
        load8(p, vec, v);
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = __float_as_uint(take(v[2 * i])), b = __float_as_uint(take(v[2 * i + 1]));
                r[part][i] = __byte_perm(a, b, 0x7632);
            }
    }
};

template <typename TA, int NT, int RT, int GROUP>
__global__ void __launch_bounds__(32 * kWarps)
gemm_w4_kernel(const TA *__restrict__ A, int64_t lda, const hx_w4_matrix m, const float *__restrict__ bias, void *__restrict__ C,
               int64_t ldc, int c_dtype, int M, int blocks, int epilogue, bool vec) {
    constexpr int kGroups = kBlockCols / GROUP, kParts = Operand<TA>::kParts;
    __shared__ float partial[kWarps][RT][NT][32][4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.x * 16 * RT, m0 = blockIdx.y * 8 * NT;
    const int64_t row_bytes = (int64_t)blocks * kBlockBytes;
    const int groups = m.cols / GROUP;

    // this lane's rows of W: 2 r + half; those past the last one read the last
    const uint8_t *codes[RT][2];
    int64_t scale_row[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int n = min(n0 + r * 16 + half * 8 + g, m.rows - 1);
            codes[r][half] = m.codes + n * row_bytes + c * 16;
            scale_row[r][half] = (int64_t)n * groups;
        }
    const TA *rows[NT];
    bool there[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        there[t] = m0 + t * 8 + g < M;
        rows[t] = A + (int64_t)(there[t] ? m0 + t * 8 + g : 0) * lda + 8 * c;
    }
    uint4 w[kAhead][RT][2];
    float s[kAhead][RT][2][kGroups];
    uint32_t z[kAhead][RT][2];   // zero points, a byte a group
    auto fetch = [&](int slot, int block) {
        if (block >= blocks) return;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                w[slot][r][half] = load_codes(codes[r][half] + (int64_t)block * kBlockBytes);
                z[slot][r][half] = 0x08080808u;
#pragma unroll
                for (int q = 0; q < kGroups; ++q) {
                    const int group = min(block * kGroups + q, groups - 1);
                    s[slot][r][half][q] = load_scale(m.scale, m.scale_dtype, scale_row[r][half] + group);
                    if (m.zero) z[slot][r][half] = q ? z[slot][r][half] | (uint32_t)m.zero[scale_row[r][half] + group] << (8 * q) : m.zero[scale_row[r][half] + group];
                }
            }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) fetch(u, warp + u * kWarps);

    float total[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[r][t][i] = 0.f;

    for (int base = warp; base < blocks; base += kAhead * kWarps) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int block = base + u * kWarps;
            if (block >= blocks) break;
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                float sum[RT][NT][4] = {};
#pragma unroll
                for (int j = q * (4 / kGroups); j < (q + 1) * (4 / kGroups); ++j) {
                    const int k = block * kBlockCols + j * 32;
                    uint32_t a[RT][2][4];
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint4 v = w[u][r][half];
                            const uint32_t word = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
                            const __nv_bfloat162 zero = __bfloat162bfloat162(__float2bfloat16_rn(128.f + (float)((z[u][r][half] >> (8 * q)) & 255)));
#pragma unroll
                            for (int p = 0; p < 4; ++p) a[r][half][p] = two_weights(word, p, zero);
                        }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        Operand<TA> b;
                        if (there[t] && k < m.cols) {
                            b.load(rows[t] + k, vec);
                        } else {
#pragma unroll
                            for (int part = 0; part < kParts; ++part)
#pragma unroll
                                for (int i = 0; i < 4; ++i) b.r[part][i] = 0;
                        }
#pragma unroll
                        for (int part = 0; part < kParts; ++part)
#pragma unroll
                            for (int r = 0; r < RT; ++r) {
                                mma_bf16(sum[r][t], a[r][0][0], a[r][1][0], a[r][0][1], a[r][1][1], b.r[part][0], b.r[part][1]);
                                mma_bf16(sum[r][t], a[r][0][2], a[r][1][2], a[r][0][3], a[r][1][3], b.r[part][2], b.r[part][3]);
                            }
                    }
                }
                // sums 0, 1: output g, rows 2 c and 2 c + 1 of A; 2, 3: output g + 8
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (GROUP == kBlockCols || (block * kBlockCols + q * GROUP < m.cols)) total[r][t][i] = fmaf(s[u][r][i >> 1][q], sum[r][t][i], total[r][t][i]);
            }
            fetch(u, block + kAhead * kWarps);
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t)
            *reinterpret_cast<float4 *>(partial[warp][r][t][lane]) = make_float4(total[r][t][0], total[r][t][1], total[r][t][2], total[r][t][3]);
    __syncthreads();
    for (int i = threadIdx.x; i < RT * NT * 128; i += 32 * kWarps) {
        const float *p = &partial[0][0][0][0][0] + i;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) v += p[q * RT * NT * 128];
        const int ln = (i >> 2) & 31, r = i / (NT * 128), t = i / 128 % NT;
        const int n = n0 + r * 16 + ((i >> 1) & 1) * 8 + (ln >> 2), row = m0 + t * 8 + 2 * (ln & 3) + (i & 1);
        if (n >= m.rows || row >= M) continue;
        if (bias) v += bias[n];
        if (epilogue == gemm::kEpiSilu) v = silu_acc(v);
        else if (epilogue == gemm::kEpiSoftplus) v = softplus_acc(v);
        if (c_dtype == HX_BF16) static_cast<__nv_bfloat16 *>(C)[row * ldc + n] = __float2bfloat16_rn(v);
        else static_cast<float *>(C)[row * ldc + n] = v;
    }
}

template <typename TA, int NT, int RT>
static hx_status launch_gemm(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                             int epilogue, bool vec, cudaStream_t st) {
    const int blocks = (m.cols + kBlockCols - 1) / kBlockCols;
    const int64_t down = ((int64_t)M + 8 * NT - 1) / (8 * NT);
    HX_REQUIRE(down <= 65535, HX_ERR_INVALID_DIMENSION, "hx_gemm_w4: %d rows", M);
    const dim3 grid((unsigned)(((int64_t)m.rows + 16 * RT - 1) / (16 * RT)), (unsigned)down);
    auto a = static_cast<const TA *>(A);
    if (m.group == 32) gemm_w4_kernel<TA, NT, RT, 32><<<grid, 32 * kWarps, 0, st>>>(a, lda, m, bias, C, ldc, c_dtype, M, blocks, epilogue, vec);
    else if (m.group == 64) gemm_w4_kernel<TA, NT, RT, 64><<<grid, 32 * kWarps, 0, st>>>(a, lda, m, bias, C, ldc, c_dtype, M, blocks, epilogue, vec);
    else gemm_w4_kernel<TA, NT, RT, 128><<<grid, 32 * kWarps, 0, st>>>(a, lda, m, bias, C, ldc, c_dtype, M, blocks, epilogue, vec);
    return check_launch("gemm_w4_kernel");
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
    const bool vec = aligned8(A, lda, a_dtype);
    auto st = (cudaStream_t)stream;
#define HX_W4_ROWS(TA)                                                                                          \
    do {                                                                                                        \
        if (M <= 8) return launch_gemm<TA, 1, 1>(A, lda, *m, bias, C, ldc, c_dtype, M, epilogue, vec, st);      \
        if (M <= 16) return launch_gemm<TA, 2, 1>(A, lda, *m, bias, C, ldc, c_dtype, M, epilogue, vec, st);     \
        if (M <= 32) return launch_gemm<TA, 4, 1>(A, lda, *m, bias, C, ldc, c_dtype, M, epilogue, vec, st);     \
        return launch_gemm<TA, 8, 1>(A, lda, *m, bias, C, ldc, c_dtype, M, epilogue, vec, st);                  \
    } while (0)
    if (a_dtype == HX_BF16) HX_W4_ROWS(__nv_bfloat16);
    HX_W4_ROWS(float);
#undef HX_W4_ROWS
}

}  // extern "C"
