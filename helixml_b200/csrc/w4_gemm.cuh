// The product of a few rows with a 4-bit matrix.
#pragma once

#include <cooperative_groups.h>

#include <algorithm>

#include "w4.cuh"

namespace hx {
namespace w4 {

// ---------------------------------------------------------------- C = A W^T for a few rows
// A stream over the codes: HBM gives an SM about 23 bytes = 46 codes a cycle, each of which has to become a tensor-core operand.  W is the left operand (16 outputs x 16 columns), the rows of A the right one
// (8 rows a tile).  Which column a k index of the MMA stands for does not matter as long as both operands agree; the layout of the
// codes is such that lane (g, c) = (lane / 4, lane mod 4) finds in its 16 bytes of row g four words, word j holding the columns
// 32 j + 8 c .. + 7 of the block, as the four k-pairs of two MMAs.  So the MMAs of word j cover columns 32 j .. 32 j + 31 whatever
// the group size, one 16-byte load brings a lane's share of 128 columns, and the matching piece of A is 8 consecutive elements.
// Products are exact in fp32, sums fp32; a group's sum is scaled in fp32 and added to the total.  fp32 rows of A are cut into three
// bf16 parts of 8 bits that add up to them exactly, each with its own MMA.

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The eight codes of a word as four pairs of bf16, each (code - zero) / 64.  The bits of a bf16 whose exponent field is 0 or 1 read
// as an integer times 2^-133, so a code in bits 0 .. 3 or in bits 4 .. 7 of a half is a number as it stands; one fused multiply-add
// by 2^127 or 2^123 makes it code / 64 and takes the zero point off, exactly.
__device__ __forceinline__ uint32_t fma_pair(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ void eight_weights(uint32_t word, uint32_t minus_zero, uint32_t (&a)[4]) {
    constexpr uint32_t low = 0x7f007f00u, high = 0x7d007d00u;   // 2^127, 2^123
    const uint32_t next = word >> 8;
    a[0] = fma_pair(word & 0x000f000fu, low, minus_zero);
    a[1] = fma_pair(word & 0x00f000f0u, high, minus_zero);
    a[2] = fma_pair(next & 0x000f000fu, low, minus_zero);
    a[3] = fma_pair(next & 0x00f000f0u, high, minus_zero);
}
constexpr float kSumScale = 64.f;   // what the sums have to be multiplied by in the end

// fp32 rows of A go into the MMA as three bf16 parts that add up to them: the high 8 bits, the next 8, the rest.  The differences are
// exact; an infinity has no rest, a NaN a NaN.  (Below 2^-110 the last part ends above the number's last bit: bf16 goes down to 2^-133.)
template <typename TA> constexpr int kPartsOf = sizeof(TA) == 2 ? 1 : 3;
__device__ __forceinline__ void cut(float v, uint32_t (&part)[3]) {
    part[0] = __float_as_uint(v) & 0xffff0000u;
    const float rest = v == __uint_as_float(part[0]) ? 0.f : v - __uint_as_float(part[0]);
    part[1] = __float_as_uint(rest) & 0xffff0000u;
    part[2] = __float_as_uint(rest - __uint_as_float(part[1]));
}

__device__ __forceinline__ void finish(float v, int n, int row, const float *bias, void *C, int64_t ldc, int c_dtype, int epilogue) {
    if (bias) v += bias[n];
    if (epilogue == gemm::kEpiSilu) v = silu_acc(v);
    else if (epilogue == gemm::kEpiSoftplus) v = softplus_acc(v);
    if (c_dtype == HX_BF16) static_cast<__nv_bfloat16 *>(C)[row * ldc + n] = __float2bfloat16_rn(v);
    else static_cast<float *>(C)[row * ldc + n] = v;
}

// How many clusters of `share` CTAs are on the device at once; clusters that have to wait for others to end double the time
// (24 x 5001 x 8192 fp32: 40 clusters of 7, 51.7 us; of as many CTAs as leave all of them resident, 37.4).  Asked for once a kernel,
// size and device.
template <typename Kernel>
static hx_status clusters_at_once(Kernel kernel, int threads, size_t smem, int share, std::atomic<int> (&known)[64][9], int &fit) {
    int dev = 0;
    HX_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && (fit = known[dev][share].load(std::memory_order_relaxed) - 1) >= 0) return HX_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)share);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)share;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    HX_CUDA(cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg));
    if (dev < 64) known[dev][share].store(fit + 1, std::memory_order_relaxed);
    return HX_OK;
}

// ---------------------------------------------------------------- more rows, or fp32 ones
// The same products where a piece of A costs as much as the codes: more than one tile of 8 rows, or fp32 rows, which have to be cut
// (1 x 16384 x 4096 fp32: 34.6 us where every warp cuts for itself, 20.0 here).  A CTA's warps take different outputs, 16 each, walk
// the columns together and share the block of A they are at, staged in shared memory (fp32 rows already cut, once a CTA).  One barrier
// a block; codes, A and scales of the next blocks are under way.  No unit is full: 1.5 instructions a cycle of an SM's 4, the
// warp-level tensor pipe 35 to 40 % busy, 21 % of the warp slots filled; a warp waits for its own chain and for the barrier of every
// block.  16 x 16384 x 4096 bf16 17.9 us, 32 rows 25.6, 64 rows 43.1; 24 x 5001 x 8192 fp32 in groups of 32 with zero points 34.7.  Where tiles of 128 outputs are few, a cluster of CTAs shares the columns; each adds up a part of
// the outputs out of the others' shared memory, in the order of the ranks.
template <typename TA, int NT> constexpr int row_warps() { return 8; }
constexpr int kRowPitch = kBlockCols * 2 + 64;   // bytes from one staged row to the next: rows g and g + 1 fall on different banks
template <typename TA, int NT> constexpr int row_ctas() { return NT * (int)sizeof(TA) <= 16 ? 2 : 1; }   // an SM holds
template <typename TA> constexpr int row_stages() { return sizeof(TA) == 2 ? 3 : 2; }   // of A

template <typename TA, int NT, int GROUP>
__global__ void __launch_bounds__(32 * row_warps<TA, NT>(), row_ctas<TA, NT>())
gemm_w4_rows_kernel(const TA *__restrict__ A, int64_t lda, const hx_w4_matrix m, const float *__restrict__ bias, void *__restrict__ C,
                    int64_t ldc, int c_dtype, int M, int blocks, int epilogue, bool vec) {
    constexpr int kGroups = kBlockCols / GROUP, kParts = kPartsOf<TA>, kRows = 8 * NT, kSlots = 3, kStages = row_stages<TA>();
    constexpr int kStage = kParts * kRows * kRowPitch, kThreads = 32 * row_warps<TA, NT>(), kRowOuts = kThreads / 2;
    extern __shared__ __align__(16) unsigned char shared[];   // [kStages][kParts][kRows][kRowPitch], then the codes' slots
    const auto cluster = cooperative_groups::this_cluster();
    const int share = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int m0 = blockIdx.y * kRows, here = min(M - m0, kRows), tile0 = blockIdx.x / share * kRowOuts;
    const int k0 = (int)((int64_t)blocks * rank / share), k1 = (int)((int64_t)blocks * (rank + 1) / share);   // this CTA's blocks
    const int groups = m.cols / GROUP;
    const int scale_shift = m.scale_dtype == HX_BF16 ? 16 : 0;
    uint4 *slots = reinterpret_cast<uint4 *>(shared + kStages * kStage) + warp * kSlots * 64 + lane;

    const uint8_t *codes[2];   // of the next block that is asked for
    int64_t at[2];             // of the next four blocks' scales
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int n = min(tile0 + warp * 16 + half * 8 + g, m.rows - 1);   // rows past the last read the last
        codes[half] = m.codes + ((int64_t)n * blocks + k0) * kBlockBytes + c * 16;
        at[half] = (int64_t)n * groups + (int64_t)(k0 + c) * kGroups;
    }
    auto fetch_codes = [&](int k, int slot) {
        if (k < k1)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                cp_async16(slots + (slot * 2 + half) * 32, codes[half]);
                codes[half] += kBlockBytes;
            }
    };
    // scales and zero points of four blocks at a time, lane c those of block c
    uint32_t scale[2][2][kGroups], zero[2][2][kGroups];
    auto fetch_scales = [&](int k, uint32_t (&s)[2][kGroups], uint32_t (&z)[2][kGroups]) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                const int64_t i = at[half] + q;
                s[half][q] = 0;
                z[half][q] = 8;
                if (k + c < k1 && (k + c) * kGroups + q < groups) {
                    if (scale_shift) s[half][q] = static_cast<const uint16_t *>(m.scale)[i];
                    else s[half][q] = static_cast<const uint32_t *>(m.scale)[i];
                    if (m.zero) z[half][q] = m.zero[i];
                }
            }
#pragma unroll
        for (int half = 0; half < 2; ++half) at[half] += 4 * kGroups;
    };
    // A: bf16 goes straight into its stage; fp32 waits in registers for a block's time and is cut on its way
    constexpr int per = 16 / (int)sizeof(TA), across = kBlockCols / per, down = kThreads / across, kPieces = (kRows + down - 1) / down;
    const int row0 = threadIdx.x / across, col = threadIdx.x % across * per;   // a thread's pieces: this column of rows row0, row0 + down, ...
    const TA *from = A + (int64_t)(m0 + row0) * lda + (int64_t)k0 * kBlockCols + col;
    unsigned char *const to = shared + row0 * kRowPitch + col * 2;
    float4 held[sizeof(TA) == 4 ? kPieces : 1];
    auto fetch_rows = [&](int k, int stage) {
        const int rows = k < k1 && k * kBlockCols + col < m.cols ? here - row0 : 0;   // cols is a multiple of 32
        if (vec) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                if (i * down < rows) {
                    if constexpr (sizeof(TA) == 2) cp_async16(to + stage * kStage + i * down * kRowPitch, from + i * down * lda);
                    else held[i] = *reinterpret_cast<const float4 *>(from + i * down * lda);
                }
        } else {
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                if (i * down < rows) {
                    const TA *p = from + i * down * lda;
                    if constexpr (sizeof(TA) == 2) {
                        TA *t = reinterpret_cast<TA *>(to + stage * kStage + i * down * kRowPitch);
#pragma unroll
                        for (int e = 0; e < per; ++e) t[e] = p[e];
                    } else {
                        held[i] = make_float4(p[0], p[1], p[2], p[3]);
                    }
                }
        }
        from += kBlockCols;
    };
    auto cut_rows = [&](int stage) {   // what is held goes into its stage
        if constexpr (sizeof(TA) == 4) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                if (kRows % down != 0 && row0 + i * down >= kRows) break;
                const float v[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
                uint32_t u[4][3];
#pragma unroll
                for (int e = 0; e < 4; ++e) cut(v[e], u[e]);
#pragma unroll
                for (int part = 0; part < 3; ++part)
                    *reinterpret_cast<uint2 *>(to + stage * kStage + (part * kRows + i * down) * kRowPitch) =
                        make_uint2(__byte_perm(u[0][part], u[1][part], 0x7632), __byte_perm(u[2][part], u[3][part], 0x7632));
            }
        }
    };

    fetch_scales(k0, scale[0], zero[0]);
#pragma unroll
    for (int k = 0; k < kSlots - 1; ++k) {
        fetch_codes(k0 + k, k);
        if constexpr (sizeof(TA) == 2) fetch_rows(k0 + k, k);
        cp_commit();
    }
    if constexpr (sizeof(TA) == 4) {
        fetch_rows(k0, 0);
        cut_rows(0);
        fetch_rows(k0 + 1, 0);
    }
    float total[NT][4] = {};
    int slot = 0, u = 0;   // of the codes (bf16: and of A), and the block's place among four
    for (int k = k0; k < k1; ++k) {
        if (u == 0) fetch_scales(k + 4, scale[1], zero[1]);
        cp_wait<kSlots - 2>();
        __syncthreads();   // block k is staged; block k - 1 is done with
        const int next = slot == 0 ? kSlots - 1 : slot - 1;   // what block k - 1 had
        fetch_codes(k + kSlots - 1, next);
        if constexpr (sizeof(TA) == 2) fetch_rows(k + kSlots - 1, next);
        cp_commit();
        if constexpr (sizeof(TA) == 4) {
            cut_rows((k + 1 - k0) & 1);
            fetch_rows(k + 2, 0);
        }
        const uint4 w[2] = {slots[(slot * 2) * 32], slots[(slot * 2 + 1) * 32]};
        const unsigned char *stage = shared + (sizeof(TA) == 2 ? slot : (k - k0) & 1) * kStage + g * kRowPitch + c * 16;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            if (GROUP < kBlockCols && k * kGroups + q >= groups) break;   // the filled-up end of a row
            float sum[NT][4], by[2];
            uint32_t offset[2];   // -(zero point) / 64, twice
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                by[half] = __uint_as_float(__shfl_sync(0xffffffffu, scale[0][half][q], u, 4) << scale_shift);
                offset[half] = 0xbe00be00u;
                if (m.zero) offset[half] = fma_pair(__shfl_sync(0xffffffffu, zero[0][half][q], u, 4) * 0x00010001u, 0xff00ff00u, 0x80008000u);
            }
#pragma unroll
            for (int j = q * (4 / kGroups); j < (q + 1) * (4 / kGroups); ++j) {
                uint32_t a[2][4];
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    eight_weights(j == 0 ? w[half].x : j == 1 ? w[half].y : j == 2 ? w[half].z : w[half].w, offset[half], a[half]);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        const uint4 b = *reinterpret_cast<const uint4 *>(stage + (part * kRows + t * 8) * kRowPitch + j * 64);
                        if (j == q * (4 / kGroups) && part == 0) mma_bf16_first(sum[t], a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
                        else mma_bf16(sum[t], a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
                        mma_bf16(sum[t], a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
                    }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) total[t][i] = fmaf(by[i >> 1], sum[t][i], total[t][i]);
        }
        slot = slot == kSlots - 1 ? 0 : slot + 1;
        u = (u + 1) & 3;
        if (u == 0) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int q = 0; q < kGroups; ++q) scale[0][half][q] = scale[1][half][q], zero[0][half][q] = zero[1][half][q];
        }
    }
    // totals 0, 1: output g, rows 2 c and 2 c + 1 of A; 2, 3: output g + 8
    if (share == 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = tile0 + warp * 16 + (i >> 1) * 8 + g, row = t * 8 + 2 * c + (i & 1);
                if (n < m.rows && row < here) finish(kSumScale * total[t][i], n, m0 + row, bias, C, ldc, c_dtype, epilogue);
            }
        return;
    }
    float *sums = reinterpret_cast<float *>(shared);   // [kRows][kRowOuts]
    cp_wait<0>();
    __syncthreads();   // the stages have been read
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[(t * 8 + 2 * c + (i & 1)) * kRowOuts + warp * 16 + (i >> 1) * 8 + g] = total[t][i];
    cluster.sync();
    for (int i = rank * kThreads + threadIdx.x; i < here * kRowOuts; i += share * kThreads) {
        const int n = tile0 + i % kRowOuts, row = i / kRowOuts;
        if (n >= m.rows) continue;
        float v = 0.f;
        for (int r = 0; r < share; ++r) v += *cluster.map_shared_rank(sums + i, r);
        finish(kSumScale * v, n, m0 + row, bias, C, ldc, c_dtype, epilogue);
    }
    cluster.sync();   // the others' shared memory stays until it has been read
}

template <typename TA, int NT, int GROUP>
static hx_status launch_rows_as(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                                int epilogue, cudaStream_t st) {
    constexpr int kRows = 8 * NT, per_sm = row_ctas<TA, NT>(), kRowWarps = row_warps<TA, NT>(), kRowOuts = 16 * kRowWarps;
    constexpr size_t staged = (size_t)row_stages<TA>() * kPartsOf<TA> * kRows * kRowPitch, smem = staged + kRowWarps * 3 * 1024;
    static_assert(smem >= (size_t)kRows * kRowOuts * sizeof(float), "the sums of a cluster's CTA fit");
    auto kernel = gemm_w4_rows_kernel<TA, NT, GROUP>;
    static std::atomic<uint64_t> done{0};
    HX_CUDA(allow_smem((const void *)kernel, smem, done));
    const int blocks = blocks_of(m.cols), tiles = (int)(((int64_t)m.rows + kRowOuts - 1) / kRowOuts);
    const int64_t down = ((int64_t)M + kRows - 1) / kRows;
    int share = (int)std::max<int64_t>(1, std::min<int64_t>({per_sm * sm_count() / (tiles * down), blocks / 2, 8}));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(32 * kRowWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    static std::atomic<int> known[64][9];
    for (int fit = 0; share > 1; --share) {
        const hx_status s = clusters_at_once(kernel, 32 * kRowWarps, smem, share, known, fit);
        if (s != HX_OK) return s;
        if (tiles * down <= fit) break;
    }
    attr.val.clusterDim.x = (unsigned)share;
    cfg.numAttrs = share > 1 ? 1 : 0;
    const bool vec = aligned8(A, lda, sizeof(TA) == 4 ? HX_F32 : HX_BF16);
    constexpr int most = 65535 * kRows;   // rows of a launch
    for (int64_t m0 = 0; m0 < M; m0 += most) {
        const int rows = (int)std::min<int64_t>(M - m0, most);
        cfg.gridDim = dim3((unsigned)(tiles * share), (unsigned)((rows + kRows - 1) / kRows));
        HX_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<const TA *>(A) + m0 * lda, lda, m, bias,
                                   static_cast<void *>(static_cast<char *>(C) + m0 * ldc * (int64_t)dtype_size(c_dtype)), ldc, c_dtype, rows, blocks,
                                   epilogue, vec));
    }
    return check_launch("gemm_w4_rows_kernel");
}
template <typename TA, int NT>
static hx_status launch_rows(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                             int epilogue, cudaStream_t st) {
    if (m.group == 32) return launch_rows_as<TA, NT, 32>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    if (m.group == 64) return launch_rows_as<TA, NT, 64>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    return launch_rows_as<TA, NT, 128>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
}

// As many tiles of 8 rows as the rows need, up to eight: a tile that holds none costs as much as any other (in us, with the count
// rounded up to 4 or 8 instead: fp32 20 x 4096 x 4096 13.7, 16.6; 48 x 16384 x 4096 80, 102; bf16 24 x 16384 x 4096 21.7, 24.4; 40 rows
// 32.4, 42.6).
template <typename TA>
static hx_status launch_rows_for(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                                 int epilogue, cudaStream_t st) {
    switch (std::min((M - 1) / 8 + 1, 8)) {
        case 1: return launch_rows<TA, 1>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
        case 2: return launch_rows<TA, 2>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
        case 3: return launch_rows<TA, 3>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
        case 4: return launch_rows<TA, 4>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
        case 5: return launch_rows<TA, 5>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
        case 6: return launch_rows<TA, 6>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
        case 7: return launch_rows<TA, 7>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
        default: return launch_rows<TA, 8>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    }
}

}  // namespace w4
}  // namespace hx
