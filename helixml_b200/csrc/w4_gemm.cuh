// The product of a few rows with a 4-bit matrix.
#pragma once

#include <cooperative_groups.h>

#include <algorithm>

#include "w4.cuh"

namespace hx {
namespace w4 {

// ---------------------------------------------------------------- C = A W^T for a few rows
// A stream over the codes: HBM gives an SM about 23 bytes = 46 codes a cycle, each of which has to become a tensor-core operand, so
// instructions per code are what the kernel is made of.  W is the left operand (16 outputs x 16 columns), the rows of A the right one
// (8 rows a tile).  Which column a k index of the MMA stands for does not matter as long as both operands agree; the layout of the
// codes is such that lane (g, c) = (lane / 4, lane mod 4) finds in its 16 bytes of row g four words, word j holding the columns
// 32 j + 8 c .. + 7 of the block, as the four k-pairs of two MMAs.  So the MMAs of word j cover columns 32 j .. 32 j + 31 whatever
// the group size, one 16-byte load brings a lane's share of 128 columns, and the matching piece of A is 8 consecutive elements.
// Products are exact in fp32, sums fp32; a group's sum is scaled in fp32 and added to the total.  fp32 rows of A are cut into three
// bf16 parts of 8 bits that add up to them exactly, each with its own MMA.
//
// A CTA works through tiles of 16 RT outputs.  A warp takes CH consecutive blocks of 128 columns at a time (a chunk); as soon as a
// block's codes have been used, the same block of the next chunk, of the next tile if need be, is asked for.  Codes come by cp.async
// into the lane's own slots and A waits in shared memory (STAGED), so that no load in the loop but the next scales is waited for by
// scoreboard: loads that miss and loads that hit would share one.  The four lanes of a row need the same scales, so lane c loads
// those of block c of the chunk and the others get them by shuffle.  The warps' partial sums are added in the order of the warps.
// Where the tiles are fewer than the SMs, a cluster of CTAs shares a tile's columns and the first one adds the others' sums out of
// their shared memory.

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

constexpr int max_warps(int NT) { return NT == 1 ? 16 : 8; }   // of a CTA, by its registers

// Eight consecutive elements of a row of A as MMA operands: one part (bf16) or three that add up to them (fp32).
template <typename TA> struct Operand;
template <> struct Operand<__nv_bfloat16> {
    static constexpr int kParts = 1;
    uint32_t r[1][4];
    template <bool VEC> __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
        if constexpr (VEC) {
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
    template <bool VEC> __device__ __forceinline__ void load(const float *p) {
        float v[8];
        load8(p, VEC, v);
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = __float_as_uint(take(v[2 * i])), b = __float_as_uint(take(v[2 * i + 1]));
                r[part][i] = __byte_perm(a, b, 0x7632);
            }
    }
};

__device__ __forceinline__ void finish(float v, int n, int row, const float *bias, void *C, int64_t ldc, int c_dtype, int epilogue) {
    if (bias) v += bias[n];
    if (epilogue == gemm::kEpiSilu) v = silu_acc(v);
    else if (epilogue == gemm::kEpiSoftplus) v = softplus_acc(v);
    if (c_dtype == HX_BF16) static_cast<__nv_bfloat16 *>(C)[row * ldc + n] = __float2bfloat16_rn(v);
    else static_cast<float *>(C)[row * ldc + n] = v;
}

// Where a warp's partial sum of output n of the tile and row `row` of A lies: [RT][NT][lane][i].
template <int NT> __device__ __forceinline__ int place(int n, int row) {
    return (((n >> 4) * NT + (row >> 3)) * 32 + (n & 7) * 4 + ((row & 7) >> 1)) * 4 + ((n >> 3) & 1) * 2 + (row & 1);
}

// Bytes from one staged row of A to the next: rows g and g + 1 fall on different banks.
template <typename TA> __host__ __device__ constexpr size_t staged_pitch(int cols) {
    return ((size_t)cols * sizeof(TA) + 127) / 128 * 128 + (sizeof(TA) == 2 ? 64 : 16);
}

enum Rows { kStaged, kDirect, kDirectAny };   // A from shared memory; from global memory in 16-byte loads; at any alignment

// NT tiles of 8 rows of A, RT of 16 outputs, CH blocks of a chunk.
template <typename TA, int NT, int RT, int GROUP, int CH, int ROWS>
__global__ void __launch_bounds__(32 * max_warps(NT), 1)
gemm_w4_kernel(const TA *__restrict__ A, int64_t lda, const hx_w4_matrix m, const float *__restrict__ bias, void *__restrict__ C,
               int64_t ldc, int c_dtype, int M, int blocks, int epilogue, bool vec) {
    constexpr int kGroups = kBlockCols / GROUP, kParts = Operand<TA>::kParts, kSums = RT * NT * 128, kOuts = 16 * RT;
    extern __shared__ __align__(16) float partial[];   // [2][warps][kSums], then the codes' slots, then A
    const auto cluster = cooperative_groups::this_cluster();
    const int share = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();   // CTAs of a tile
    const int warps = blockDim.x / 32, threads = blockDim.x;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int m0 = blockIdx.y * 8 * NT, here = min(M - m0, 8 * NT);                 // rows of A
    const int64_t row_bytes = (int64_t)blocks * kBlockBytes;
    const int groups = m.cols / GROUP, tiles = (m.rows + kOuts - 1) / kOuts, stride = gridDim.x / share;
    const int first = (rank * warps + warp) * CH, apart = share * warps * CH;   // first block of this warp's chunks
    const int chunks = (blocks + apart - 1) / apart;                            // of a tile, the last one not for all warps
    const bool scale_bf16 = m.scale_dtype == HX_BF16;
    const int scale_shift = scale_bf16 ? 16 : 0;
    uint4 *slots = reinterpret_cast<uint4 *>(partial + 2 * warps * kSums) + warp * CH * RT * 64 + lane;

    if constexpr (ROWS == kStaged) {
        unsigned char *staged = reinterpret_cast<unsigned char *>(partial + 2 * warps * kSums) + warps * CH * RT * 1024;
        const size_t pitch = staged_pitch<TA>(m.cols);
        constexpr int per = 16 / (int)sizeof(TA);
        const int pieces = m.cols / per;
        for (int i = threadIdx.x; i < here * pieces; i += threads) {
            const int row = i / pieces, k = i % pieces * per;
            TA *to = reinterpret_cast<TA *>(staged + row * pitch) + k;
            const TA *from = A + (int64_t)(m0 + row) * lda + k;
            if (vec) {
                cp_async16(to, from);
            } else {
#pragma unroll
                for (int e = 0; e < per; ++e) to[e] = from[e];
            }
        }
        cp_commit();
    }
    const TA *rows[NT];   // this lane's rows of A; past the last one the last, whose sums are then not stored
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = min(t * 8 + g, here - 1);
        if constexpr (ROWS == kStaged)
            rows[t] = reinterpret_cast<const TA *>(reinterpret_cast<unsigned char *>(partial + 2 * warps * kSums) + warps * CH * RT * 1024 +
                                                   row * staged_pitch<TA>(m.cols)) + 8 * c;
        else rows[t] = A + (int64_t)(m0 + row) * lda + 8 * c;
    }

    // the chunk that is asked for: its tile, its number there, where its rows of codes and scales are
    int ahead_tile = blockIdx.x / share, ahead = 0;
    const uint8_t *codes[RT][2];
    int64_t at[RT][2];
    auto rows_of = [&](int tile) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int n = min(tile * kOuts + r * 16 + half * 8 + g, m.rows - 1);   // rows past the last read the last
                codes[r][half] = m.codes + n * row_bytes + first * kBlockBytes + c * 16;
                at[r][half] = (int64_t)n * groups + (first + c) * kGroups;
            }
    };
    auto fetch_codes = [&](int u) {
        if (ahead_tile < tiles && first + ahead * apart + u < blocks)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int half = 0; half < 2; ++half) cp_async16(slots + ((u * RT + r) * 2 + half) * 32, codes[r][half] + u * kBlockBytes);
        cp_commit();
    };
    // Scales and zero points under way stay as they are loaded: any arithmetic on them would wait for them.
    uint32_t scale[2][RT][2][kGroups], zero[2][RT][2][kGroups];   // of block c of this chunk and of the next
    auto fetch_scales = [&](uint32_t (&s)[RT][2][kGroups], uint32_t (&z)[RT][2][kGroups]) {
        const int block = first + ahead * apart + c;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int q = 0; q < kGroups; ++q) {
                    s[r][half][q] = 0;
                    z[r][half][q] = 8;
                    if (ahead_tile < tiles && c < CH && block * kGroups + q < groups) {
                        if (scale_bf16) s[r][half][q] = static_cast<const uint16_t *>(m.scale)[at[r][half] + q];
                        else s[r][half][q] = static_cast<const uint32_t *>(m.scale)[at[r][half] + q];
                        if (m.zero) z[r][half][q] = m.zero[at[r][half] + q];
                    }
                }
    };
    auto advance = [&]() {
        if (++ahead == chunks) {
            ahead = 0;
            ahead_tile += stride;
            rows_of(ahead_tile);
        } else {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    codes[r][half] += (int64_t)apart * kBlockBytes;
                    at[r][half] += (int64_t)apart * kGroups;
                }
        }
    };
    rows_of(ahead_tile);
#pragma unroll
    for (int u = 0; u < CH; ++u) fetch_codes(u);
    fetch_scales(scale[0], zero[0]);
    advance();
    if constexpr (ROWS == kStaged) {
        cp_wait<CH>();
        __syncthreads();
    }

    float total[RT][NT][4] = {};
    int buffer = 0;
    for (int tile = blockIdx.x / share; tile < tiles; tile += stride) {
        for (int chunk = 0; chunk < chunks; ++chunk) {
            fetch_scales(scale[1], zero[1]);
#pragma unroll
            for (int u = 0; u < CH; ++u) {
                const int block = first + chunk * apart + u;
                cp_wait<CH - 1>();   // the lane's own slots: nobody else to wait for
                if (block < blocks) {
                    uint4 w[RT][2];
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int half = 0; half < 2; ++half) w[r][half] = slots[((u * RT + r) * 2 + half) * 32];
#pragma unroll
                    for (int q = 0; q < kGroups; ++q) {
                        if (GROUP < kBlockCols && block * kGroups + q >= groups) break;   // the filled-up end of a row
                        float sum[RT][NT][4], by[RT][2];
                        uint32_t offset[RT][2];   // -(zero point) / 64, twice
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                by[r][half] = __uint_as_float(__shfl_sync(0xffffffffu, scale[0][r][half][q], u, 4) << scale_shift);
                                offset[r][half] = 0xbe00be00u;
                                if (m.zero) offset[r][half] = fma_pair(__shfl_sync(0xffffffffu, zero[0][r][half][q], u, 4) * 0x00010001u, 0xff00ff00u, 0x80008000u);
                            }
#pragma unroll
                        for (int j = q * (4 / kGroups); j < (q + 1) * (4 / kGroups); ++j) {
                            uint32_t a[RT][2][4];
#pragma unroll
                            for (int r = 0; r < RT; ++r)
#pragma unroll
                                for (int half = 0; half < 2; ++half)
                                    eight_weights(j == 0 ? w[r][half].x : j == 1 ? w[r][half].y : j == 2 ? w[r][half].z : w[r][half].w, offset[r][half], a[r][half]);
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                Operand<TA> b;
                                b.template load<ROWS != kDirectAny>(rows[t] + block * kBlockCols + j * 32);
#pragma unroll
                                for (int part = 0; part < kParts; ++part)
#pragma unroll
                                    for (int r = 0; r < RT; ++r) {
                                        if (j == q * (4 / kGroups) && part == 0) mma_bf16_first(sum[r][t], a[r][0][0], a[r][1][0], a[r][0][1], a[r][1][1], b.r[part][0], b.r[part][1]);
                                        else mma_bf16(sum[r][t], a[r][0][0], a[r][1][0], a[r][0][1], a[r][1][1], b.r[part][0], b.r[part][1]);
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
                                for (int i = 0; i < 4; ++i) total[r][t][i] = fmaf(by[r][i >> 1], sum[r][t][i], total[r][t][i]);
                    }
                }
                fetch_codes(u);
            }
            advance();
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int q = 0; q < kGroups; ++q) scale[0][r][half][q] = scale[1][r][half][q], zero[0][r][half][q] = zero[1][r][half][q];
        }
        // the tile's sums: every warp's into this tile's buffer, then added in the order of the warps
        float *mine = partial + (buffer * warps + warp) * kSums + lane * 4;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                *reinterpret_cast<float4 *>(mine + (r * NT + t) * 128) = make_float4(total[r][t][0], total[r][t][1], total[r][t][2], total[r][t][3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) total[r][t][i] = 0.f;
            }
        __syncthreads();
        for (int i = threadIdx.x; i < kOuts * here; i += threads) {
            const int n = i % kOuts, row = i / kOuts;
            if (tile * kOuts + n >= m.rows) continue;
            float *p = partial + buffer * warps * kSums + place<NT>(n, row);
            float v = 0.f;
            for (int q = 0; q < warps; ++q) v += p[q * kSums];
            if (share > 1) *p = v;   // for the cluster's first CTA
            else finish(kSumScale * v, tile * kOuts + n, m0 + row, bias, C, ldc, c_dtype, epilogue);
        }
        buffer ^= 1;
    }
    if (share > 1) {   // one tile a cluster: its sums are in buffer 0
        cluster.sync();
        if (rank == 0)
            for (int i = threadIdx.x; i < kOuts * here; i += threads) {
                const int n = i % kOuts, row = i / kOuts, out = blockIdx.x / share * kOuts + n;
                if (out >= m.rows) continue;
                float v = 0.f;
                for (int q = 0; q < share; ++q) v += *cluster.map_shared_rank(partial + place<NT>(n, row), q);
                finish(kSumScale * v, out, m0 + row, bias, C, ldc, c_dtype, epilogue);
            }
        cluster.sync();   // the others' shared memory stays until it has been read
    }
}

// How a product is laid out on the SMs.  More tiles than SMs: chunks of four blocks, and 16 warps' worth of CTAs on an SM, as many
// as the staged rows of A leave room for; of fewer warps the CTAs have less to add up per tile, of more they have less to walk
// (1 x 16384 x 4096 bf16: 13.1 us with 4 CTAs of 4, 14.1 with 2 of 8; 1 x 4096 x 4096: 7.4 and 6.9).  Otherwise one tile a CTA, or a
// cluster, with as many warps as there are blocks.
constexpr size_t kSmemBytes = 200 * 1024;   // of an SM, for the staged rows and the slots
struct Plan { int share, warps, chunk, grid; };
static Plan plan_of(const hx_w4_matrix &m, int outs, int most, size_t staged) {
    const int sms = sm_count(), blocks = blocks_of(m.cols), tiles = (int)(((int64_t)m.rows + outs - 1) / outs);
    Plan p;
    p.share = std::max(1, std::min({sms / tiles, (blocks + most - 1) / most, 8}));
    const int part = (blocks + p.share - 1) / p.share;   // blocks of a CTA
    if (tiles > sms) {
        int ctas = tiles >= 3 * sms ? 4 : 2;
        while (ctas > 1 && ctas * (staged + 24 * 1024) > kSmemBytes) ctas /= 2;
        p.chunk = part >= 4 ? 4 : part >= 2 ? 2 : 1;
        p.warps = std::max(1, std::min(most / ctas, (part + p.chunk - 1) / p.chunk));
        p.grid = std::min(tiles, std::max(ctas, most / p.warps) * sms);
    } else {
        p.chunk = part <= most ? 1 : part <= 2 * most ? 2 : 4;
        p.warps = std::min(most, (part + p.chunk - 1) / p.chunk);
        p.grid = tiles * p.share;
    }
    return p;
}

template <typename TA, int NT, int RT, int GROUP, int CH, int ROWS>
static hx_status launch_as(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                           int epilogue, const Plan &p, size_t smem, bool vec, cudaStream_t st) {
    auto kernel = gemm_w4_kernel<TA, NT, RT, GROUP, CH, ROWS>;
    static std::atomic<uint64_t> done{0};
    if (smem > 48 * 1024) HX_CUDA(allow_smem((const void *)kernel, kSmemBytes + 16 * 1024, done));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(32 * p.warps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.share;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.share > 1 ? 1 : 0;
    constexpr int most = 65535 * 8 * NT;   // rows of a launch
    for (int64_t m0 = 0; m0 < M; m0 += most) {
        const int rows = (int)std::min<int64_t>(M - m0, most);
        cfg.gridDim = dim3((unsigned)p.grid, (unsigned)((rows + 8 * NT - 1) / (8 * NT)));
        HX_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<const TA *>(A) + m0 * lda, lda, m, bias,
                                   static_cast<void *>(static_cast<char *>(C) + m0 * ldc * (int64_t)dtype_size(c_dtype)), ldc, c_dtype, rows,
                                   blocks_of(m.cols), epilogue, vec));
    }
    return check_launch("gemm_w4_kernel");
}
template <typename TA, int NT, int RT>
static hx_status launch_gemm(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                             int epilogue, cudaStream_t st) {
    const bool vec = aligned8(A, lda, sizeof(TA) == 4 ? HX_F32 : HX_BF16);
    size_t staged = (size_t)std::min(M, 8 * NT) * staged_pitch<TA>(m.cols);
    const bool stage = staged + (size_t)max_warps(NT) * RT * (NT * 1024 + (RT > 1 ? 2048 : 4096)) <= kSmemBytes;
    if (!stage) staged = 0;
    Plan p = plan_of(m, 16 * RT, max_warps(NT), staged);
    if (RT > 1 || !stage) p.chunk = 2;   // instances there are; the walk covers any number of blocks
    else if (NT > 1 && p.chunk == 1) p.chunk = 2;
    const size_t smem = (size_t)p.warps * RT * (NT * 1024 + p.chunk * 1024) + staged;   // sums twice, slots
#define HX_W4_AS(G, CH, ROWS) return launch_as<TA, NT, RT, G, CH, ROWS>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, p, smem, vec, st)
#define HX_W4_GROUP(G)                                                \
    do {                                                              \
        if (!stage && vec) HX_W4_AS(G, 2, kDirect);                   \
        if (!stage) HX_W4_AS(G, 2, kDirectAny);                       \
        if constexpr (RT == 1) {                                      \
            if constexpr (NT == 1) {                                  \
                if (p.chunk == 1) HX_W4_AS(G, 1, kStaged);            \
            }                                                         \
            if (p.chunk == 4) HX_W4_AS(G, 4, kStaged);                \
        }                                                             \
        HX_W4_AS(G, 2, kStaged);                                      \
    } while (0)
    if (m.group == 32) HX_W4_GROUP(32);
    if (m.group == 64) HX_W4_GROUP(64);
    HX_W4_GROUP(128);
#undef HX_W4_GROUP
#undef HX_W4_AS
}

// ---------------------------------------------------------------- more than eight rows
// The same products where a piece of A is read for more than one tile of rows: here it costs as much as the codes, so a CTA's warps take
// different outputs, 16 each, walk the columns together and share the block of A they are at, staged in shared memory (fp32 rows
// already cut into their three parts, once a CTA).  One barrier a block; codes, A and scales of the next blocks are under way.  What
// bounds it is the warp-level tensor pipe and the instructions that feed it.  Where tiles of 128 outputs are few, a cluster of CTAs
// shares the columns; each adds up a part of the outputs out of the others' shared memory, in the order of the ranks.
constexpr int kRowWarps = 8, kRowOuts = 16 * kRowWarps;
constexpr int kRowPitch = kBlockCols * 2 + 64;   // bytes from one staged row to the next: rows g and g + 1 fall on different banks
template <typename TA> constexpr int row_stages() { return sizeof(TA) == 2 ? 3 : 2; }   // of A

template <typename TA, int NT, int GROUP>
__global__ void __launch_bounds__(32 * kRowWarps, NT * (int)sizeof(TA) <= 16 ? 2 : 1)
gemm_w4_rows_kernel(const TA *__restrict__ A, int64_t lda, const hx_w4_matrix m, const float *__restrict__ bias, void *__restrict__ C,
                    int64_t ldc, int c_dtype, int M, int blocks, int epilogue, bool vec) {
    constexpr int kGroups = kBlockCols / GROUP, kParts = Operand<TA>::kParts, kRows = 8 * NT, kSlots = 3, kStages = row_stages<TA>();
    constexpr int kStage = kParts * kRows * kRowPitch, kThreads = 32 * kRowWarps;
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
    constexpr int per = 16 / (int)sizeof(TA), across = kBlockCols / per, kPieces = kRows * across / kThreads, down = kThreads / across;
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
                float v[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
#pragma unroll
                for (int part = 0; part < 3; ++part) {
                    uint32_t u[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(Operand<float>::take(v[e]));
                    *reinterpret_cast<uint2 *>(to + stage * kStage + (part * kRows + i * down) * kRowPitch) =
                        make_uint2(__byte_perm(u[0], u[1], 0x7632), __byte_perm(u[2], u[3], 0x7632));
                }
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
    constexpr int kRows = 8 * NT, per_sm = NT * (int)sizeof(TA) <= 16 ? 2 : 1;
    constexpr size_t staged = (size_t)row_stages<TA>() * Operand<TA>::kParts * kRows * kRowPitch, smem = staged + kRowWarps * 3 * 1024;
    static_assert(staged + kRowWarps * 3 * 1024 >= (size_t)kRows * kRowOuts * sizeof(float), "the sums of a cluster's CTA fit");
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
    // Clusters that are not all resident at once take twice the time: how many fit is asked for once a kernel, size and device.
    static std::atomic<int> resident[64][9];
    int dev = 0;
    HX_CUDA(cudaGetDevice(&dev));
    for (; share > 1; --share) {
        std::atomic<int> *known = dev < 64 ? &resident[dev][share] : nullptr;
        int fit = known ? known->load(std::memory_order_relaxed) : 0;
        if (fit == 0) {
            attr.val.clusterDim.x = (unsigned)share;
            cfg.numAttrs = 1;
            cfg.gridDim = dim3((unsigned)share);
            HX_CUDA(cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg));
            fit = std::max(fit, 1);
            if (known) known->store(fit, std::memory_order_relaxed);
        }
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

}  // namespace w4
}  // namespace hx
