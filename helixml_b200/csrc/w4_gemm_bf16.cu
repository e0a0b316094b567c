// hx_gemm_w4 with bf16 rows of A: the kernel for up to eight of them, and the choice between it and the one for more.
#include "w4_gemm.cuh"

namespace hx {
namespace w4 {

// ---------------------------------------------------------------- up to eight bf16 rows
// A CTA works through tiles of 16 outputs.  A warp takes CH consecutive blocks of 128 columns at a time (a chunk); as soon as a
// block's codes have been used, the same block of the next chunk, of the next tile if need be, is asked for.  Codes come by cp.async
// into the lane's own slots and A waits in shared memory, so that no load in the loop but the next scales is waited for by
// scoreboard: loads that miss and loads that hit would share one.  The four lanes of a row need the same scales, so lane c loads
// those of block c of the chunk and the others get them by shuffle.  The warps' partial sums are added in the order of the warps.
// Where the tiles are fewer than the SMs, a cluster of CTAs shares a tile's columns and the first one adds the others' sums out of
// their shared memory.  16384 x 4096, groups of 128: one row 12.7 us out of HBM (42 % of its rate; the loads alone take 8.7), eight
// rows 15.8.  No unit is full: half of the issue slots, 18 % of the warp-level tensor pipe, 22 % of the warp slots (16 warps an SM, by
// their registers).  What a warp waits for is its own chain of convert, multiply and scale, and a stream that starts cold.
constexpr int kMostWarps = 16;   // of a CTA, by its registers

// Where a warp's partial sum of output n of the tile and row `row` of A lies: [lane][i].
__device__ __forceinline__ int place(int n, int row) { return ((n & 7) * 4 + (row >> 1)) * 4 + (n >> 3) * 2 + (row & 1); }

// Bytes from one staged row of A to the next: rows g and g + 1 fall on different banks.
__host__ __device__ constexpr size_t staged_pitch(int cols) { return ((size_t)cols * 2 + 127) / 128 * 128 + 64; }

template <int GROUP, int CH>
__global__ void __launch_bounds__(32 * kMostWarps, 1)
gemm_w4_kernel(const __nv_bfloat16 *__restrict__ A, int64_t lda, const hx_w4_matrix m, const float *__restrict__ bias,
               void *__restrict__ C, int64_t ldc, int c_dtype, int M, int blocks, int epilogue, bool vec) {
    constexpr int kGroups = kBlockCols / GROUP, kSums = 128, kOuts = 16;
    extern __shared__ __align__(16) float partial[];   // [2][warps][kSums], then the codes' slots, then A
    const auto cluster = cooperative_groups::this_cluster();
    const int share = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();   // CTAs of a tile
    const int warps = blockDim.x / 32, threads = blockDim.x;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int64_t row_bytes = (int64_t)blocks * kBlockBytes;
    const int groups = m.cols / GROUP, tiles = (m.rows + kOuts - 1) / kOuts, stride = gridDim.x / share;
    const int first = (rank * warps + warp) * CH, apart = share * warps * CH;   // first block of this warp's chunks
    const int chunks = (blocks + apart - 1) / apart;                            // of a tile, the last one not for all warps
    const bool scale_bf16 = m.scale_dtype == HX_BF16;
    const int scale_shift = scale_bf16 ? 16 : 0;
    uint4 *slots = reinterpret_cast<uint4 *>(partial + 2 * warps * kSums) + warp * CH * 64 + lane;

    unsigned char *staged = reinterpret_cast<unsigned char *>(partial + 2 * warps * kSums) + warps * CH * 1024;
    const size_t pitch = staged_pitch(m.cols);
    const int pieces = m.cols / 8;
    for (int i = threadIdx.x; i < M * pieces; i += threads) {
        const int row = i / pieces, k = i % pieces * 8;
        __nv_bfloat16 *to = reinterpret_cast<__nv_bfloat16 *>(staged + row * pitch) + k;
        const __nv_bfloat16 *from = A + row * lda + k;
        if (vec) {
            cp_async16(to, from);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) to[e] = from[e];
        }
    }
    cp_commit();
    // this lane's row of A; past the last one the last, whose sums are then not stored
    const unsigned char *mine_a = staged + min(g, M - 1) * pitch + c * 16;

    // the chunk that is asked for: its tile, its number there, where its rows of codes and scales are
    int ahead_tile = blockIdx.x / share, ahead = 0;
    const uint8_t *codes[2];
    int64_t at[2];
    auto rows_of = [&](int tile) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int n = min(tile * kOuts + half * 8 + g, m.rows - 1);   // rows past the last read the last
            codes[half] = m.codes + n * row_bytes + first * kBlockBytes + c * 16;
            at[half] = (int64_t)n * groups + (first + c) * kGroups;
        }
    };
    auto fetch_codes = [&](int u) {
        if (ahead_tile < tiles && first + ahead * apart + u < blocks)
#pragma unroll
            for (int half = 0; half < 2; ++half) cp_async16(slots + (u * 2 + half) * 32, codes[half] + u * kBlockBytes);
        cp_commit();
    };
    // Scales and zero points under way stay as they are loaded: any arithmetic on them would wait for them.
    uint32_t scale[2][2][kGroups], zero[2][2][kGroups];   // of block c of this chunk and of the next
    auto fetch_scales = [&](uint32_t (&s)[2][kGroups], uint32_t (&z)[2][kGroups]) {
        const int block = first + ahead * apart + c;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                s[half][q] = 0;
                z[half][q] = 8;
                if (ahead_tile < tiles && c < CH && block * kGroups + q < groups) {
                    if (scale_bf16) s[half][q] = static_cast<const uint16_t *>(m.scale)[at[half] + q];
                    else s[half][q] = static_cast<const uint32_t *>(m.scale)[at[half] + q];
                    if (m.zero) z[half][q] = m.zero[at[half] + q];
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
            for (int half = 0; half < 2; ++half) {
                codes[half] += (int64_t)apart * kBlockBytes;
                at[half] += (int64_t)apart * kGroups;
            }
        }
    };
    rows_of(ahead_tile);
#pragma unroll
    for (int u = 0; u < CH; ++u) fetch_codes(u);
    fetch_scales(scale[0], zero[0]);
    advance();
    cp_wait<CH>();
    __syncthreads();   // A is staged

    float total[4] = {};
    int buffer = 0;
    for (int tile = blockIdx.x / share; tile < tiles; tile += stride) {
        for (int chunk = 0; chunk < chunks; ++chunk) {
            fetch_scales(scale[1], zero[1]);
#pragma unroll
            for (int u = 0; u < CH; ++u) {
                const int block = first + chunk * apart + u;
                cp_wait<CH - 1>();   // the lane's own slots: nobody else to wait for
                if (block < blocks) {
                    const uint4 w[2] = {slots[(u * 2) * 32], slots[(u * 2 + 1) * 32]};
#pragma unroll
                    for (int q = 0; q < kGroups; ++q) {
                        if (GROUP < kBlockCols && block * kGroups + q >= groups) break;   // the filled-up end of a row
                        float sum[4], by[2];
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
                            const uint4 b = *reinterpret_cast<const uint4 *>(mine_a + (size_t)block * (kBlockCols * 2) + j * 64);
                            if (j == q * (4 / kGroups)) mma_bf16_first(sum, a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
                            else mma_bf16(sum, a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
                            mma_bf16(sum, a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
                        }
                        // sums 0, 1: output g, rows 2 c and 2 c + 1 of A; 2, 3: output g + 8
#pragma unroll
                        for (int i = 0; i < 4; ++i) total[i] = fmaf(by[i >> 1], sum[i], total[i]);
                    }
                }
                fetch_codes(u);
            }
            advance();
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int q = 0; q < kGroups; ++q) scale[0][half][q] = scale[1][half][q], zero[0][half][q] = zero[1][half][q];
        }
        // the tile's sums: every warp's into this tile's buffer, then added in the order of the warps
        *reinterpret_cast<float4 *>(partial + (buffer * warps + warp) * kSums + lane * 4) = make_float4(total[0], total[1], total[2], total[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) total[i] = 0.f;
        __syncthreads();
        for (int i = threadIdx.x; i < kOuts * M; i += threads) {
            const int n = i % kOuts, row = i / kOuts;
            if (tile * kOuts + n >= m.rows) continue;
            float *p = partial + buffer * warps * kSums + place(n, row);
            float v = 0.f;
            for (int q = 0; q < warps; ++q) v += p[q * kSums];
            if (share > 1) *p = v;   // for the cluster's first CTA
            else finish(kSumScale * v, tile * kOuts + n, row, bias, C, ldc, c_dtype, epilogue);
        }
        buffer ^= 1;
    }
    if (share > 1) {   // one tile a cluster: its sums are in buffer 0
        cluster.sync();
        if (rank == 0)
            for (int i = threadIdx.x; i < kOuts * M; i += threads) {
                const int n = i % kOuts, row = i / kOuts, out = blockIdx.x / share * kOuts + n;
                if (out >= m.rows) continue;
                float v = 0.f;
                for (int q = 0; q < share; ++q) v += *cluster.map_shared_rank(partial + place(n, row), q);
                finish(kSumScale * v, out, row, bias, C, ldc, c_dtype, epilogue);
            }
        cluster.sync();   // the others' shared memory stays until it has been read
    }
}

// How a product is laid out on the SMs.  More tiles than SMs: chunks of four blocks, and 16 warps' worth of CTAs on an SM, as many
// as the staged rows of A leave room for; of fewer warps the CTAs have less to add up per tile, of more they have less to walk
// (1 x 16384 x 4096 bf16: 13.1 us with 4 CTAs of 4, 14.1 with 2 of 8; 1 x 4096 x 4096: 7.4 and 6.9).  Otherwise one tile a CTA, or a
// cluster, with as many warps as there are blocks.
constexpr size_t kSmemBytes = 200 * 1024;   // of an SM, for the staged rows, the sums and the slots
struct Plan { int share, warps, chunk, grid; };
static hx_status plan_of(const hx_w4_matrix &m, size_t staged, Plan &p) {
    const int sms = sm_count(), blocks = blocks_of(m.cols), tiles = (int)(((int64_t)m.rows + 15) / 16), most = kMostWarps;
    p.share = std::max(1, std::min({sms / tiles, (blocks + most - 1) / most, 8}));
    static std::atomic<uint64_t> done{0};
    static std::atomic<int> known[64][9];
    for (int fit = 0; p.share > 1; --p.share) {   // with an SM for each CTA
        HX_CUDA(allow_smem((const void *)gemm_w4_kernel<128, 4>, kSmemBytes, done));
        const hx_status s = clusters_at_once(gemm_w4_kernel<128, 4>, 32 * most, kSmemBytes, p.share, known, fit);
        if (s != HX_OK) return s;
        if (tiles <= fit) break;
    }
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
    return HX_OK;
}

template <int GROUP, int CH>
static hx_status launch_few_as(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                               int epilogue, const Plan &p, size_t smem, cudaStream_t st) {
    auto kernel = gemm_w4_kernel<GROUP, CH>;
    static std::atomic<uint64_t> done{0};
    if (smem > 48 * 1024) HX_CUDA(allow_smem((const void *)kernel, kSmemBytes, done));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid);
    cfg.blockDim = dim3(32 * p.warps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.share;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.share > 1 ? 1 : 0;
    HX_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<const __nv_bfloat16 *>(A), lda, m, bias, C, ldc, c_dtype, M, blocks_of(m.cols), epilogue,
                               aligned8(A, lda, HX_BF16)));
    return check_launch("gemm_w4_kernel");
}

// Whether M rows of A fit into shared memory beside the warps' sums and slots.
static bool fits_staged(const hx_w4_matrix &m, int M) { return M * staged_pitch(m.cols) + kMostWarps * (1024 + 4096) <= kSmemBytes; }

static hx_status launch_few(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M,
                            int epilogue, cudaStream_t st) {
    const size_t staged = M * staged_pitch(m.cols);
    Plan p;
    const hx_status s = plan_of(m, staged, p);
    if (s != HX_OK) return s;
    const size_t smem = (size_t)p.warps * (1024 + p.chunk * 1024) + staged;   // sums twice, slots
#define HX_W4_GROUP(G)                                                                                            \
    do {                                                                                                          \
        if (p.chunk == 1) return launch_few_as<G, 1>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, p, smem, st); \
        if (p.chunk == 2) return launch_few_as<G, 2>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, p, smem, st); \
        return launch_few_as<G, 4>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, p, smem, st);                   \
    } while (0)
    if (m.group == 32) HX_W4_GROUP(32);
    if (m.group == 64) HX_W4_GROUP(64);
    HX_W4_GROUP(128);
#undef HX_W4_GROUP
}

hx_status gemm_bf16(const void *A, int64_t lda, const hx_w4_matrix &m, const float *bias, void *C, int64_t ldc, int c_dtype, int M, int epilogue,
                    cudaStream_t st) {
    // In us, this kernel and the one for more: 1 x 16384 x 4096 11.7, 13.5; 1 x 768 x 12288 6.7, 9.7; 4 x 2048 x 1536 4.2, 4.9; at eight rows
    // they meet: 8 x 16384 x 4096 15.0, 14.6; 8 x 4096 x 4096 8.6, 7.0; 8 x 2048 x 1536 4.3, 5.1.
    if (M <= 8 && fits_staged(m, M)) return launch_few(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
    return launch_rows_for<__nv_bfloat16>(A, lda, m, bias, C, ldc, c_dtype, M, epilogue, st);
}

}  // namespace w4
}  // namespace hx
