// Gated linear recurrence h_t = a_t h_{t-1} + b_t over [batch, seq_len, d_inner], its gradients, and its single-token step.
//
// The work per point is a handful of instructions, so both directions are bound by HBM: x and g read and h written once, or x, g
// and dh read and dx and dg written once.  A warp owns 64 neighbouring channels of one batch row (two a lane) and walks the steps;
// its rows arrive through a ring of cp.async fetches in its own part of shared memory, so warps never wait for one another.
// Where the chains alone are too few warps to keep HBM busy, the sequence is cut into segments: run t..t' composes to the affine map
// h -> A h + B (A the product of its decays, B its result from zero), a first launch writes the map of every segment but the last,
// and the second folds the maps before its segment onto h0 and walks the segment with outputs.  That reads x and g twice, the second
// time from L2 as far as they fit: the first launch walks every segment from its end (a map can be built from either side), so what
// it read last is what the second needs first.  The order of a channel's sums is a function of the shape and of its own numbers.
// The backward pass is the same recurrence from the end, e_t = a_t (dh_t + e_{t+1}); h_{t-1} is recomputed from the state that the
// forward pass saved every 16 steps, so h itself, rounded to the io type, is not needed.
//
// Folding maps is not the recurrence where numbers leave the format.  A state that overflows in the middle of a segment stays infinite
// when its steps are walked, but a map knows the ends of a segment only, and what overflowed may have decayed by then; a product of
// decays that underflows has lost what a large state, or growth before it, would have made of it.  So the first launch also bounds how
// far a state can get within a segment and what its products have lost, marks a map that cannot stand for the walk (A is NaN), and the
// segment is walked instead, for the channels that meet such a map or a state that the map is not made for (Reach, odd).
#include <algorithm>
#include <initializer_list>

#include "hx_common.cuh"
#include "hx_overlap.h"
#include "hx_tma.cuh"

namespace hx {
namespace gated {

constexpr int kC = 64;                    // channels of a warp, two a lane
constexpr int kRun = 8;                   // steps of a forward fetch
constexpr int kBlock = HX_GATED_SCAN_STATE_STEPS;   // steps of a backward fetch: from one saved state to the next
// Warps of a CTA, each on its own.  Small CTAs spread evenly over the SMs: backward 5 x 1003 x 1001 fp32 36.9 us with two, 42.3 with
// four, 49.5 with one, whose CTAs cost more to start.
constexpr int kWarps = 2;
constexpr int kStages = 6, kBlockStages = 3;        // fetches a ring of runs, of blocks holds: all but one are under way
// CTAs an SM is to hold by its registers (128 and 168 a thread).  By its shared memory it holds 9 and 6 of bf16 rows; of fp32 rows, whose
// rings take 48 and 72 KiB, 4 and 3, so that more registers would be free there.
constexpr int kOccupancy = 8, kBlockOccupancy = 6;
static_assert(kBlock == 2 * kRun, "segments are multiples of both");

template <int BYTES> __device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int bytes) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One tensor's way into a warp's ring: pieces of ROWS rows of kC channels, from row `t` of src on.  `cols` channels exist, those
// behind them are zeros.  PIECE: what every address is a multiple of, in bytes.
template <int ROWS, int PIECE, typename T> struct Feed {
    static constexpr int per = PIECE / (int)sizeof(T), across = kC / per;   // elements of a piece, pieces of a row
    static constexpr int wide = across < 32 ? across : 32, high = 32 / wide;    // one instruction of the warp: high rows x wide pieces
    static constexpr int turns = across / wide;
    const T *from;        // this lane's first piece of the next fetch
    int64_t row_stride, advance;
    int cols, bytes[turns];
    uint32_t offset;      // of that piece in a slot
    __device__ __forceinline__ Feed(const T *src, int64_t t, int64_t rs, int steps, int cols_, int lane) {
        const int r0 = lane / wide, col = lane % wide * per;
        row_stride = rs;
        advance = steps * rs;
        cols = cols_;
        from = src + t * rs + r0 * rs + col;
        offset = (uint32_t)(r0 * kC + col) * (uint32_t)sizeof(T);
#pragma unroll
        for (int q = 0; q < turns; ++q) bytes[q] = min(max(cols - col - q * wide * per, 0), per) * (int)sizeof(T);
    }
    // all ROWS rows exist
    __device__ __forceinline__ void whole(uint32_t slot) {
        const T *f = from;
        from += advance;
#pragma unroll
        for (int r = 0; r < ROWS; r += high) {
#pragma unroll
            for (int q = 0; q < turns; ++q)
                cp_async<PIECE>(slot + offset + (r * kC + q * wide * per) * (int)sizeof(T), f + q * wide * per, bytes[q]);
            f += high * row_stride;
        }
    }
    // `rows` of them do
    __device__ __forceinline__ void part(uint32_t slot, int rows) {
        const T *f = from;
        from += advance;
        const int r0 = (threadIdx.x & 31) / wide;
#pragma unroll
        for (int r = 0; r < ROWS; r += high) {
#pragma unroll
            for (int q = 0; q < turns; ++q) {
                const int n = r0 + r < rows ? bytes[q] : 0;   // nothing is read where n is 0
                cp_async<PIECE>(slot + offset + (r * kC + q * wide * per) * (int)sizeof(T), f + q * wide * per, n);
            }
            f += high * row_stride;
        }
    }
    __device__ __forceinline__ int shift(int) const { return 0; }
};

// Elements from one row of a slot to the next.
constexpr int pitch_of(int piece) { return piece >= 4 ? kC : kC + 2; }

// Two-byte elements at any address: the aligned words that hold a row, 32 or 33 of them, of which an odd row uses the first from its
// upper half on.  (The lower half of that word is the element before the row or, before a tensor's first, whatever shares its four
// bytes: it is fetched and not used.)
template <int ROWS, typename T> struct Feed<ROWS, 2, T> {
    const T *from;
    int64_t row_stride, advance;
    int cols, first, odd;   // halves before row 0's first element in its word, and whether rows take turns
    __device__ __forceinline__ Feed(const T *src, int64_t t, int64_t rs, int steps, int cols_, int) {
        row_stride = rs;
        advance = steps * rs;
        cols = min(cols_, kC);
        from = src + t * rs;
        first = (int)((uintptr_t)from >> 1) & 1;
        odd = (int)rs & 1;   // steps is even, so the first row of every fetch lies like the first
    }
    __device__ __forceinline__ int shift(int row) const { return first ^ (row & odd); }
    __device__ __forceinline__ void whole(uint32_t slot) { part(slot, ROWS); }
    __device__ __forceinline__ int bytes(int word, int before) const { return min(max((cols - (2 * word - before)) * 2, 0), 4); }
    // word `word` of a row; nothing is read where n is 0
    __device__ __forceinline__ void copy(uint32_t dst, const T *row, int word, int n) const {
        cp_async<4>(dst + 4 * word, reinterpret_cast<const char *>((uintptr_t)row & ~(uintptr_t)3) + 4 * word, n);
    }
    __device__ __forceinline__ void part(uint32_t slot, int rows) {
        const int lane = threadIdx.x & 31;
        const int n[2] = {bytes(lane, first), bytes(lane, first ^ odd)};   // of even rows, of odd ones
        const T *f = from;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            copy(slot + r * pitch_of(2) * 2, f, lane, r < rows ? n[r & 1] : 0);
            f += row_stride;
        }
        if (lane < ROWS) copy(slot + lane * pitch_of(2) * 2, from + lane * row_stride, 32, lane < rows ? bytes(32, shift(lane)) : 0);
        from += advance;
    }
};

// A lane's two channels.
__device__ __forceinline__ float2 load2(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 load2(const __nv_bfloat16 *p) {
    const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
// the same of a row of a slot, which begins `shift` elements into its first word
template <int PIECE, typename T> __device__ __forceinline__ float2 slot2(const T *p, int shift) {
    if constexpr (PIECE >= 4) {
        return load2(p);
    } else {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(p);
        const uint32_t u = __funnelshift_r(w[0], w[1], 16 * shift);
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
}
__device__ __forceinline__ void store2(float *p, float2 v) { *reinterpret_cast<float2 *>(p) = v; }
__device__ __forceinline__ void store2(__nv_bfloat16 *p, float2 v) { *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(v.x, v.y); }
// what another launch of the call may have written: from L2
__device__ __forceinline__ float2 load_carry(const float *p, int n) { return make_float2(n > 0 ? __ldcg(p) : 0.f, n > 1 ? __ldcg(p + 1) : 0.f); }
// the first n of them, at any alignment
template <typename T> __device__ __forceinline__ float2 load_some(const T *p, int n) {
    return make_float2(n > 0 ? ld_f32(p) : 0.f, n > 1 ? ld_f32(p + 1) : 0.f);
}
template <typename T> __device__ __forceinline__ void store_some(T *p, float2 v, int n) {
    if (n > 0) st_f32(p, v.x);
    if (n > 1) st_f32(p + 1, v.y);
}

// A pair of gates -> decays a = sigmoid(g) and 1 - a, both good relative to themselves: with e = exp(-g), a = 1 / (1 + e) and
// 1 - a = e a, neither of which cancels.  e is held to about 2^126, where 1 - a comes out as 1 and a, which would be the smallest normal
// number there and below it behind, is set to zero.  A NaN goes through.
// FAST, for bf16 tensors: one exp2 and one reciprocal of the special-function unit, a off by at most (|g| + 9) 2^-24 of itself, a few
// 2^-24 where it is near one (e's error counts for e / (1 + e) of itself).  The step takes the other form for every type.
// Along a memory of 1 / (1 - a) steps an error of a counts that often: constant inputs settle at 1 + (a's error) / (1 - a) times what
// they should, in either form, because 1 + e is rounded: off by 1e-4 at g = 7.5, 6e-4 at 10, 4e-3 at 13, where an exact a rounded to
// fp32 leaves 1e-5, 5e-4 and 4e-4.
// Otherwise e = 2^t (1 + (t' - t) ln 2), t the rounded and t' the exact product -g log2(e), and one Newton step on the reciprocal.
template <bool FAST> __device__ __forceinline__ void sigmoid2(float2 g, float2 &a, float2 &rest) {
    float2 e, end;   // end: 1 where e is held
    if constexpr (FAST) {
        float2 t = mul2(g, make_float2(-kLog2e, -kLog2e));
        asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(t.x));   // 126
        asm("min.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(t.y));
        asm("set.ge.f32.f32 %0, %1, 0f42FC0000;" : "=f"(end.x) : "f"(t.x));
        asm("set.ge.f32.f32 %0, %1, 0f42FC0000;" : "=f"(end.y) : "f"(t.y));
        e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
    } else {
        constexpr float kLog2eLow = (float)(1.44269504088896340736 - (double)kLog2e);
        asm("max.NaN.f32 %0, %0, 0fC2AEAC4F;" : "+f"(g.x));   // -126 ln 2
        asm("max.NaN.f32 %0, %0, 0fC2AEAC4F;" : "+f"(g.y));
        asm("set.le.f32.f32 %0, %1, 0fC2AEAC4F;" : "=f"(end.x) : "f"(g.x));
        asm("set.le.f32.f32 %0, %1, 0fC2AEAC4F;" : "=f"(end.y) : "f"(g.y));
        asm("min.NaN.f32 %0, %0, 0f43480000;" : "+f"(g.x));   // 200: e is zero there, and t finite
        asm("min.NaN.f32 %0, %0, 0f43480000;" : "+f"(g.y));
        const float2 t = mul2(g, splat2(-kLog2e));
        const float2 low = fma2(g, splat2(-kLog2eLow), fma2(g, splat2(-kLog2e), make_float2(-t.x, -t.y)));
        e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
        e = fma2(e, mul2(low, splat2(kLn2)), e);
    }
    const float2 d = add2(e, splat2(1.f));
    float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    if constexpr (!FAST) r = fma2(r, fma2(make_float2(-d.x, -d.y), r, splat2(1.f)), r);
    rest = mul2(e, r);
    a = fma2(end, make_float2(-r.x, -r.y), r);
}

constexpr float kLargest = 3.402823466e38f;

// One step's decay and input from its gate and x; `rest` is 1 - a (sigmoid only).
template <int GATE, bool FAST> __device__ __forceinline__ void gate_step(float2 g, float2 x, float2 &a, float2 &b, float2 &rest) {
    if constexpr (GATE == HX_GATE_SIGMOID) {
        sigmoid2<FAST>(g, a, rest);
        b = mul2(rest, x);
    } else {
        a = g;
        b = x;
    }
}

// The steps a launch covers, and the state (backwards: e) it starts from and leaves behind.
struct Span {
    int begin, end;
    const float *in;   // [batch, d_inner] or NULL: zero
    float *out;        // or NULL
    bool more;         // another launch of the same call follows
};

// What one warp works on.
struct Part {
    int b, d0, seg, lane, c, n, cols;   // batch row, first channel of the tile, segment; the lane's channels c.. and how many exist
    int len, end;                       // of the batch row, and of what the launch covers of it
    int t0, t1;                         // the segment's steps, before `end`
    bool live;
};
__device__ __forceinline__ Part part_of(int batch, int seq_len, int d_inner, const int32_t *lengths, const Span &span, int seg_len, int segs,
                                        int first_seg, int count) {   // segments first_seg .. first_seg + count - 1 of segs
    Part q;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int tiles = (d_inner + kC - 1) / kC;
    const int64_t w = (int64_t)blockIdx.x * kWarps + warp;
    q.live = w < (int64_t)tiles * batch * count;
    const int64_t row = q.live ? w / tiles : 0;
    q.d0 = q.live ? (int)(w % tiles) * kC : 0;
    q.b = (int)(row % batch);
    q.seg = (int)(row / batch) + first_seg;
    q.lane = threadIdx.x & 31;
    q.c = q.d0 + 2 * q.lane;
    q.cols = d_inner - q.d0;
    q.n = min(max(d_inner - q.c, 0), 2);
    q.len = lengths ? min(max(lengths[q.b], 0), seq_len) : seq_len;
    q.end = min(q.len, span.end);
    q.t0 = (int)min(span.begin + (int64_t)q.seg * seg_len, (int64_t)q.end);
    q.t1 = q.seg == segs - 1 ? q.end : (int)min(span.begin + (int64_t)(q.seg + 1) * seg_len, (int64_t)q.end);
    return q;
}
// maps: [segment][batch][d_inner rounded up to 2] pairs (A, B) of a channel
__device__ __forceinline__ float4 *map_at(float2 *maps, int seg, int b, int c, int batch, int d_inner) {
    return reinterpret_cast<float4 *>(maps + ((int64_t)seg * batch + b) * ((d_inner + 1) & ~1) + c);
}

// A segment's map h -> A h + B of a channel and what it is good for, built from its last run of steps to its first.
// A run has gone from the state 0 to r and has multiplied by p; `least` and `most` are the smallest and the largest |product| on the way.
//   overflow   A walk of the run from 0 that overflows leaves r, and then B, infinite or NaN.  What a state entering the run adds to it
//              is at most lift |h| from before the segment and `reach` from its own runs; where both are below 2^102, half the last
//              place of the largest number and less, the walk from h overflows where that from 0 does.
//   underflow  lost_a and lost_b bound the absolute error that products below 2^-126 have left in A and B: 2^-149 a rounding, times
//              the products that follow.  They are kept times 2^100, so that a bound does not underflow itself before the largest
//              run result (2^102) makes less than 2^-126 of it.
// A map is marked where lift or reach is too large, or where more is lost than 2^-24 of the value and than what odd() accepts.
// All this costs 2 to 5 % of a cut call (1 x 32768 x 1536 fp32 130 us without, 134 with; 7 x 731 x 1000 bf16 15.7, 16.2; 1 x 16384 x 256
// bf16 decays, of 128 segments, 17.4, 19.1).
constexpr float kMostLift = 0x1p22f, kMostState = 0x1p80f, kMostReach = 0x1p102f, kNormal = 0x1p-126f, kStep = 0x1p-49f;   // 2^-149
template <int GATE> struct Reach {
    float lift = 1.f, reach = 0.f, lost_a = 0.f, lost_b = 0.f;
    // before A and B take the run up; ep: the error of p
    __device__ __forceinline__ void add(float A, float p, float r, float most, float ep) {
        lost_b = fmaf(lost_a, fabsf(r), lost_b);
        reach = fmaf(lift, fabsf(r), reach);
        if constexpr (GATE == HX_GATE_DECAY) lift = fmaxf(fmaxf(most, 1.f), lift * fabsf(p));   // a sigmoid's is 1
        lost_a = fmaf(lost_a, fmaf(ep, 0x1p-100f, fabsf(p)), fmaf(fabsf(A), ep, A != 0.f && fabsf(A * p) < kNormal ? kStep : 0.f));
    }
    __device__ __forceinline__ float mark(float A, float B) const {
        const bool good = lift < kMostLift && reach < kMostReach && (lost_a <= 0x1p-40f || lost_a <= 0x1p76f * fabsf(A)) &&
                          (lost_b <= 0x1p-26f || lost_b <= 0x1p76f * fabsf(B));
        return good ? A : __int_as_float(0x7fc00000);
    }
};
// The run's error of p where products on the way are below 2^-126: nearly never with decays, and then worth a second look, unless
// nothing that it multiplies is left (A is zero, and exactly so).  A sigmoid's decays are at most 1, so that each rounding counts once.
template <int GATE> __device__ __forceinline__ float lost_in_run(const float (&a)[kRun], float least, float A, float lost_a) {
    if (!(least < kNormal) || (A == 0.f && lost_a == 0.f)) return 0.f;
    if constexpr (GATE == HX_GATE_SIGMOID) {
        return kRun * kStep;
    } else {
        float p = 1.f, lost = 0.f;
        for (int s = 0; s < kRun; ++s) {
            const float next = p * a[s];
            lost = fmaf(lost, fabsf(a[s]), p != 0.f && a[s] != 0.f && fabsf(next) < kNormal ? kStep : 0.f);
            p = next;
        }
        return lost;
    }
}
// Takes a run up into A and B.  The run itself is walked as the recurrence goes; BACK: e -> a (v + e) from its last step to its first.
template <int GATE, bool BACK>
__device__ __forceinline__ void add_run(const float2 (&a)[kRun], const float2 (&v)[kRun], float2 &A, float2 &B, Reach<GATE> (&reach)[2]) {
    float2 p, r, least, most;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const int s = BACK ? kRun - 1 - i : i;
        p = i == 0 ? a[s] : mul2(p, a[s]);
        if constexpr (BACK) r = mul2(a[s], i == 0 ? v[s] : add2(v[s], r));
        else r = i == 0 ? v[s] : fma2(a[s], r, v[s]);
        const float2 size = make_float2(fabsf(p.x), fabsf(p.y));
        if (i == 0) least = most = size;
        if constexpr (GATE == HX_GATE_DECAY) {
            least = make_float2(fminf(least.x, size.x), fminf(least.y, size.y));
            most = make_float2(fmaxf(most.x, size.x), fmaxf(most.y, size.y));
        } else {
            least = size;   // the products of a sigmoid only shrink
        }
    }
    float ax[kRun], ay[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) ax[i] = a[BACK ? kRun - 1 - i : i].x, ay[i] = a[BACK ? kRun - 1 - i : i].y;
    reach[0].add(A.x, p.x, r.x, most.x, lost_in_run<GATE>(ax, least.x, A.x, reach[0].lost_a));
    reach[1].add(A.y, p.y, r.y, most.y, lost_in_run<GATE>(ay, least.y, A.y, reach[1].lost_a));
    B = fma2(A, r, B);
    A = mul2(A, p);
}
// A map may not be applied to h, where that gave `next`: it is marked; h is beyond what it is good for, or infinite and A zero, which
// may be an underflow (infinity over any other A, and NaN, are as in the walk); or A has lost what h would have made larger than both
// 2^-126 and 2^-24 of the result (A is off by up to 2^-140, or by less than 2^-24 of itself).
__device__ __forceinline__ bool odd(float A, float h, float next) {
    const float ah = fabsf(h);
    if (ah <= 0x1p14f) return A != A;
    return h == h && (A != A || (ah > kMostState && !(ah > kLargest && A != 0.f)) || (fabsf(A) < 0x1p-116f && ah * 0x1p-116f > fabsf(next)));
}

// Folds `count` maps onto h, the k-th at `first + k * step`, kFold of them in one round trip to L2 and the next kFold under way.  Where
// one may not be applied, its channel takes what walk(k, h), the walk of the k-th map's segment from h, gives instead.  A channel's
// result depends on its own numbers alone, whatever the other channels of the warp hold.
// Every later segment's warp walks such a segment for itself.  Two NaN in one channel: 1 x 32768 x 1536 fp32 159 us for 135, 7 x 731 x
// 1000 bf16 43 for 17; a channel whose states are beyond 2^80 from end to end, where every segment is walked: 3.8 ms and 0.26.
constexpr int kFold = 8;
template <typename Walk>
__device__ __forceinline__ void fold(const float4 *first, int64_t step, int count, bool real, float2 &h, Walk walk) {
    float4 m[2][kFold];
    auto load = [&](float4 (&b)[kFold], int k0) {
#pragma unroll
        for (int k = 0; k < kFold; ++k) b[k] = k0 + k < count && real ? __ldcg(first + (k0 + k) * step) : make_float4(1.f, 0.f, 1.f, 0.f);
    };
    int done = 0;
    auto fast = [&]() {   // until all are folded, or up to eight of which one may not be
        load(m[0], done);
        while (true)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (done >= count) return;
                load(m[half ^ 1], done + kFold);
                float2 s = h;
                bool large = false;   // a marked map leaves NaN, so that nothing is odd where no state is large
#pragma unroll
                for (int k = 0; k < kFold; ++k) {
                    large |= !(fabsf(s.x) <= 0x1p14f) || !(fabsf(s.y) <= 0x1p14f);
                    s = make_float2(fmaf(m[half][k].x, s.x, m[half][k].y), fmaf(m[half][k].z, s.y, m[half][k].w));
                }
                large |= !(fabsf(s.x) <= 0x1p14f) || !(fabsf(s.y) <= 0x1p14f);
                if (__any_sync(0xffffffffu, large)) {
                    bool any = false;
                    s = h;
#pragma unroll
                    for (int k = 0; k < kFold; ++k) {
                        const float2 next = make_float2(fmaf(m[half][k].x, s.x, m[half][k].y), fmaf(m[half][k].z, s.y, m[half][k].w));
                        any |= odd(m[half][k].x, s.x, next.x) || odd(m[half][k].z, s.y, next.y);
                        s = next;
                    }
                    if (__any_sync(0xffffffffu, any)) return;
                }
                h = s;
                done += kFold;
            }
    };
    while (true) {
        fast();
        if (done >= count) return;
        for (const int end = min(done + kFold, count); done < end; ++done) {   // one by one
            const float4 one = real ? __ldcg(first + done * step) : make_float4(1.f, 0.f, 1.f, 0.f);
            float2 next = make_float2(fmaf(one.x, h.x, one.y), fmaf(one.z, h.y, one.w));
            const bool x = odd(one.x, h.x, next.x), y = odd(one.z, h.y, next.y);
            if (__any_sync(0xffffffffu, x || y)) {
                const float2 w = walk(done, h);
                next = make_float2(x ? w.x : next.x, y ? w.y : next.y);
            }
            h = next;
        }
    }
}

// ---------------------------------------------------------------- forward
// MAP: writes the maps of segments 0 .. segs - 2.  Otherwise: outputs of all segments.
template <typename T, int GATE, int PIECE, bool MAP>
__global__ void __launch_bounds__(32 * kWarps, kOccupancy)
gated_scan_kernel(const hx_gated_scan_args p, const Span span, float2 *maps, int seg_len, int segs) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int STAGES = kStages;
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int P = pitch_of(PIECE);
    using Ring = T[STAGES][2][kRun][P];
    Ring &ring = reinterpret_cast<Ring *>(smem)[threadIdx.x >> 5];
    if (MAP || span.more) chain_trigger();
    const Part q = part_of(p.batch, p.seq_len, p.d_inner, p.lengths, span, seg_len, segs, 0, MAP ? segs - 1 : segs);
    if (!q.live) return;
    const T *x = static_cast<const T *>(p.x) + q.b * p.x_batch_stride + q.d0;
    const T *g = static_cast<const T *>(p.g) + q.b * p.g_batch_stride + q.d0;
    const int ragged = (q.t1 - q.t0) % kRun, runs = (q.t1 - q.t0) / kRun + (ragged > 0);   // rows of the last run, 0: all
    // MAP walks from the last run to the first
    const int64_t first = q.t0 + (int64_t)(MAP ? runs - 1 : 0) * kRun;
    Feed<kRun, PIECE, T> feed_g(g, first, p.g_row_stride, MAP ? -kRun : kRun, q.cols, q.lane);
    Feed<kRun, PIECE, T> feed_x(x, first, p.x_row_stride, MAP ? -kRun : kRun, q.cols, q.lane);
    constexpr uint32_t slot_bytes = sizeof(ring[0]), ring_bytes = sizeof(ring);
    const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(&ring[0][0][0][0]);
    uint32_t to = 0;                           // slot that is filled next
    auto issue = [&](int r) {                  // the r-th run of the walk
        if (r < runs) {
            __syncwarp();   // the warp is done with what the slot held
            const uint32_t slot = ring0 + to;
            if (ragged && r == (MAP ? 0 : runs - 1)) {
                feed_g.part(slot, ragged);
                feed_x.part(slot + slot_bytes / 2, ragged);
            } else {
                feed_g.whole(slot);
                feed_x.whole(slot + slot_bytes / 2);
            }
            to = to + slot_bytes == ring_bytes ? 0 : to + slot_bytes;
        }
        cp_commit();
    };
#pragma unroll
    for (int r = 0; r < STAGES - 1; ++r) issue(r);

    float2 h = make_float2(0.f, 0.f), A = make_float2(1.f, 1.f);   // MAP: B and A of the runs walked so far
    Reach<GATE> reach[2];
    T *out = static_cast<T *>(p.h) + q.b * p.h_batch_stride + q.c;
    const int64_t blocks = ((int64_t)p.seq_len + kBlock - 1) / kBlock;
    float *states = !MAP && p.states ? p.states + q.b * blocks * p.d_inner + q.c : nullptr;
    const bool whole = PIECE >= 2 * (int)sizeof(T) && q.n == 2;
    const bool even = p.d_inner % 2 == 0 && (uintptr_t)p.states % 8 == 0;   // two states at a time
    if constexpr (!MAP) {
        if (segs > 1) chain_wait();
        if (span.in) h = load_carry(span.in + (int64_t)q.b * p.d_inner + q.c, q.n);
        if (segs > 1) {
            const int64_t step = map_at(maps, 1, 0, 0, p.batch, p.d_inner) - map_at(maps, 0, 0, 0, p.batch, p.d_inner);
            fold(map_at(maps, 0, q.b, q.c, p.batch, p.d_inner), step, q.seg, q.n > 0, h, [&](int j, float2 h) {
                const int64_t end = min(span.begin + (int64_t)(j + 1) * seg_len, (int64_t)q.end);
                for (int64_t t = span.begin + (int64_t)j * seg_len; t < end; t += kRun) {
                    float2 gv[kRun], xv[kRun];
#pragma unroll
                    for (int s = 0; s < kRun; ++s) {
                        const int n = t + s < end ? q.n : 0;
                        gv[s] = load_some(g + (t + s) * p.g_row_stride + 2 * q.lane, n);
                        xv[s] = load_some(x + (t + s) * p.x_row_stride + 2 * q.lane, n);
                    }
#pragma unroll
                    for (int s = 0; s < kRun; ++s)
                        if (t + s < end) {
                            float2 a, b, rest;
                            gate_step<GATE, FAST>(gv[s], xv[s], a, b, rest);
                            h = fma2(a, h, b);
                        }
                }
                return h;
            });
        }
    }
    const T *slot_g = &ring[0][0][0][2 * q.lane], *const slot_end = slot_g + STAGES * 2 * kRun * P;
    T *o = out + q.t0 * p.h_row_stride;
    float *st = states ? states + (int64_t)(q.t0 / kBlock) * p.d_inner : nullptr;
    bool keep = states != nullptr;   // every other run starts at a state to be kept
    for (int r = 0; r < runs; ++r) {
        cp_wait<STAGES - 2>();
        __syncwarp();
        float2 a[kRun], v[kRun];
#pragma unroll
        for (int s = 0; s < kRun; ++s) {
            float2 rest;
            gate_step<GATE, FAST>(slot2<PIECE>(slot_g + s * P, feed_g.shift(s)), slot2<PIECE>(slot_g + (kRun + s) * P, feed_x.shift(s)), a[s], v[s], rest);
        }
        slot_g += 2 * kRun * P;
        if (slot_g == slot_end) slot_g = &ring[0][0][0][2 * q.lane];
        issue(r + STAGES - 1);
        const int rows = ragged && r == (MAP ? 0 : runs - 1) ? ragged : kRun;
        if constexpr (MAP) {
            if (rows < kRun) {   // steps that are not there: identities
#pragma unroll
                for (int s = 0; s < kRun; ++s)
                    if (s >= rows) a[s] = make_float2(1.f, 1.f), v[s] = make_float2(0.f, 0.f);
            }
            add_run<GATE, false>(a, v, A, h, reach);
        } else {
            if (keep) {
                if (even && q.n == 2) store2(st, h);
                else store_some(st, h, q.n);
                st += p.d_inner;
            }
            keep = !keep && states;
            if (rows == kRun && whole) {
#pragma unroll
                for (int s = 0; s < kRun; ++s) {
                    h = fma2(a[s], h, v[s]);
                    store2(o, h);
                    o += p.h_row_stride;
                }
            } else {
#pragma unroll
                for (int s = 0; s < kRun; ++s)
                    if (s < rows) {
                        h = fma2(a[s], h, v[s]);
                        store_some(o, h, q.n);
                        o += p.h_row_stride;
                    }
            }
        }
    }
    if constexpr (MAP) {
        chain_wait();   // the launch before this one has read the maps of its span
        if (q.n) *map_at(maps, q.seg, q.b, q.c, p.batch, p.d_inner) = make_float4(reach[0].mark(A.x, h.x), h.x, reach[1].mark(A.y, h.y), h.y);
    } else {
        const int64_t end = q.seg == segs - 1 ? span.end : min(span.begin + (int64_t)(q.seg + 1) * seg_len, (int64_t)span.end);
        for (int64_t t = max(span.begin + (int64_t)q.seg * seg_len, (int64_t)q.len); t < end; ++t) store_some(out + t * p.h_row_stride, make_float2(0.f, 0.f), q.n);
        if (span.out && q.seg == segs - 1) store_some(span.out + (int64_t)q.b * p.d_inner + q.c, h, q.n);
    }
}

// ---------------------------------------------------------------- backward
// MAP: writes the maps e behind the segment -> e before it, of segments 1 .. segs - 1, walking forward.  Otherwise: the gradients,
// walking from the end.
template <typename T, int GATE, int PIECE, bool MAP>
__global__ void __launch_bounds__(32 * kWarps, MAP ? kOccupancy : kBlockOccupancy)
gated_scan_bwd_kernel(const hx_gated_scan_bwd_args p, const Span span, float2 *maps, int seg_len, int segs) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int STAGES = MAP ? kStages : kBlockStages, ROWS = MAP ? kRun : kBlock, TENSORS = MAP ? 2 : 3;
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int P = pitch_of(PIECE);
    using Ring = T[STAGES][TENSORS][ROWS][P];   // g, dh, x
    Ring &ring = reinterpret_cast<Ring *>(smem)[threadIdx.x >> 5];
    if (MAP || span.more) chain_trigger();
    const Part q = part_of(p.batch, p.seq_len, p.d_inner, p.lengths, span, seg_len, segs, MAP ? 1 : 0, MAP ? segs - 1 : segs);
    if (!q.live) return;
    const T *x = static_cast<const T *>(p.x) + q.b * p.x_batch_stride + q.d0;
    const T *g = static_cast<const T *>(p.g) + q.b * p.g_batch_stride + q.d0;
    const T *dh = static_cast<const T *>(p.dh) + q.b * p.dh_batch_stride + q.d0;
    const int ragged = (q.t1 - q.t0) % ROWS, runs = (q.t1 - q.t0) / ROWS + (ragged > 0);
    const int64_t first = q.t0 + (int64_t)(MAP ? 0 : runs - 1) * ROWS;
    constexpr int way = MAP ? ROWS : -ROWS;
    Feed<ROWS, PIECE, T> feed_g(g, first, p.g_row_stride, way, q.cols, q.lane);
    Feed<ROWS, PIECE, T> feed_d(dh, first, p.dh_row_stride, way, q.cols, q.lane);
    Feed<ROWS, PIECE, T> feed_x(x, first, p.x_row_stride, way, q.cols, q.lane);
    constexpr uint32_t part_bytes = sizeof(ring[0][0]), slot_bytes = sizeof(ring[0]), ring_bytes = sizeof(ring);
    const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(&ring[0][0][0][0]);
    uint32_t to = 0;
    auto issue = [&](int r) {
        if (r < runs) {
            __syncwarp();
            const uint32_t slot = ring0 + to;
            if (ragged && r == (MAP ? runs - 1 : 0)) {
                feed_g.part(slot, ragged);
                feed_d.part(slot + part_bytes, ragged);
                if constexpr (!MAP) feed_x.part(slot + 2 * part_bytes, ragged);
            } else {
                feed_g.whole(slot);
                feed_d.whole(slot + part_bytes);
                if constexpr (!MAP) feed_x.whole(slot + 2 * part_bytes);
            }
            to = to + slot_bytes == ring_bytes ? 0 : to + slot_bytes;
        }
        cp_commit();
    };
#pragma unroll
    for (int r = 0; r < STAGES - 1; ++r) issue(r);
    const T *slot = &ring[0][0][0][2 * q.lane], *const slot_end = slot + STAGES * TENSORS * ROWS * P;

    if constexpr (MAP) {
        float2 E = make_float2(0.f, 0.f), A = make_float2(1.f, 1.f);
        Reach<GATE> reach[2];
        for (int r = 0; r < runs; ++r) {
            cp_wait<STAGES - 2>();
            __syncwarp();
            float2 a[kRun], v[kRun];
#pragma unroll
            for (int s = 0; s < kRun; ++s) {
                float2 rest, b;
                v[s] = slot2<PIECE>(slot + (ROWS + s) * P, feed_d.shift(s));
                gate_step<GATE, FAST>(slot2<PIECE>(slot + s * P, feed_g.shift(s)), v[s], a[s], b, rest);
            }
            slot += TENSORS * ROWS * P;
            if (slot == slot_end) slot = &ring[0][0][0][2 * q.lane];
            issue(r + STAGES - 1);
            if (ragged && r == runs - 1) {
#pragma unroll
                for (int s = 0; s < kRun; ++s)
                    if (s >= ragged) a[s] = make_float2(1.f, 1.f), v[s] = make_float2(0.f, 0.f);
            }
            add_run<GATE, true>(a, v, A, E, reach);
        }
        chain_wait();   // the launch before this one has read the maps of its span
        if (q.n) *map_at(maps, q.seg - 1, q.b, q.c, p.batch, p.d_inner) = make_float4(reach[0].mark(A.x, E.x), E.x, reach[1].mark(A.y, E.y), E.y);
    } else {
        const int64_t blocks = ((int64_t)p.seq_len + kBlock - 1) / kBlock;
        const bool even = p.d_inner % 2 == 0 && (uintptr_t)p.states % 8 == 0;   // two states at a time
        auto state_of = [&](int r) {   // the state before the r-th block of the walk
            if (r >= runs) return make_float2(0.f, 0.f);
            const float *st = p.states + (q.b * blocks + q.t0 / kBlock + (runs - 1 - r)) * p.d_inner + q.c;
            return even && q.n == 2 ? load2(st) : load_some(st, q.n);
        };
        float2 state = state_of(0);
        if (segs > 1) chain_wait();
        float2 e = span.in ? load_carry(span.in + (int64_t)q.b * p.d_inner + q.c, q.n) : make_float2(0.f, 0.f);
        if (segs > 1) {
            const int64_t step = map_at(maps, 1, 0, 0, p.batch, p.d_inner) - map_at(maps, 0, 0, 0, p.batch, p.d_inner);
            fold(map_at(maps, segs - 2, q.b, q.c, p.batch, p.d_inner), -step, segs - 1 - q.seg, q.n > 0, e, [&](int k, float2 e) {
                const int64_t begin = span.begin + (int64_t)(segs - 1 - k) * seg_len;   // of the k-th segment from the end
                for (int64_t t = min(begin + seg_len, (int64_t)q.end) - 1; t >= begin; t -= kRun) {
                    float2 gv[kRun], dv[kRun];
#pragma unroll
                    for (int s = 0; s < kRun; ++s) {
                        const int n = t - s >= begin ? q.n : 0;
                        gv[s] = load_some(g + (t - s) * p.g_row_stride + 2 * q.lane, n);
                        dv[s] = load_some(dh + (t - s) * p.dh_row_stride + 2 * q.lane, n);
                    }
#pragma unroll
                    for (int s = 0; s < kRun; ++s)
                        if (t - s >= begin) {
                            float2 a, b, rest;
                            gate_step<GATE, FAST>(gv[s], dv[s], a, b, rest);
                            e = mul2(a, add2(e, dv[s]));
                        }
                }
                return e;
            });
        }
        const bool whole = PIECE >= 2 * (int)sizeof(T) && q.n == 2;
        T *dx = static_cast<T *>(p.dx) + q.b * p.dx_batch_stride + q.c;
        T *dg = static_cast<T *>(p.dg) + q.b * p.dg_batch_stride + q.c;
        T *ox = dx + ((int64_t)q.t1 - 1) * p.dx_row_stride, *og = dg + ((int64_t)q.t1 - 1) * p.dg_row_stride;
        for (int r = 0; r < runs; ++r) {
            cp_wait<STAGES - 2>();
            __syncwarp();
            const int rows = ragged && r == 0 ? ragged : kBlock;
            float2 a[kBlock], rest[kBlock], before[kBlock];
            const float2 next_state = state_of(r + 1);
#pragma unroll
            for (int s = 0; s < kBlock; ++s) {   // rows behind the end are zeros here: what they give is not used
                float2 b;
                gate_step<GATE, FAST>(slot2<PIECE>(slot + s * P, feed_g.shift(s)), slot2<PIECE>(slot + (2 * kBlock + s) * P, feed_x.shift(s)), a[s], b, rest[s]);
                before[s] = state;
                state = fma2(a[s], state, b);
            }
            state = next_state;
            issue(r + STAGES - 1);
            auto gradients = [&](int s, float2 &dxv, float2 &dgv) {
                const float2 d = add2(slot2<PIECE>(slot + (kBlock + s) * P, feed_d.shift(s)), e);   // delta
                e = mul2(a[s], d);
                if constexpr (GATE == HX_GATE_SIGMOID) {
                    dxv = mul2(d, rest[s]);
                    // delta (h - x) a (1 - a), with e = a delta
                    dgv = mul2(mul2(e, rest[s]), fma2(slot2<PIECE>(slot + (2 * kBlock + s) * P, feed_x.shift(s)), make_float2(-1.f, -1.f), before[s]));
                } else {
                    dxv = d;
                    dgv = mul2(d, before[s]);
                }
            };
            float2 dxv, dgv;
            if (rows == kBlock && whole) {
#pragma unroll
                for (int s = kBlock - 1; s >= 0; --s) {
                    gradients(s, dxv, dgv);
                    store2(ox, dxv);
                    store2(og, dgv);
                    ox -= p.dx_row_stride;
                    og -= p.dg_row_stride;
                }
            } else {
#pragma unroll
                for (int s = kBlock - 1; s >= 0; --s)
                    if (s < rows) {
                        gradients(s, dxv, dgv);
                        store_some(ox, dxv, q.n);
                        store_some(og, dgv, q.n);
                        ox -= p.dx_row_stride;
                        og -= p.dg_row_stride;
                    }
            }
            slot += TENSORS * ROWS * P;
            if (slot == slot_end) slot = &ring[0][0][0][2 * q.lane];
        }
        const int64_t end = q.seg == segs - 1 ? span.end : min(span.begin + (int64_t)(q.seg + 1) * seg_len, (int64_t)span.end);
        for (int64_t t = max(span.begin + (int64_t)q.seg * seg_len, (int64_t)q.len); t < end; ++t) {
            store_some(dx + t * p.dx_row_stride, make_float2(0.f, 0.f), q.n);
            store_some(dg + t * p.dg_row_stride, make_float2(0.f, 0.f), q.n);
        }
        if (span.out && q.seg == 0) store_some(span.out + (int64_t)q.b * p.d_inner + q.c, e, q.n);
    }
}

// ---------------------------------------------------------------- one token
// Two channels a thread, so that a row's halves of a projection are read in words where they are aligned (`pairs`).
template <typename T, int GATE>
__global__ void __launch_bounds__(128)
gated_step_kernel(const T *x, int64_t x_stride, const T *g, int64_t g_stride, const float *h, float *h_out, T *y, int64_t y_stride,
                  int batch, int d_inner, bool pairs) {
    const int half = (d_inner + 1) / 2;
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (i >= (int64_t)batch * half) return;
    const int b = (int)(i / half), d = (int)(i % half) * 2, n = min(d_inner - d, 2);
    const int64_t at = (int64_t)b * d_inner + d;
    x += b * x_stride + d;
    g += b * g_stride + d;
    y += b * y_stride + d;
    float2 a, in, rest;
    if (pairs) {
        gate_step<GATE, false>(load2(g), load2(x), a, in, rest);
        const float2 v = fma2(a, load2(h + at), in);
        store2(h_out + at, v);
        store2(y, v);
    } else {
        gate_step<GATE, false>(load_some(g, n), load_some(x, n), a, in, rest);
        const float2 v = fma2(a, load_some(h + at, n), in);
        store_some(h_out + at, v, n);
        store_some(y, v, n);
    }
}

// Rows of an output [B, L, D] with these strides do not overlap.
static bool rows_apart(int64_t bs, int64_t rs, int64_t B, int64_t L, int64_t D) {
    if (B <= 1 && L <= 1) return true;
    if (L <= 1) return bs >= D;
    if (B <= 1) return rs >= D;
    return (rs >= D && bs >= (L - 1) * rs + D) || (bs >= D && rs >= (B - 1) * bs + D);
}

static hx_status check_common(const char *who, int batch, int seq_len, int d_inner, int gate, int io_dtype) {
    HX_REQUIRE(batch >= 0 && seq_len >= 0 && d_inner >= 0, HX_ERR_INVALID_DIMENSION, "%s: batch %d, seq_len %d, d_inner %d", who, batch,
               seq_len, d_inner);
    HX_REQUIRE(io_dtype == HX_F32 || io_dtype == HX_BF16, HX_ERR_DTYPE_MISMATCH, "%s: io_dtype %d is neither HX_F32 nor HX_BF16", who,
               io_dtype);
    HX_REQUIRE(gate == HX_GATE_DECAY || gate == HX_GATE_SIGMOID, HX_ERR_INVALID_INPUT, "%s: unknown gate %d", who, gate);
    return HX_OK;
}

// The largest of 16, 4 and the element size that divides every address the kernel forms.
static int piece_of(size_t element, std::initializer_list<const void *> bases, std::initializer_list<int64_t> strides) {
    uint64_t bits = 0;
    for (const void *p : bases) bits |= (uint64_t)(uintptr_t)p;
    for (int64_t s : strides) bits |= (uint64_t)s * element;
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : (int)element;
}

// How the sequence is cut.  One segment where a step's channels are at least kStepBytes: a warp takes about 0.04 us a step however
// little else runs, so from there on a single pass is done before two passes (five tensors instead of three, seven instead of five)
// have moved their bytes.  16 x 2048 x 1536 fp32 sigmoid: 111 us whole, 144 in two; 4 x 4096 x 1024 bf16: 182 whole, 40 in 27.
// Otherwise as many segments as give an SM kWarpBytes / element size warps (1 x 16384 x 1536 bf16: 61, 49, 49 us with 32, 48, 96;
// 1 x 32768 x 1536 fp32: 157, 153, 160 with 16, 24, 64), but no more than kMostSegments, whose maps every warp folds
// (1 x 16384 x 256 bf16: 25 us with 96, 34 with 342).
constexpr int64_t kStepBytes = 45000, kWarpBytes = 24, kMostSegments = 128;
// Cut sequences whose two tensors of the first launch are more than L2 holds go span by span, so that the second launch of a span
// finds in L2 what the first has read; the first launch of the next span runs as the second of this one ends.  Forward, 1 x 32768 x
// 1536 fp32: 161 us whole, 143 in spans of 112 MiB, 133 of 56, 140 of 28.  Backward the second launch has a third tensor to read and
// two to write, and shorter spans gain less: 1 x 16384 x 4096 bf16 167 us whole, 154 of 112, 147 of 56; fp32 as above 223, 222, 232.  (All
// with CTAs of four warps and maps without bounds; with two and with bounds, fp32 decays 134 forward and 215 backward.)
constexpr int64_t kSpanBytes = (int64_t)56 << 20, kSpanBytesBwd = (int64_t)112 << 20;
struct Plan { int segs, seg_len, span; };
static Plan whole(int seq_len) { return {1, 0x7fffffff / kBlock * kBlock, seq_len}; }
static Plan plan_of(int batch, int seq_len, int d_inner, int io_dtype, int64_t span_bytes) {
    const int64_t chains = (int64_t)batch * ((d_inner + kC - 1) / kC), e = (int64_t)dtype_size(io_dtype), step = (int64_t)batch * d_inner * e;
    int64_t segs = 1, span = seq_len;
    if (step < kStepBytes) {
        segs = std::min(std::max<int64_t>(kWarpBytes / e * sm_count() / chains, 1), kMostSegments);
        const int64_t spans = (2 * step * seq_len + span_bytes / 2) / span_bytes;
        if (spans > 1 && segs > 1) span = ((seq_len + spans - 1) / spans + kBlock - 1) / kBlock * kBlock;
    }
    int64_t seg_len = (span + segs - 1) / segs;
    seg_len = std::max<int64_t>((seg_len + kBlock - 1) / kBlock * kBlock, 2 * kBlock);
    segs = std::max<int64_t>((span + seg_len - 1) / seg_len, 1);
    if (segs == 1) return whole(seq_len);
    return {(int)segs, (int)seg_len, (int)span};
}
static size_t row_floats(int batch, int d_inner) { return (size_t)batch * ((d_inner + 1) & ~1); }   // of one map's A or B, a multiple of 2
// the maps, and the states between spans, two that take turns
static size_t plan_bytes(int batch, int seq_len, int d_inner, const Plan &plan) {
    if (plan.segs == 1) return 0;
    return ((size_t)(plan.segs - 1) * 2 + (plan.span < seq_len ? 2 : 0)) * row_floats(batch, d_inner) * sizeof(float);
}

template <auto KERNEL, typename Args>
static hx_status launch(size_t ring, bool chained, int64_t warps, const Args &args, const Span &span, const Plan &plan, const char *name, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    const int64_t ctas = (warps + kWarps - 1) / kWarps;
    HX_REQUIRE(ctas <= 0x7fffffff, HX_ERR_INVALID_DIMENSION, "%s: batch * d_inner is too large for one launch", name);
    if (kWarps * ring > 48 * 1024) HX_CUDA(allow_smem((const void *)KERNEL, kWarps * ring, done));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = kWarps * ring;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = chained ? 1 : 0;
    HX_CUDA(cudaLaunchKernelEx(&cfg, KERNEL, args, span, static_cast<float2 *>(args.workspace), plan.seg_len, plan.segs));
    return check_launch(name);
}
// One launch, or two for every span in the order of the walk, each programmatically behind the one before it: MAP(span) starts while
// OUT(span - 1) ends and waits for it before it writes, OUT(span) waits for MAP(span).
template <auto MAP, auto OUT, typename Args>
static hx_status launch_all(size_t map_ring, size_t ring, bool backwards, const float *in, float *out, const Args &a, const Plan &plan,
                            const char *name, cudaStream_t st) {
    const int64_t chains = (int64_t)a.batch * ((a.d_inner + kC - 1) / kC);
    if (plan.segs == 1) return launch<OUT>(ring, false, chains, a, Span{0, a.seq_len, in, out, false}, plan, name, st);
    float *between = static_cast<float *>(a.workspace) + (size_t)(plan.segs - 1) * 2 * row_floats(a.batch, a.d_inner);
    const int spans = (int)(((int64_t)a.seq_len + plan.span - 1) / plan.span);
    for (int i = 0; i < spans; ++i) {
        const int64_t begin = (int64_t)(backwards ? spans - 1 - i : i) * plan.span;
        Span span{(int)begin, (int)std::min<int64_t>(begin + plan.span, a.seq_len), in, out, i + 1 < spans};
        if (i > 0) span.in = between + ((i - 1) & 1) * row_floats(a.batch, a.d_inner);
        if (span.more) span.out = between + (i & 1) * row_floats(a.batch, a.d_inner);
        hx_status s = launch<MAP>(map_ring, i > 0, chains * (plan.segs - 1), a, span, plan, name, st);
        if (s == HX_OK) s = launch<OUT>(ring, true, chains * plan.segs, a, span, plan, name, st);
        if (s != HX_OK) return s;
    }
    return HX_OK;
}
template <typename T, int GATE, int PIECE> static hx_status launch_fwd(const hx_gated_scan_args &a, const Plan &plan, cudaStream_t st) {
    constexpr size_t ring = sizeof(T[kStages][2][kRun][pitch_of(PIECE)]);
    return launch_all<gated_scan_kernel<T, GATE, PIECE, true>, gated_scan_kernel<T, GATE, PIECE, false>>(ring, ring, false, a.h0, a.h_last, a, plan,
                                                                                                         "gated_scan_kernel", st);
}
template <typename T, int GATE, int PIECE> static hx_status launch_bwd(const hx_gated_scan_bwd_args &a, const Plan &plan, cudaStream_t st) {
    return launch_all<gated_scan_bwd_kernel<T, GATE, PIECE, true>, gated_scan_bwd_kernel<T, GATE, PIECE, false>>(
        sizeof(T[kStages][2][kRun][pitch_of(PIECE)]), sizeof(T[kBlockStages][3][kBlock][pitch_of(PIECE)]), true, a.dh_last, a.dh0, a, plan, "gated_scan_bwd_kernel", st);
}

// The plan a call may use: one segment where it brings no workspace.
template <typename Args> static hx_status choose_plan(const char *who, const Args &a, int64_t span_bytes, Plan *plan) {
    *plan = plan_of(a.batch, a.seq_len, a.d_inner, a.io_dtype, span_bytes);
    if (plan->segs == 1) return HX_OK;
    if (a.workspace == nullptr) {
        *plan = whole(a.seq_len);
        return HX_OK;
    }
    const size_t need = plan_bytes(a.batch, a.seq_len, a.d_inner, *plan);
    HX_REQUIRE(a.workspace_bytes >= need, HX_ERR_INVALID_INPUT, "%s: a workspace of %zu bytes, %zu are needed", who, a.workspace_bytes, need);
    HX_REQUIRE(((uintptr_t)a.workspace & 15) == 0, HX_ERR_INVALID_INPUT, "%s: the workspace must be 16-byte aligned", who);
    return HX_OK;
}

template <typename Args> static int64_t states_bytes(const Args &a) {
    return (int64_t)a.batch * (((int64_t)a.seq_len + kBlock - 1) / kBlock) * a.d_inner * 4;
}

}  // namespace gated
}  // namespace hx

using namespace hx;
using namespace hx::gated;

// Picks the instance for a type, a gate and an alignment.
#define HX_GATED_PIECE(FN, T, GATE, PIECE, ...)                                                              \
    do {                                                                                                     \
        if ((PIECE) == 16) return FN<T, GATE, 16>(__VA_ARGS__);                                              \
        if ((PIECE) >= 4) return FN<T, GATE, 4>(__VA_ARGS__);                                                \
        if constexpr (sizeof(T) == 2) return FN<T, GATE, 2>(__VA_ARGS__);                                    \
    } while (0)
#define HX_GATED_LAUNCH(FN, GATE, DTYPE, PIECE, ...)                                                         \
    do {                                                                                                     \
        if ((DTYPE) == HX_BF16) {                                                                            \
            if ((GATE) == HX_GATE_DECAY) HX_GATED_PIECE(FN, __nv_bfloat16, HX_GATE_DECAY, PIECE, __VA_ARGS__); \
            else HX_GATED_PIECE(FN, __nv_bfloat16, HX_GATE_SIGMOID, PIECE, __VA_ARGS__);                     \
        } else {                                                                                             \
            if ((GATE) == HX_GATE_DECAY) HX_GATED_PIECE(FN, float, HX_GATE_DECAY, PIECE, __VA_ARGS__);       \
            else HX_GATED_PIECE(FN, float, HX_GATE_SIGMOID, PIECE, __VA_ARGS__);                             \
        }                                                                                                    \
        return HX_ERR_BACKEND;                                                                               \
    } while (0)

extern "C" {

hx_status hx_gated_scan_fwd(const hx_gated_scan_args *a, void *stream) {
    HX_REQUIRE(a != nullptr, HX_ERR_INVALID_INPUT, "hx_gated_scan_fwd: args is NULL");
    const hx_status s = check_common("hx_gated_scan_fwd", a->batch, a->seq_len, a->d_inner, a->gate, a->io_dtype);
    if (s != HX_OK) return s;
    const int64_t chains = (int64_t)a->batch * a->d_inner;
    if (chains == 0) return HX_OK;
    HX_REQUIRE(a->seq_len == 0 || (a->x && a->g && a->h), HX_ERR_INVALID_INPUT, "hx_gated_scan_fwd: x, g and h must not be NULL");
    HX_REQUIRE(a->x_batch_stride >= 0 && a->x_row_stride >= 0 && a->g_batch_stride >= 0 && a->g_row_stride >= 0 &&
                   a->h_batch_stride >= 0 && a->h_row_stride >= 0,
               HX_ERR_INVALID_INPUT, "hx_gated_scan_fwd: negative stride");
    HX_REQUIRE(rows_apart(a->h_batch_stride, a->h_row_stride, a->batch, a->seq_len, a->d_inner), HX_ERR_SHAPE_MISMATCH,
               "hx_gated_scan_fwd: rows of h overlap (strides %lld, %lld)", (long long)a->h_batch_stride, (long long)a->h_row_stride);
    const int piece = piece_of(dtype_size(a->io_dtype), {a->x, a->g, a->h},
                               {a->x_batch_stride, a->x_row_stride, a->g_batch_stride, a->g_row_stride, a->h_batch_stride, a->h_row_stride});
    Plan plan;
    const hx_status ps = choose_plan("hx_gated_scan_fwd", *a, kSpanBytes, &plan);
    if (ps != HX_OK) return ps;
    auto view = [&](const void *at, int64_t bs, int64_t rs) { return rows_of(at, a->batch, bs, a->seq_len, rs, a->d_inner, dtype_size(a->io_dtype)); };
    const Operand outs[] = {{"h", view(a->h, a->h_batch_stride, a->h_row_stride)},
                            {"h_last", dense_of(a->h_last, chains * 4)},
                            {"states", dense_of(a->states, states_bytes(*a))},
                            {"the workspace", dense_of(a->workspace, (int64_t)a->workspace_bytes)}};
    const Operand ins[] = {{"x", view(a->x, a->x_batch_stride, a->x_row_stride)},
                           {"g", view(a->g, a->g_batch_stride, a->g_row_stride)},
                           {"h0", dense_of(a->h0, chains * 4)},
                           {"lengths", dense_of(a->lengths, (int64_t)a->batch * 4)}};
    const char *one, *other;
    HX_REQUIRE(!shared_operands(outs, ins, one, other), HX_ERR_INVALID_INPUT, "hx_gated_scan_fwd: %s and %s share memory", one, other);
    HX_GATED_LAUNCH(launch_fwd, a->gate, a->io_dtype, piece, *a, plan, (cudaStream_t)stream);
}

hx_status hx_gated_scan_workspace_bytes(int32_t batch, int32_t seq_len, int32_t d_inner, int32_t io_dtype, size_t *bytes) {
    HX_REQUIRE(bytes != nullptr, HX_ERR_INVALID_INPUT, "hx_gated_scan_workspace_bytes: bytes is NULL");
    const hx_status s = check_common("hx_gated_scan_workspace_bytes", batch, seq_len, d_inner, HX_GATE_DECAY, io_dtype);
    if (s != HX_OK) return s;
    *bytes = 0;
    if ((int64_t)batch * d_inner > 0)
        for (int64_t span_bytes : {kSpanBytes, kSpanBytesBwd})
            *bytes = std::max(*bytes, plan_bytes(batch, seq_len, d_inner, plan_of(batch, seq_len, d_inner, io_dtype, span_bytes)));
    return HX_OK;
}

hx_status hx_gated_scan_bwd(const hx_gated_scan_bwd_args *a, void *stream) {
    HX_REQUIRE(a != nullptr, HX_ERR_INVALID_INPUT, "hx_gated_scan_bwd: args is NULL");
    const hx_status s = check_common("hx_gated_scan_bwd", a->batch, a->seq_len, a->d_inner, a->gate, a->io_dtype);
    if (s != HX_OK) return s;
    const int64_t chains = (int64_t)a->batch * a->d_inner;
    if (chains == 0) return HX_OK;
    HX_REQUIRE(a->seq_len == 0 || (a->x && a->g && a->dh && a->dx && a->dg && a->states), HX_ERR_INVALID_INPUT,
               "hx_gated_scan_bwd: x, g, dh, dx, dg and states must not be NULL");
    HX_REQUIRE(a->x_batch_stride >= 0 && a->x_row_stride >= 0 && a->g_batch_stride >= 0 && a->g_row_stride >= 0 &&
                   a->dh_batch_stride >= 0 && a->dh_row_stride >= 0 && a->dx_batch_stride >= 0 && a->dx_row_stride >= 0 &&
                   a->dg_batch_stride >= 0 && a->dg_row_stride >= 0,
               HX_ERR_INVALID_INPUT, "hx_gated_scan_bwd: negative stride");
    HX_REQUIRE(rows_apart(a->dx_batch_stride, a->dx_row_stride, a->batch, a->seq_len, a->d_inner) &&
                   rows_apart(a->dg_batch_stride, a->dg_row_stride, a->batch, a->seq_len, a->d_inner),
               HX_ERR_SHAPE_MISMATCH, "hx_gated_scan_bwd: rows of dx or dg overlap");
    const int piece = piece_of(dtype_size(a->io_dtype), {a->x, a->g, a->dh, a->dx, a->dg},
                               {a->x_batch_stride, a->x_row_stride, a->g_batch_stride, a->g_row_stride, a->dh_batch_stride,
                                a->dh_row_stride, a->dx_batch_stride, a->dx_row_stride, a->dg_batch_stride, a->dg_row_stride});
    Plan plan;
    const hx_status ps = choose_plan("hx_gated_scan_bwd", *a, kSpanBytesBwd, &plan);
    if (ps != HX_OK) return ps;
    auto view = [&](const void *at, int64_t bs, int64_t rs) { return rows_of(at, a->batch, bs, a->seq_len, rs, a->d_inner, dtype_size(a->io_dtype)); };
    const Operand outs[] = {{"dx", view(a->dx, a->dx_batch_stride, a->dx_row_stride)},
                            {"dg", view(a->dg, a->dg_batch_stride, a->dg_row_stride)},
                            {"dh0", dense_of(a->dh0, chains * 4)},
                            {"the workspace", dense_of(a->workspace, (int64_t)a->workspace_bytes)}};
    const Operand ins[] = {{"x", view(a->x, a->x_batch_stride, a->x_row_stride)},
                           {"g", view(a->g, a->g_batch_stride, a->g_row_stride)},
                           {"dh", view(a->dh, a->dh_batch_stride, a->dh_row_stride)},
                           {"states", dense_of(a->states, states_bytes(*a))},
                           {"dh_last", dense_of(a->dh_last, chains * 4)},
                           {"lengths", dense_of(a->lengths, (int64_t)a->batch * 4)}};
    const char *one, *other;
    HX_REQUIRE(!shared_operands(outs, ins, one, other), HX_ERR_INVALID_INPUT, "hx_gated_scan_bwd: %s and %s share memory", one, other);
    HX_GATED_LAUNCH(launch_bwd, a->gate, a->io_dtype, piece, *a, plan, (cudaStream_t)stream);
}

hx_status hx_gated_scan_step(const void *x, int64_t x_row_stride, const void *g, int64_t g_row_stride, const float *h, float *h_out,
                             void *y, int64_t y_row_stride, int32_t batch, int32_t d_inner, int32_t gate, int32_t io_dtype,
                             void *stream) {
    const hx_status s = check_common("hx_gated_scan_step", batch, 1, d_inner, gate, io_dtype);
    if (s != HX_OK) return s;
    const int64_t n = (int64_t)batch * d_inner;
    if (n == 0) return HX_OK;
    HX_REQUIRE(x && g && h && h_out && y, HX_ERR_INVALID_INPUT, "hx_gated_scan_step: NULL operand");
    HX_REQUIRE(x_row_stride >= 0 && g_row_stride >= 0, HX_ERR_INVALID_INPUT, "hx_gated_scan_step: negative stride");
    HX_REQUIRE(batch <= 1 || y_row_stride >= d_inner, HX_ERR_SHAPE_MISMATCH, "hx_gated_scan_step: rows of y overlap (stride %lld)",
               (long long)y_row_stride);
    const int64_t grid = ((int64_t)batch * ((d_inner + 1) / 2) + 127) / 128;
    HX_REQUIRE(grid <= 0x7fffffff, HX_ERR_INVALID_DIMENSION, "hx_gated_scan_step: batch * d_inner is too large for one launch");
    const size_t e = dtype_size(io_dtype);
    // a thread reads its elements of every operand before it writes them, so that an output in an input's very place is right
    auto same = [&](const void *in, int64_t stride) { return y == in && (stride == y_row_stride || batch == 1); };
    auto view = [&](const void *at, int64_t rs) { return rows_of(at, batch, rs, 1, 0, d_inner, e); };
    const Operand outs[] = {{"y", view(y, y_row_stride)}, {"h_out", dense_of(h_out, n * 4)}};
    const Operand ins[] = {{"x", view(same(x, x_row_stride) ? nullptr : x, x_row_stride)},
                           {"g", view(same(g, g_row_stride) ? nullptr : g, g_row_stride)}};
    const Operand state[] = {{"h", dense_of(h == h_out ? nullptr : h, n * 4)}};
    const char *one, *other;
    HX_REQUIRE(!shared_operands(outs, ins, one, other) && !shared_operands(outs, state, one, other), HX_ERR_INVALID_INPUT,
               "hx_gated_scan_step: %s and %s share memory", one, other);
    const uint64_t io = (uintptr_t)x | (uintptr_t)g | (uintptr_t)y | (uint64_t)(x_row_stride | g_row_stride | y_row_stride) * e;
    const bool pairs = d_inner % 2 == 0 && io % (2 * e) == 0 && ((uintptr_t)h | (uintptr_t)h_out) % 8 == 0;
#define HX_GATED_STEP(T, GATE)                                                                                               \
    gated_step_kernel<T, GATE><<<(unsigned)grid, 128, 0, (cudaStream_t)stream>>>(                                            \
        static_cast<const T *>(x), x_row_stride, static_cast<const T *>(g), g_row_stride, h, h_out, static_cast<T *>(y),     \
        y_row_stride, batch, d_inner, pairs)
    if (io_dtype == HX_BF16) {
        if (gate == HX_GATE_DECAY) HX_GATED_STEP(__nv_bfloat16, HX_GATE_DECAY);
        else HX_GATED_STEP(__nv_bfloat16, HX_GATE_SIGMOID);
    } else {
        if (gate == HX_GATE_DECAY) HX_GATED_STEP(float, HX_GATE_DECAY);
        else HX_GATED_STEP(float, HX_GATE_SIGMOID);
    }
#undef HX_GATED_STEP
    return check_launch("gated_step_kernel");
}

}  // extern "C"
