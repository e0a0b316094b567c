// Gated linear recurrence h_t = a_t h_{t-1} + b_t over [batch, seq_len, d_inner], its gradients, and its single-token step.
// One thread per (batch row, channel) walks the sequence; neighbouring lanes hold neighbouring channels.
#include "hx_common.cuh"

namespace hx {
namespace gated {

constexpr int kStateSteps = HX_GATED_SCAN_STATE_STEPS;

// a = sigmoid(g) and rest = 1 - a, both to full relative precision: exp is taken of -|g|, so it neither overflows nor cancels.
__device__ __forceinline__ void sigmoid_pair(float g, float &a, float &rest) {
    const float e = expf(-fabsf(g));
    const float big = 1.0f / (1.0f + e), small = e * big;
    a = g >= 0.f ? big : small;   // a NaN goes through as NaN
    rest = g >= 0.f ? small : big;
}

template <int GATE> __device__ __forceinline__ void decay_and_input(float g, float x, float &a, float &b) {
    if constexpr (GATE == HX_GATE_DECAY) {
        a = g;
        b = x;
    } else {
        float rest;
        sigmoid_pair(g, a, rest);
        b = rest * x;
    }
}

template <typename T, int GATE>
__global__ void __launch_bounds__(128) gated_scan_kernel(const hx_gated_scan_args p) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.batch * p.d_inner) return;
    const int b = (int)(i / p.d_inner), d = (int)(i % p.d_inner);
    const T *x = static_cast<const T *>(p.x) + b * p.x_batch_stride + d;
    const T *g = static_cast<const T *>(p.g) + b * p.g_batch_stride + d;
    T *out = static_cast<T *>(p.h) + b * p.h_batch_stride + d;
    const int len = p.lengths ? min(max(p.lengths[b], 0), p.seq_len) : p.seq_len;
    const int64_t tiles = (p.seq_len + (int64_t)kStateSteps - 1) / kStateSteps;
    float h = p.h0 ? p.h0[i] : 0.f;
    for (int t = 0; t < len; ++t) {
        if (p.states && t % kStateSteps == 0) p.states[(b * tiles + t / kStateSteps) * p.d_inner + d] = h;
        float a, in;
        decay_and_input<GATE>(ld_f32(g + t * p.g_row_stride), ld_f32(x + t * p.x_row_stride), a, in);
        h = fmaf(a, h, in);
        st_f32(out + t * p.h_row_stride, h);
    }
    for (int64_t t = len; t < p.seq_len; ++t) st_f32(out + t * p.h_row_stride, 0.f);
    if (p.h_last) p.h_last[i] = h;
}

template <typename T, int GATE>
__global__ void __launch_bounds__(128) gated_scan_bwd_kernel(const hx_gated_scan_bwd_args p) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.batch * p.d_inner) return;
    const int b = (int)(i / p.d_inner), d = (int)(i % p.d_inner);
    const T *x = static_cast<const T *>(p.x) + b * p.x_batch_stride + d;
    const T *g = static_cast<const T *>(p.g) + b * p.g_batch_stride + d;
    const T *dh = static_cast<const T *>(p.dh) + b * p.dh_batch_stride + d;
    T *dx = static_cast<T *>(p.dx) + b * p.dx_batch_stride + d;
    T *dg = static_cast<T *>(p.dg) + b * p.dg_batch_stride + d;
    const int len = p.lengths ? min(max(p.lengths[b], 0), p.seq_len) : p.seq_len;
    const int64_t tiles = (p.seq_len + (int64_t)kStateSteps - 1) / kStateSteps;
    for (int64_t t = len; t < p.seq_len; ++t) {
        st_f32(dx + t * p.dx_row_stride, 0.f);
        st_f32(dg + t * p.dg_row_stride, 0.f);
    }
    float e = p.dh_last ? p.dh_last[i] : 0.f;   // a_{t+1} delta_{t+1}
    float before[kStateSteps];
    for (int tile = (len + kStateSteps - 1) / kStateSteps - 1; tile >= 0; --tile) {
        const int t0 = tile * kStateSteps, n = min(kStateSteps, len - t0);
        float h = p.states[(b * tiles + tile) * p.d_inner + d];
        for (int k = 0; k < n; ++k) {
            before[k] = h;
            float a, in;
            decay_and_input<GATE>(ld_f32(g + (t0 + k) * p.g_row_stride), ld_f32(x + (t0 + k) * p.x_row_stride), a, in);
            h = fmaf(a, h, in);
        }
        for (int k = n - 1; k >= 0; --k) {
            const int64_t t = t0 + k;
            const float delta = ld_f32(dh + t * p.dh_row_stride) + e;
            const float gv = ld_f32(g + t * p.g_row_stride);
            if constexpr (GATE == HX_GATE_DECAY) {
                st_f32(dx + t * p.dx_row_stride, delta);
                st_f32(dg + t * p.dg_row_stride, delta * before[k]);
                e = gv * delta;
            } else {
                float a, rest;
                sigmoid_pair(gv, a, rest);
                st_f32(dx + t * p.dx_row_stride, delta * rest);
                st_f32(dg + t * p.dg_row_stride, delta * (before[k] - ld_f32(x + t * p.x_row_stride)) * a * rest);
                e = a * delta;
            }
        }
    }
    if (p.dh0) p.dh0[i] = e;
}

template <typename T, int GATE>
__global__ void __launch_bounds__(256)
gated_step_kernel(const T *x, int64_t x_stride, const T *g, int64_t g_stride, const float *h, float *h_out, T *y, int64_t y_stride,
                  int batch, int d_inner) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)batch * d_inner) return;
    const int b = (int)(i / d_inner), d = (int)(i % d_inner);
    float a, in;
    decay_and_input<GATE>(ld_f32(g + b * g_stride + d), ld_f32(x + b * x_stride + d), a, in);
    const float v = fmaf(a, h[i], in);
    h_out[i] = v;
    st_f32(y + b * y_stride + d, v);
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

}  // namespace gated
}  // namespace hx

using namespace hx;
using namespace hx::gated;

#define HX_GATED_LAUNCH(KERNEL, GATE, DTYPE, ...)                                                              \
    do {                                                                                                       \
        if ((DTYPE) == HX_BF16) {                                                                              \
            if ((GATE) == HX_GATE_DECAY) KERNEL<__nv_bfloat16, HX_GATE_DECAY> __VA_ARGS__;                     \
            else KERNEL<__nv_bfloat16, HX_GATE_SIGMOID> __VA_ARGS__;                                           \
        } else {                                                                                               \
            if ((GATE) == HX_GATE_DECAY) KERNEL<float, HX_GATE_DECAY> __VA_ARGS__;                             \
            else KERNEL<float, HX_GATE_SIGMOID> __VA_ARGS__;                                                   \
        }                                                                                                      \
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
    const dim3 grid((unsigned)((chains + 127) / 128));
    HX_GATED_LAUNCH(gated_scan_kernel, a->gate, a->io_dtype, <<<grid, 128, 0, (cudaStream_t)stream>>>(*a));
    return check_launch("gated_scan_kernel");
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
    const dim3 grid((unsigned)((chains + 127) / 128));
    HX_GATED_LAUNCH(gated_scan_bwd_kernel, a->gate, a->io_dtype, <<<grid, 128, 0, (cudaStream_t)stream>>>(*a));
    return check_launch("gated_scan_bwd_kernel");
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
    const unsigned grid = (unsigned)((n + 255) / 256);
    if (io_dtype == HX_BF16) {
        auto xp = static_cast<const __nv_bfloat16 *>(x), gp = static_cast<const __nv_bfloat16 *>(g);
        auto yp = static_cast<__nv_bfloat16 *>(y);
        if (gate == HX_GATE_DECAY)
            gated_step_kernel<__nv_bfloat16, HX_GATE_DECAY><<<grid, 256, 0, (cudaStream_t)stream>>>(xp, x_row_stride, gp, g_row_stride, h, h_out, yp, y_row_stride, batch, d_inner);
        else
            gated_step_kernel<__nv_bfloat16, HX_GATE_SIGMOID><<<grid, 256, 0, (cudaStream_t)stream>>>(xp, x_row_stride, gp, g_row_stride, h, h_out, yp, y_row_stride, batch, d_inner);
    } else {
        auto xp = static_cast<const float *>(x), gp = static_cast<const float *>(g);
        auto yp = static_cast<float *>(y);
        if (gate == HX_GATE_DECAY)
            gated_step_kernel<float, HX_GATE_DECAY><<<grid, 256, 0, (cudaStream_t)stream>>>(xp, x_row_stride, gp, g_row_stride, h, h_out, yp, y_row_stride, batch, d_inner);
        else
            gated_step_kernel<float, HX_GATE_SIGMOID><<<grid, 256, 0, (cudaStream_t)stream>>>(xp, x_row_stride, gp, g_row_stride, h, h_out, yp, y_row_stride, batch, d_inner);
    }
    return check_launch("gated_step_kernel");
}

}  // extern "C"
