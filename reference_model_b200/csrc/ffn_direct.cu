// Feed-forward operators with one thread per result: every type, size and alignment, plain stream order.  The kernel policy that
// forces CUDA-core kernels comes here.  Neighbouring threads take neighbouring columns; sums of 64 products in fp32 are
// added up in fp32, so that a sum's error grows with its length over 64.  What bounds it: the loads of each product (one row, 4-bit 8192 x 8192:
// 100 times the tiled kernels' time).
#include <algorithm>

#include "ffn.h"
#include "ffn_math.cuh"

namespace tb200
{
namespace ffn
{
namespace
{

constexpr int kDirectThreads = 256, kDirectRun = 64;

int direct_grid(const tb200_ctx* ctx, int64_t items)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>((items + kDirectThreads - 1) / kDirectThreads, (int64_t)ctx->num_sms * 16));
}

__device__ __forceinline__ float w4_dot(const W4Problem& q, const W4Mat& w, int64_t m, int col, bool& bad_zero)
{
    const uint8_t* row = w.data + (int64_t)col * w.pitch;
    float total        = 0.f;
    for (int64_t c0 = 0, g = 0; c0 < q.C; g++)
    {
        const int64_t c1 = min((int64_t)q.C, c0 + q.group);
        const int64_t at = g * q.W + col;
        const int z   = w.zero ? (int)w.zero[at] : 0;
        bad_zero |= z < -8 || z > 7;
        float s = 0.f;
        while (c0 < c1)
        {
            const int64_t run = min(c1, c0 + kDirectRun);
            float part    = 0.f;
            for (; c0 < run; c0++)
            {
                const int b = row[c0 >> 1], n = (c0 & 1) ? b >> 4 : b & 15;
                part += load_fp(q.a, m * q.C + c0, q.dt) * (float)(((n ^ 8) - 8) - z);
            }
            s += part;
        }
        total += load_fp(w.scale, at, w.scale_dt) * s;
    }
    return total;
}

__global__ void __launch_bounds__(kDirectThreads) w4_direct_kernel(const __grid_constant__ W4Problem q, int* status)
{
    const int64_t n = q.M * q.W;
    bool bad        = false;
    for (int64_t i = (int64_t)blockIdx.x * kDirectThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kDirectThreads)
    {
        const int64_t m = i / q.W;
        const int col   = (int)(i - m * q.W);
        float v         = w4_dot(q, q.w[0], m, col, bad);
        if (q.mats == 2)
            v = act_value(q.act, v) * w4_dot(q, q.w[1], m, col, bad);
        store_fp(q.out, i, q.out_dt, v);
    }
    if (bad)
        atomicOr(status, TB200_DEV_UNPREDICTABLE);
}

// The two projections of one output; backward: dG and dU, forward: the result.
__global__ void __launch_bounds__(kDirectThreads) gated_direct_kernel(const __grid_constant__ GatedProblem q, float* dg, float* du)
{
    const int64_t n = (int64_t)q.NB * q.H * q.W;
    for (int64_t i = (int64_t)blockIdx.x * kDirectThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kDirectThreads)
    {
        const int64_t row = i / q.W, batch = row / q.H;
        const int64_t b0  = batch * q.C * q.W + (i - row * q.W);
        float g = 0.f, u = 0.f;
        for (int64_t c0 = 0; c0 < q.C; c0 += kDirectRun)
        {
            float pg = 0.f, pu = 0.f;
            const int64_t c1 = min((int64_t)q.C, c0 + kDirectRun);
            for (int64_t c = c0; c < c1; c++)
            {
                const float x = load_fp(q.a, row * q.C + c, q.dt);
                pg += x * load_fp(q.gate, b0 + c * q.W, q.dt);
                pu += x * load_fp(q.up, b0 + c * q.W, q.dt);
            }
            g += pg;
            u += pu;
        }
        if (!dg)
        {
            store_fp(q.out, i, q.out_dt, act_value(q.act, g) * u);
            continue;
        }
        float value, slope;
        act_slope(q.act, g, value, slope);
        const float d = load_fp(q.dout, i, q.dt);
        dg[i]         = d * slope * u;    // (the slope is 1.13 at most: only the result itself can overflow)
        du[i]         = d * value;
    }
}

__global__ void __launch_bounds__(kDirectThreads) gated_grad_a_direct_kernel(const __grid_constant__ GatedProblem q, const float* dg, const float* du)
{
    const int64_t n = (int64_t)q.NB * q.H * q.C;
    for (int64_t i = (int64_t)blockIdx.x * kDirectThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kDirectThreads)
    {
        const int64_t row = i / q.C, batch = row / q.H;
        const int64_t b0  = (batch * q.C + (i - row * q.C)) * q.W;
        float total       = 0.f;
        for (int64_t w0 = 0; w0 < q.W; w0 += kDirectRun)
        {
            float part       = 0.f;
            const int64_t w1 = min((int64_t)q.W, w0 + kDirectRun);
            for (int64_t w = w0; w < w1; w++)
                part += dg[row * q.W + w] * load_fp(q.gate, b0 + w, q.dt) + du[row * q.W + w] * load_fp(q.up, b0 + w, q.dt);
            total += part;
        }
        store_fp(q.da, i, q.da_dt, total);
    }
}

__global__ void __launch_bounds__(kDirectThreads) gated_grad_b_direct_kernel(const __grid_constant__ GatedProblem q, const float* d, void* out,
                                                                             tb200_dtype out_dt)
{
    const int64_t n = (int64_t)q.NB * q.C * q.W;
    for (int64_t i = (int64_t)blockIdx.x * kDirectThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kDirectThreads)
    {
        const int64_t r = i / q.W, batch = r / q.C, c = r - batch * q.C, w = i - r * q.W;
        float total = 0.f;
        for (int64_t h0 = 0; h0 < q.H; h0 += kDirectRun)
        {
            float part       = 0.f;
            const int64_t h1 = min(q.H, h0 + kDirectRun);
            for (int64_t h = h0; h < h1; h++)
            {
                const int64_t row = batch * q.H + h;
                part += load_fp(q.a, row * q.C + c, q.dt) * d[row * q.W + w];
            }
            total += part;
        }
        store_fp(out, i, out_dt, total);
    }
}

}    // namespace

tb200_status w4_direct_launch(tb200_ctx* ctx, const W4Problem& q)
{
    timer_begin(ctx);
    w4_direct_kernel<<<direct_grid(ctx, q.M * q.W), kDirectThreads, 0, ctx->stream>>>(q, ctx->d_status);
    timer_end(ctx);
    return post_launch(ctx, q.mats == 2 ? "gated_w4_direct" : "matmul_w4_direct");
}

tb200_status gated_direct_launch(tb200_ctx* ctx, const GatedProblem& q)
{
    timer_begin(ctx);
    gated_direct_kernel<<<direct_grid(ctx, (int64_t)q.NB * q.H * q.W), kDirectThreads, 0, ctx->stream>>>(q, nullptr, nullptr);
    timer_end(ctx);
    return post_launch(ctx, "gated_direct");
}

tb200_status gated_backward_direct_launch(tb200_ctx* ctx, const GatedProblem& q, float* dg, float* du)
{
    timer_begin(ctx);
    int launches = 1;
    gated_direct_kernel<<<direct_grid(ctx, (int64_t)q.NB * q.H * q.W), kDirectThreads, 0, ctx->stream>>>(q, dg, du);
    if (q.da)
    {
        gated_grad_a_direct_kernel<<<direct_grid(ctx, (int64_t)q.NB * q.H * q.C), kDirectThreads, 0, ctx->stream>>>(q, dg, du);
        launches++;
    }
    for (int i = 0; i < 2; i++)
    {
        void* out = i ? q.dup : q.dgate;
        if (!out)
            continue;
        gated_grad_b_direct_kernel<<<direct_grid(ctx, (int64_t)q.NB * q.C * q.W), kDirectThreads, 0, ctx->stream>>>(q, i ? du : dg, out,
                                                                                                               i ? q.dup_dt : q.dgate_dt);
        launches++;
    }
    timer_end(ctx);
    return post_launch(ctx, "gated_backward_direct", launches);
}

}    // namespace ffn
}    // namespace tb200
