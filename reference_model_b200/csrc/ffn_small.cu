// Copies and elementwise passes around the feed-forward products.  All are bound by the bytes they move.
#include <algorithm>

#include "ffn.h"
#include "ffn_math.cuh"

namespace tb200
{
namespace ffn
{
namespace
{

constexpr int kSmallThreads = 256;

int small_grid(const tb200_ctx* ctx, int64_t items)
{
    return (int)std::max<int64_t>(1, std::min<int64_t>((items + kSmallThreads - 1) / kSmallThreads, (int64_t)ctx->num_sms * 16));
}

// A thread writes eight elements; rows of any length start at any even address, so they are read one element at a time (neighbouring
// threads read neighbouring runs).
__global__ void __launch_bounds__(kSmallThreads) pitch_copy_kernel(const uint16_t* __restrict__ in, uint16_t* __restrict__ out, int64_t rows, int64_t inner,
                                                                   int64_t pitch)
{
    const int64_t runs = pitch / 8, n = rows * runs;
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kSmallThreads)
    {
        const int64_t r = i / runs, c = (i - r * runs) * 8;
        const uint16_t* s = in + r * inner + c;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
        {
            const uint32_t lo = c + 2 * j < inner ? s[2 * j] : 0, hi = c + 2 * j + 1 < inner ? s[2 * j + 1] : 0;
            w[j]              = lo | hi << 16;
        }
        *reinterpret_cast<uint4*>(out + r * pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// fp32 rows as three bf16 rows each: the leading eight bits of the significand, the next eight, and the rest; every part is cut off, not rounded, so
// that none overflows and the last is exact.  What is not finite goes into the first part alone.
__global__ void __launch_bounds__(kSmallThreads) split_rows_kernel(const float* __restrict__ in, uint16_t* __restrict__ out, int64_t rows, int64_t inner,
                                                                   int64_t pitch)
{
    const int64_t n = rows * inner;
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kSmallThreads)
    {
        const int64_t r = i / inner, c = i - r * inner;
        const float x        = in[i];
        const uint32_t bits  = __float_as_uint(x);
        const bool finite    = (bits & 0x7F800000u) != 0x7F800000u;
        const uint32_t first = (bits & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC00000u : bits & 0xFFFF0000u;
        const float rest     = finite ? x - __uint_as_float(first) : 0.f;
        const uint32_t mid   = __float_as_uint(rest) & 0xFFFF0000u;
        const uint32_t last  = __float_as_uint(rest - __uint_as_float(mid));
        uint16_t* o          = out + 3 * r * pitch + c;
        o[0]                 = (uint16_t)(first >> 16);
        o[pitch]             = (uint16_t)(mid >> 16);
        o[2 * pitch]         = (uint16_t)(last >> 16);
    }
}

// Rows of bytes that start anywhere; a thread writes sixteen.
__global__ void __launch_bounds__(kSmallThreads) byte_copy_kernel(const uint8_t* __restrict__ in, uint8_t* __restrict__ out, int64_t rows, int64_t inner,
                                                                  int64_t in_pitch, int64_t pitch)
{
    const int64_t runs = pitch / 16, n = rows * runs;
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kSmallThreads)
    {
        const int64_t r = i / runs, c = (i - r * runs) * 16;
        const uint8_t* s = in + r * in_pitch + c;
        uint32_t w[4]    = { 0, 0, 0, 0 };
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (c + j < inner)
                w[j >> 2] |= (uint32_t)s[j] << (8 * (j & 3));
        *reinterpret_cast<uint4*>(out + r * pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The values of a 4-bit matrix, a thread for 32 elements of a row (which share a group).  16 bits: rows [W][pitch], a value rounded once; fp32: [C][W],
// neighbouring threads on neighbouring columns.
template <bool F32>
__global__ void __launch_bounds__(kSmallThreads) w4_dense_kernel(const W4Mat w, int C, int W, int group, tb200_dtype dt, void* out, int64_t pitch, int* status)
{
    const int64_t runs = (C + 31) / 32, n = runs * W;
    bool bad = false;
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kSmallThreads)
    {
        const int64_t row = F32 ? i % W : i / runs, run = F32 ? i / W : i % runs;
        const int c0      = (int)(run * 32), count = min(32, C - c0);
        const int64_t at  = (int64_t)(c0 / group) * W + row;
        const float s     = load_fp(w.scale, at, w.scale_dt);
        const int z       = w.zero ? (int)w.zero[at] : 0;
        bad |= z < -8 || z > 7;
        const uint8_t* src = w.data + row * w.pitch + c0 / 2;
        uint32_t b[4]      = { 0, 0, 0, 0 };
        if (w.pitch % 16 == 0)
        {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            b[0] = v.x; b[1] = v.y; b[2] = v.z; b[3] = v.w;
        }
        else
        {
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (2 * j < count)
                    b[j >> 2] |= (uint32_t)src[j] << (8 * (j & 3));
        }
        if (F32)
        {
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (j < count)
                    reinterpret_cast<float*>(out)[(int64_t)(c0 + j) * W + row] = (float)((int)(((b[j >> 3] >> (4 * (j & 7))) & 15) ^ 8) - 8 - z) * s;
        }
        else
        {
            uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(out) + row * pitch + c0);
#pragma unroll
            for (int q = 0; q < 4; q++)
            {
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; j++)
                {
                    const int lo = (int)(((b[q] >> (8 * j)) & 15) ^ 8) - 8 - z, hi = (int)(((b[q] >> (8 * j + 4)) & 15) ^ 8) - 8 - z;
                    v[j] = pack2((float)lo * s, (float)hi * s, dt == TB200_BF16);
                }
                reinterpret_cast<uint4*>(o)[q] = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
    }
    if (bad)
        atomicOr(status, TB200_DEV_UNPREDICTABLE);
}

// fp32 gated product behind its two projections
__global__ void __launch_bounds__(kSmallThreads) gate_f32_kernel(const float* __restrict__ g, const float* __restrict__ u, float* __restrict__ out, int64_t n, int act)
{
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kSmallThreads)
        out[i] = act_value(act, g[i]) * u[i];
}

// ... and its gradients: dG and dU in place of G and U, and side by side [rows][2 W] for the product with both matrices (where asked for)
__global__ void __launch_bounds__(kSmallThreads) grad_f32_kernel(float* __restrict__ g, float* __restrict__ u, const float* __restrict__ d, float* __restrict__ both,
                                                                 int64_t rows, int W, int act)
{
    const int64_t n = rows * W;
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kSmallThreads)
    {
        float value, slope;
        act_slope(act, g[i], value, slope);
        const float dg = d[i] * u[i] * slope, du = d[i] * value;
        g[i]           = dg;
        u[i]           = du;
        if (both)
        {
            const int64_t r          = i / W, c = i - r * W;
            both[r * 2 * W + c]      = dg;
            both[r * 2 * W + W + c]  = du;
        }
    }
}

// [batches][R][C] fp32 to [batches][C][R], tiles of 32 x 32 through shared memory; batches `out_batch` elements apart in the result
__global__ void __launch_bounds__(256) transpose_f32_kernel(const float* __restrict__ in, float* __restrict__ out, int64_t R, int64_t C, int64_t out_batch,
                                                            int64_t tiles_r, int64_t tiles_c, int64_t num_tiles)
{
    __shared__ float t[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int64_t i = blockIdx.x; i < num_tiles; i += gridDim.x)
    {
        const int64_t b = i / (tiles_r * tiles_c), k = i - b * tiles_r * tiles_c, r0 = k / tiles_c * 32, c0 = k % tiles_c * 32;
        for (int j = y; j < 32; j += 8)
            if (r0 + j < R && c0 + x < C)
                t[j][x] = in[(b * R + r0 + j) * C + c0 + x];
        __syncthreads();
        for (int j = y; j < 32; j += 8)
            if (c0 + j < C && r0 + x < R)
                out[b * out_batch + (c0 + j) * R + r0 + x] = t[x][j];
        __syncthreads();
    }
}

}    // namespace

tb200_status split_rows_launch(tb200_ctx* ctx, const float* in, void* out, int64_t rows, int64_t inner, int64_t pitch)
{
    split_rows_kernel<<<small_grid(ctx, rows * inner), kSmallThreads, 0, ctx->stream>>>(in, reinterpret_cast<uint16_t*>(out), rows, inner, pitch);
    return post_launch(ctx, "split_rows");
}

tb200_status byte_copy_launch(tb200_ctx* ctx, const uint8_t* in, uint8_t* out, int64_t rows, int64_t inner, int64_t in_pitch, int64_t pitch)
{
    byte_copy_kernel<<<small_grid(ctx, rows * (pitch / 16)), kSmallThreads, 0, ctx->stream>>>(in, out, rows, inner, in_pitch, pitch);
    return post_launch(ctx, "byte_copy");
}

tb200_status w4_dense_launch(tb200_ctx* ctx, const W4Mat& w, int C, int W, int group, tb200_dtype dt, void* out, int64_t pitch)
{
    const int grid = small_grid(ctx, (int64_t)((C + 31) / 32) * W);
    if (dt == TB200_FP32)
        w4_dense_kernel<true><<<grid, kSmallThreads, 0, ctx->stream>>>(w, C, W, group, dt, out, pitch, ctx->d_status);
    else
        w4_dense_kernel<false><<<grid, kSmallThreads, 0, ctx->stream>>>(w, C, W, group, dt, out, pitch, ctx->d_status);
    return post_launch(ctx, "w4_dense");
}

tb200_status gate_f32_launch(tb200_ctx* ctx, const float* g, const float* u, float* out, int64_t n, int act)
{
    gate_f32_kernel<<<small_grid(ctx, n), kSmallThreads, 0, ctx->stream>>>(g, u, out, n, act);
    return post_launch(ctx, "gate_f32");
}

tb200_status grad_f32_launch(tb200_ctx* ctx, float* g, float* u, const float* d, float* both, int64_t rows, int W, int act)
{
    grad_f32_kernel<<<small_grid(ctx, rows * W), kSmallThreads, 0, ctx->stream>>>(g, u, d, both, rows, W, act);
    return post_launch(ctx, "grad_f32");
}

tb200_status transpose_f32_launch(tb200_ctx* ctx, const float* in, float* out, int64_t batches, int64_t R, int64_t C, int64_t out_batch)
{
    const int64_t tr = (R + 31) / 32, tc = (C + 31) / 32, n = batches * tr * tc;
    transpose_f32_kernel<<<(unsigned)std::min<int64_t>(n, (int64_t)ctx->num_sms * 8), 256, 0, ctx->stream>>>(in, out, R, C, out_batch, tr, tc, n);
    return post_launch(ctx, "transpose_f32");
}

tb200_status pitch_copy_launch(tb200_ctx* ctx, const void* in, void* out, int64_t rows, int64_t inner, int64_t pitch)
{
    pitch_copy_kernel<<<small_grid(ctx, rows * (pitch / 8)), kSmallThreads, 0, ctx->stream>>>(reinterpret_cast<const uint16_t*>(in),
                                                                                             reinterpret_cast<uint16_t*>(out), rows, inner, pitch);
    return post_launch(ctx, "pitch_copy");
}

}    // namespace ffn
}    // namespace tb200
