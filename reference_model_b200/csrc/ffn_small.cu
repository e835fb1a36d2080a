// Copies and elementwise passes around the feed-forward products.  All are bound by the bytes they move, small ones by their launch: each lets
// the next kernel in at its start and waits for the one before (fp32 434 x 176 x 176 backward: 43 -> 31 us with this and one launch for all transposes).
#include <algorithm>

#include "ffn.h"
#include "ffn_math.cuh"
#include "ptx_sm100.cuh"

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

// A launch that may start while the kernel before it drains (the kernel waits for it before it reads or writes).
template <typename K, typename... A>
cudaError_t launch_overlapped(tb200_ctx* ctx, K kernel, dim3 grid, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = grid;
    cfg.blockDim           = dim3(kSmallThreads);
    cfg.stream             = ctx->stream;
    cudaLaunchAttribute at[1];
    at[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs    = at;
    cfg.numAttrs = ctx->launch_overlap ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Sixteen bytes of a row that starts anywhere, in words of UNIT bytes, zeros behind its end
template <typename T>
__device__ __forceinline__ uint4 row_piece(const uint8_t* src, int64_t left)
{
    constexpr int kWords = 16 / (int)sizeof(T);
    T w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; i++)
        w[i] = (int64_t)(i * sizeof(T)) < left ? reinterpret_cast<const T*>(src)[i] : T(0);
    return *reinterpret_cast<const uint4*>(w);
}

// The same from any byte: the two aligned sixteens that hold it, shifted (two bytes at a time, copies ran at 2 TB/s)
__device__ __forceinline__ uint4 row_piece_shifted(const uint8_t* src, int64_t left)
{
    const uintptr_t at = reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15;
    const int by       = (int)(reinterpret_cast<uintptr_t>(src) & 15);
    const uint4 p      = shifted_piece(*reinterpret_cast<const uint4*>(at), *reinterpret_cast<const uint4*>(at + 16), by);
    uint32_t v[4]      = { p.x, p.y, p.z, p.w };
#pragma unroll
    for (int i = 0; i < 4; i++)
    {
        const int keep = (int)min((int64_t)4, left - 4 * i);    // bytes of the row
        v[i]           = keep >= 4 ? v[i] : keep <= 0 ? 0u : v[i] & ((1u << (8 * keep)) - 1u);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// All copies of a call in one launch, a thread for sixteen bytes of a result row.  Words as wide as rows and addresses allow.  Split rows: an fp32 row
// becomes three bf16 rows whose sum it is: the leading eight bits of the significand, the next eight, and the rest; every part is cut
// off, not rounded, so that none overflows and the last is exact.  What is not finite goes into the first part alone.
__global__ void __launch_bounds__(kSmallThreads) row_copies_kernel(const __grid_constant__ RowCopies q)
{
    ptx::dep_launch_trigger();
    ptx::dep_launch_wait();
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < q.items[q.n - 1]; i += (int64_t)gridDim.x * kSmallThreads)
    {
        int k = 0;
        while (i >= q.items[k])
            k++;
        const RowCopy& c  = q.copy[k];
        const int64_t at  = i - (k ? q.items[k - 1] : 0), runs = c.pitch / 16;
        const int64_t row = at / runs, byte = (at - row * runs) * 16;
        if (c.split)
        {
            // eight elements of the row and of its three parts
            const float* const src = reinterpret_cast<const float*>(c.in + row * c.in_pitch) + byte / 2;
            const int64_t left     = c.inner / 4 - byte / 2;
            uint16_t part[3][8];
#pragma unroll
            for (int e = 0; e < 8; e++)
            {
                const float x        = e < left ? src[e] : 0.f;
                const uint32_t bits  = __float_as_uint(x);
                const bool finite    = (bits & 0x7F800000u) != 0x7F800000u;
                const uint32_t first = (bits & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC00000u : bits & 0xFFFF0000u;
                const float rest     = finite ? x - __uint_as_float(first) : 0.f;
                const uint32_t mid   = __float_as_uint(rest) & 0xFFFF0000u;
                part[0][e]           = (uint16_t)(first >> 16);
                part[1][e]           = (uint16_t)(mid >> 16);
                part[2][e]           = (uint16_t)(__float_as_uint(rest - __uint_as_float(mid)) >> 16);
            }
#pragma unroll
            for (int e = 0; e < 3; e++)
                *reinterpret_cast<uint4*>(c.out + (3 * row + e) * c.pitch + byte) = *reinterpret_cast<const uint4*>(part[e]);
            continue;
        }
        const uint8_t* const src = c.in + row * c.in_pitch + byte;
        const int64_t left       = c.inner - byte;
        // both sixteens within the operand
        const uintptr_t first = reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15;
        const bool inside     = first >= reinterpret_cast<uintptr_t>(c.in) && first + 32 <= reinterpret_cast<uintptr_t>(c.in) + (uintptr_t)c.bytes;
        const uint4 v            = inside        ? row_piece_shifted(src, left)
                                   : c.word == 8 ? row_piece<uint64_t>(src, left)
                                   : c.word == 4 ? row_piece<uint32_t>(src, left)
                                   : c.word == 2 ? row_piece<uint16_t>(src, left)
                                                 : row_piece<uint8_t>(src, left);
        *reinterpret_cast<uint4*>(c.out + row * c.pitch + byte) = v;
    }
}

// The values of a 4-bit matrix in fp32, [C][W]: a thread for 32 elements of a row, neighbouring threads on neighbouring columns
__global__ void __launch_bounds__(kSmallThreads) w4_dense_32_kernel(const W4Mat w, int C, int W, int group, float* out, int* status)
{
    const int64_t runs = (C + 31) / 32, n = runs * W;
    bool bad = false;
    for (int64_t i = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kSmallThreads)
    {
        const int64_t row = i % W, run = i / W;
        const int c0      = (int)(run * 32), count = min(32, C - c0);
        const int64_t g   = c0 / group;
        const float s     = load_fp(w.scale, (int64_t)g * W + row, w.scale_dt);
        const int z       = w.zero ? (int)w.zero[(int64_t)g * W + row] : 0;
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
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (j < count)
                out[(int64_t)(c0 + j) * W + row] = (float)((int)(((b[j >> 3] >> (4 * (j & 7))) & 15) ^ 8) - 8 - z) * s;
    }
    if (bad)
        atomicOr(status, TB200_DEV_UNPREDICTABLE);
}

// fp32 gated product behind its two projections, four elements a thread where `n` allows
__global__ void __launch_bounds__(kSmallThreads) gate_f32_kernel(const float* g, const float* u, float* out, int64_t n, int act)
{
    ptx::dep_launch_trigger();
    ptx::dep_launch_wait();
    const int64_t first = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x, step = (int64_t)gridDim.x * kSmallThreads;
    if (n % 4 == 0)
    {
        for (int64_t i = first; i < n / 4; i += step)
        {
            const float4 x = reinterpret_cast<const float4*>(g)[i], y = reinterpret_cast<const float4*>(u)[i];
            reinterpret_cast<float4*>(out)[i] =
                make_float4(act_value(act, x.x) * y.x, act_value(act, x.y) * y.y, act_value(act, x.z) * y.z, act_value(act, x.w) * y.w);
        }
        return;
    }
    for (int64_t i = first; i < n; i += step)
        out[i] = act_value(act, g[i]) * u[i];
}

// ... and its gradients: dG and dU in place of G and U, and side by side [rows][2 W] for the product with both matrices (where asked for)
__global__ void __launch_bounds__(kSmallThreads) grad_f32_kernel(float* g, float* u, const float* d, float* both, int64_t rows, int W, int act)
{
    ptx::dep_launch_trigger();
    ptx::dep_launch_wait();
    const int64_t n = rows * W, first = (int64_t)blockIdx.x * kSmallThreads + threadIdx.x, step = (int64_t)gridDim.x * kSmallThreads;
    auto gradients = [&](float G, float U, float D, float& dg, float& du) {
        float value, slope;
        act_slope(act, G, value, slope);
        dg = D * slope * U;
        du = D * value;
    };
    if (W % 4 == 0)
    {
        for (int64_t i = first; i < n / 4; i += step)
        {
            const float4 x = reinterpret_cast<const float4*>(g)[i], y = reinterpret_cast<const float4*>(u)[i], z = reinterpret_cast<const float4*>(d)[i];
            float4 dg, du;
            gradients(x.x, y.x, z.x, dg.x, du.x);
            gradients(x.y, y.y, z.y, dg.y, du.y);
            gradients(x.z, y.z, z.z, dg.z, du.z);
            gradients(x.w, y.w, z.w, dg.w, du.w);
            reinterpret_cast<float4*>(g)[i] = dg;
            reinterpret_cast<float4*>(u)[i] = du;
            if (both)
            {
                const int64_t r = i / (W / 4), c = i - r * (W / 4);
                reinterpret_cast<float4*>(both)[r * 2 * (W / 4) + c]         = dg;
                reinterpret_cast<float4*>(both)[(r * 2 + 1) * (W / 4) + c] = du;
            }
        }
        return;
    }
    for (int64_t i = first; i < n; i += step)
    {
        float dg, du;
        gradients(g[i], u[i], d[i], dg, du);
        g[i] = dg;
        u[i] = du;
        if (both)
        {
            const int64_t r         = i / W, c = i - r * W;
            both[r * 2 * W + c]     = dg;
            both[r * 2 * W + W + c] = du;
        }
    }
}

// [batches][R][C] fp32 to [batches][C][R], tiles of 32 x 32 through shared memory, all transposes of a call in one launch
__global__ void __launch_bounds__(256) transposes_f32_kernel(const __grid_constant__ Transposes q)
{
    __shared__ float t[32][33];
    ptx::dep_launch_trigger();
    ptx::dep_launch_wait();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int64_t i = blockIdx.x; i < q.tiles[q.n - 1]; i += gridDim.x)
    {
        int job = 0;
        while (i >= q.tiles[job])
            job++;
        const Transpose& j   = q.job[job];
        const int64_t tile   = i - (job ? q.tiles[job - 1] : 0), tiles_c = (j.C + 31) / 32, per = (j.R + 31) / 32 * tiles_c;
        const int64_t b = tile / per, k = tile - b * per, r0 = k / tiles_c * 32, c0 = k % tiles_c * 32;
        for (int e = y; e < 32; e += 8)
            if (r0 + e < j.R && c0 + x < j.C)
                t[e][x] = j.in[(b * j.R + r0 + e) * j.C + c0 + x];
        __syncthreads();
        for (int e = y; e < 32; e += 8)
            if (c0 + e < j.C && r0 + x < j.R)
                j.out[b * j.out_batch + (c0 + e) * j.R + r0 + x] = t[x][e];
        __syncthreads();
    }
}

}    // namespace

void RowCopies::add(const void* in, void* out, int64_t rows, int64_t inner, int64_t in_pitch, int64_t pitch, bool split)
{
    RowCopy& c = copy[n];
    c.in       = reinterpret_cast<const uint8_t*>(in);
    c.out      = reinterpret_cast<uint8_t*>(out);
    c.inner    = inner;
    c.in_pitch = in_pitch;
    c.pitch    = pitch;
    c.split    = split ? 1 : 0;
    c.bytes    = rows ? (rows - 1) * in_pitch + inner : 0;
    // a word never reaches behind the row: its width divides the row's length too
    const uint64_t bits = (uint64_t)reinterpret_cast<uintptr_t>(in) | (uint64_t)in_pitch | (uint64_t)inner;
    c.word              = bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    items[n]            = (n ? items[n - 1] : 0) + rows * (pitch / 16);
    n++;
}

tb200_status row_copies_launch(tb200_ctx* ctx, const RowCopies& q)
{
    if (q.n == 0 || q.items[q.n - 1] == 0)
        return TB200_OK;
    const cudaError_t e = launch_overlapped(ctx, row_copies_kernel, dim3((unsigned)small_grid(ctx, q.items[q.n - 1])), q);
    if (e != cudaSuccess)
        return fail(ctx, TB200_INTERNAL, "launch of row_copies failed: %s", cudaGetErrorString(e));
    return post_launch(ctx, "row_copies");
}

tb200_status w4_dense_launch(tb200_ctx* ctx, const W4Mat* w, int mats, int C, int W, int group, void* const* out)
{
    for (int i = 0; i < mats; i++)
        w4_dense_32_kernel<<<small_grid(ctx, (int64_t)((C + 31) / 32) * W), kSmallThreads, 0, ctx->stream>>>(w[i], C, W, group, reinterpret_cast<float*>(out[i]),
                                                                                                         ctx->d_status);
    return post_launch(ctx, "w4_dense", mats);
}

tb200_status gate_f32_launch(tb200_ctx* ctx, const float* g, const float* u, float* out, int64_t n, int act)
{
    const cudaError_t e = launch_overlapped(ctx, gate_f32_kernel, dim3((unsigned)small_grid(ctx, (n + 3) / 4)), g, u, out, n, act);
    if (e != cudaSuccess)
        return fail(ctx, TB200_INTERNAL, "launch of gate_f32 failed: %s", cudaGetErrorString(e));
    return post_launch(ctx, "gate_f32");
}

tb200_status grad_f32_launch(tb200_ctx* ctx, float* g, float* u, const float* d, float* both, int64_t rows, int W, int act)
{
    const cudaError_t e = launch_overlapped(ctx, grad_f32_kernel, dim3((unsigned)small_grid(ctx, (rows * W + 3) / 4)), g, u, d, both, rows, W, act);
    if (e != cudaSuccess)
        return fail(ctx, TB200_INTERNAL, "launch of grad_f32 failed: %s", cudaGetErrorString(e));
    return post_launch(ctx, "grad_f32");
}

void Transposes::add(const float* in, float* out, int64_t batches, int64_t R, int64_t C, int64_t out_batch)
{
    job[n]   = { in, out, R, C, out_batch };
    tiles[n] = (n ? tiles[n - 1] : 0) + batches * ((R + 31) / 32) * ((C + 31) / 32);
    n++;
}

tb200_status transposes_f32_launch(tb200_ctx* ctx, const Transposes& q)
{
    const cudaError_t e = launch_overlapped(ctx, transposes_f32_kernel, dim3((unsigned)std::min<int64_t>(q.tiles[q.n - 1], (int64_t)ctx->num_sms * 8)), q);
    if (e != cudaSuccess)
        return fail(ctx, TB200_INTERNAL, "launch of transposes_f32 failed: %s", cudaGetErrorString(e));
    return post_launch(ctx, "transposes_f32");
}

}    // namespace ffn
}    // namespace tb200
