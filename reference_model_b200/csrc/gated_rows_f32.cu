// fp32 gated product of one row: a weight is used once, so the operator reads both matrices and nothing else counts.  Every product and sum
// is an IEEE fp32 operation.
//
// A block takes 128 columns of the gate and the same 128 of the up projection, a lane four of each; its eight warps take K's elements in turn,
// eight loads of a lane on their way together, four blocks to an SM (sixteen loads and two blocks: 4096 x 8192 56 us).  Blocks of a cluster
// share K out while all run at once.  Sums of warps, then of blocks, are added up in a fixed order.  4096 x 8192: 44 us, 6.1 TB/s, the rate of
// a plain copy (76 by the fp32 product's tiles and a pass over both projections); 1480 x 7328 17 us from memory, 15 again (31); 100 x 4000 4.5 us.  Two rows by
// the same code took 94 us, which leaves them to the tiles.
#include <algorithm>
#include <cstring>

#include "ffn.h"
#include "ffn_math.cuh"
#include "ptx_sm100.cuh"

namespace tb200
{
namespace ffn
{
namespace
{

constexpr int kF32Threads = 256, kF32Warps = 8, kF32Cols = 128, kF32Ahead = 4;    // elements of K whose weights are on their way

struct FewF32Params
{
    const float *a, *gate, *up;    // [NB][C], [NB][C][W]
    float* out;
    int C, W, act, splits, per_split;    // K of a block
};

// Four columns of row k: neighbours (VEC: 16 bytes), or every 32nd
template <bool VEC>
__device__ __forceinline__ void weights4(const float* row, int col0, int lane, int W, float (&v)[4])
{
    if (VEC)
    {
        const int c    = col0 + lane * 4;
        const float4 x = c < W ? *reinterpret_cast<const float4*>(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
    else
    {
#pragma unroll
        for (int j = 0; j < 4; j++)
        {
            const int c = col0 + lane + 32 * j;
            v[j]        = c < W ? row[c] : 0.f;
        }
    }
}

template <bool VEC>
__global__ void __launch_bounds__(kF32Threads, 4) gated_rows_f32_kernel(const __grid_constant__ FewF32Params p)
{
    extern __shared__ float sums[];    // [warps][2][128]; the block's own in the first warp's place
    ptx::dep_launch_trigger();
    ptx::dep_launch_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank    = p.splits > 1 ? (int)ptx::cluster_ctarank() : 0;
    const int col0    = (int)(blockIdx.x / (unsigned)p.splits) * kF32Cols;
    const int k_end   = min(p.C, (rank + 1) * p.per_split);
    const float* const a    = p.a + (int64_t)blockIdx.y * p.C;
    const float* const gate = p.gate + (int64_t)blockIdx.y * p.C * p.W;
    const float* const up   = p.up + (int64_t)blockIdx.y * p.C * p.W;
    float total[2][4] = {};
    for (int k0 = rank * p.per_split + warp; k0 < k_end; k0 += kF32Warps * kF32Ahead)
    {
        float g[kF32Ahead][4], u[kF32Ahead][4], x[kF32Ahead];
#pragma unroll
        for (int i = 0; i < kF32Ahead; i++)
        {
            const int64_t k = min(k0 + i * kF32Warps, k_end - 1);
            weights4<VEC>(gate + k * p.W, col0, lane, p.W, g[i]);
            weights4<VEC>(up + k * p.W, col0, lane, p.W, u[i]);
            x[i] = a[k];
        }
#pragma unroll
        for (int i = 0; i < kF32Ahead; i++)
        {
            if (k0 + i * kF32Warps >= k_end)
                break;
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                total[0][j] = fmaf(x[i], g[i][j], total[0][j]);
                total[1][j] = fmaf(x[i], u[i][j], total[1][j]);
            }
        }
    }
    constexpr int kSums = 2 * kF32Cols;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            sums[warp * kSums + m * kF32Cols + (VEC ? lane * 4 + j : lane + 32 * j)] = total[m][j];
    __syncthreads();
    for (int e = tid; e < kSums; e += kF32Threads)
    {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kF32Warps; w++)
            v += sums[w * kSums + e];
        sums[e] = v;
    }
    if (p.splits > 1)
        ptx::cluster_sync();
    else
        __syncthreads();
    for (int c = rank * kF32Threads + tid; c < kF32Cols && col0 + c < p.W; c += p.splits * kF32Threads)
    {
        float v[2];
#pragma unroll
        for (int m = 0; m < 2; m++)
        {
            const float* const at = sums + m * kF32Cols + c;
            v[m]                  = *at;
            if (p.splits > 1)
            {
                float x[8];
#pragma unroll
                for (int s = 0; s < 8; s++)
                {
                    x[s] = 0.f;
                    if (s < p.splits)
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[s]) : "r"(ptx::map_to_cta(ptx::smem_u32(at), (uint32_t)s)) : "memory");
                }
                v[m] = 0.f;
#pragma unroll
                for (int s = 0; s < 8; s++)
                    v[m] += x[s];
            }
        }
        p.out[(int64_t)blockIdx.y * p.W + col0 + c] = act_value(p.act, v[0]) * v[1];
    }
    if (p.splits > 1)
        ptx::cluster_sync();    // nobody leaves while another block may still read its sums
}

typedef void (*FewF32Kern)(const FewF32Params);

}    // namespace

tb200_status gated_rows_f32_launch(tb200_ctx* ctx, const GatedProblem& q)
{
    FewF32Params p;
    memset(&p, 0, sizeof(p));
    p.a    = reinterpret_cast<const float*>(q.a);
    p.gate = reinterpret_cast<const float*>(q.gate);
    p.up   = reinterpret_cast<const float*>(q.up);
    p.out  = reinterpret_cast<float*>(q.out);
    p.C = q.C; p.W = q.W; p.act = q.act;
    const int64_t tiles = (p.W + kF32Cols - 1) / kF32Cols;
    // K over a cluster while all blocks run at once (four to an SM, less what clusters leave) and a warp keeps two batches of loads
    p.splits = 1;
    while (p.splits < 8 && p.C >= 4 * p.splits * kF32Warps * kF32Ahead && tiles * q.NB * p.splits * 2 <= ctx->num_sms * 7 / 2)
        p.splits *= 2;
    p.per_split           = (p.C + p.splits - 1) / p.splits;
    const size_t smem     = (size_t)kF32Warps * 2 * kF32Cols * sizeof(float);
    const bool vec        = p.W % 4 == 0;
    const FewF32Kern kern = vec ? gated_rows_f32_kernel<true> : gated_rows_f32_kernel<false>;
    const tb200_status st = raise_smem_limit(ctx, 146 + (vec ? 1 : 0), reinterpret_cast<const void*>(kern), (int)smem);
    if (st != TB200_OK)
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned)(tiles * p.splits), (unsigned)q.NB);
    cfg.blockDim           = dim3(kF32Threads);
    cfg.dynamicSmemBytes   = smem;
    cfg.stream             = ctx->stream;
    cudaLaunchAttribute at[2];
    at[0].id               = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs    = at;
    cfg.numAttrs = ctx->launch_overlap ? 2 : 1;
    timer_begin(ctx);
    const cudaError_t le = cudaLaunchKernelEx(&cfg, kern, p);
    timer_end(ctx);
    if (le != cudaSuccess)
        return fail(ctx, TB200_INTERNAL, "launch of a gated product failed: %s", cudaGetErrorString(le));
    return post_launch(ctx, "gated_rows_f32");
}

}    // namespace ffn
}    // namespace tb200
