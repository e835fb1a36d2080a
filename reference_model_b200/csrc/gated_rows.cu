// Gated product with up to 32 rows (a decoder's tokens), 16-bit weights: each weight meets only those rows, so the operator reads both
// matrices once and nothing else counts.  Warp-level matrix instructions (m16n8k16) take sixteen output columns as their rows
// and eight rows of `a` as their columns; a 256-row tile of the CTA-pair kernel would be padding.
//
// A block takes 64 columns of the gate and the same 64 of the up projection, and a piece of K.  One thread feeds a ring of 128-row
// stages by TMA (128-byte swizzle); warps 0-3 multiply the gate's columns, 4-7 the up projection's, reading the weights through
// transposing matrix loads as they lie, K across rows.  Blocks of a cluster share K out while the grid leaves SMs idle.  The sums
// of a stage are added up in fp32 apart from the instruction's own; G and U meet in shared memory, in a fixed order, where the
// activation and the product are taken.
// One row, 4096 x 16384 bf16: 42 us for 268 MB, the rate of a plain copy (6.4 TB/s; DRAM 73 % of its peak).  2048 x 8192: 14.2 us for 67 MB that come from
// memory (six sets of operands in turn), 9.2 where a call finds much of them in L2 (the same operands again).  Small calls are latency: 4.3 us.
// Matrices whose rows are not multiples of sixteen bytes apart, which TMA cannot address, are read as they lie by warps of their own (SHIFT):
// 3248 x 3748 27.2 us from memory, 18.5 again, where 3752 columns take 12.1 and 10.5; a copy of both matrices first took 35 again.
#include <algorithm>
#include <cstring>
#include <cuda.h>

#include "ffn.h"
#include "ffn_math.cuh"
#include "ptx_sm100.cuh"

namespace tb200
{
namespace ffn
{
namespace
{

constexpr int kFewWarps     = 8;
constexpr int kFewLoaders   = 16;                      // warps that fetch matrices whose rows are not multiples of 16 bytes apart, in two groups
constexpr int few_threads(bool shift)
{
    return 32 * (kFewWarps + 1 + (shift ? kFewLoaders : 0));    // and the TMA warp
}
constexpr int kFewCols      = 64;                      // output columns of a block
constexpr int kFewStageK    = 128;
constexpr int kFewWBytes    = 2 * kFewStageK * kFewCols * 2;    // gate and up: 32 KB
constexpr int kFewMaxStages = 6;
constexpr int kFewRedLd     = 2 * kFewCols + 4;

struct FewParams
{
    CUtensorMap tmG, tmU;    // [NB][C][W], box 64 columns x 64 rows
    CUtensorMap tmX;         // [NB][H][C], box 64 x 8 NT
    const uint8_t* w[2];     // without tmG and tmU: the matrices, and their bytes
    int64_t w_bytes;
    int W, C, H;
    int act;
    int stages_total, splits, per_split, num_stages, stage_bytes;
    void* out;
    tb200_dtype out_dt;
    long long wait_limit;
    int* status;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <bool BF16>
__device__ __forceinline__ void few_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool BF16, int NT, bool SHIFT>
__global__ void __launch_bounds__(few_threads(SHIFT)) gated_rows_kernel(const __grid_constant__ FewParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[kFewMaxStages];                  // a stage's copies; SHIFT: its weights, made by the loaders
    __shared__ __align__(8) uint64_t bar_rows[SHIFT ? kFewMaxStages : 1];      // SHIFT: the copies of a's rows
    __shared__ __align__(8) uint64_t bar_empty[kFewMaxStages];
    __shared__ int gave_up;

    const int tid            = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank      = p.splits > 1 ? ptx::cluster_ctarank() : 0;
    const int col0           = (int)(blockIdx.x / (unsigned)p.splits) * kFewCols;
    const int row0           = blockIdx.y * 8 * NT, batch = blockIdx.z;
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const int first          = (int)rank * p.per_split;
    const int mine           = max(0, min(p.per_split, p.stages_total - first));

    if (tid == 0)
    {
        for (int s = 0; s < p.num_stages; s++)
        {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), SHIFT ? kFewLoaders / 2 : 1);
            if (SHIFT)
                ptx::mbar_init(ptx::smem_u32(&bar_rows[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), kFewWarps);
        }
        ptx::fence_barrier_init();
        if (!SHIFT)
        {
            ptx::prefetch_tmap(&p.tmG);
            ptx::prefetch_tmap(&p.tmU);
        }
        ptx::prefetch_tmap(&p.tmX);
        gave_up = 0;
        ptx::dep_launch_trigger();
    }
    __syncthreads();
    // everything a kernel before this one may have written is read behind this wait
    ptx::dep_launch_wait();

    float total[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
        total[j][0] = total[j][1] = total[j][2] = total[j][3] = 0.f;

    if (warp == kFewWarps)
    {
        if (lane == 0)
        {
            uint64_t* const bar_copies = SHIFT ? bar_rows : bar_full;
            bool ok = true;
            int i = 0, s = 0;
            uint32_t phase = 0;
            for (; i < mine; i++)
            {
                if (!ptx::mbar_wait_bounded(ptx::smem_u32(&bar_empty[s]), phase ^ 1u, p.wait_limit))
                {
                    ok = false;
                    break;
                }
                const uint32_t full = ptx::smem_u32(&bar_copies[s]);
                const uint32_t sW   = smem_base + (uint32_t)(s * p.stage_bytes), sX = sW + kFewWBytes;
                ptx::mbar_arrive_expect_tx(full, (uint32_t)(p.stage_bytes - (SHIFT ? kFewWBytes : 0)));
                const int k = (first + i) * kFewStageK;
#pragma unroll
                for (int j = 0; j < 2; j++)
                {
                    // 64 rows of K: the gate's columns, the up projection's, a's elements
                    if (!SHIFT)
                    {
                        ptx::tma_load_3d(sW + (uint32_t)(j * 8192), &p.tmG, full, col0, k + j * 64, batch);
                        ptx::tma_load_3d(sW + (uint32_t)(16384 + j * 8192), &p.tmU, full, col0, k + j * 64, batch);
                    }
                    ptx::tma_load_3d(sX + (uint32_t)(j * 8 * NT * 128), &p.tmX, full, k + j * 64, row0, batch);
                }
                if (++s == p.num_stages)
                {
                    s = 0;
                    phase ^= 1u;
                }
            }
            if (!ok)
                atomicOr(p.status, TB200_DEV_TIMEOUT);
            // Copies in flight land before the block leaves, whichever role may have given up on them.  (Nothing but copies counts on these
            // barriers, and a block whose roles all go on waits for them anyway.)
            for (int j = max(0, i - p.num_stages); j < i; j++)
                ptx::mbar_wait_bounded(ptx::smem_u32(&bar_copies[j % p.num_stages]), (uint32_t)(j / p.num_stages) & 1u, ptx::kDrainCycles);
        }
    }
    else if (SHIFT && warp > kFewWarps)
    {
        // Matrix rows that start anywhere: a thread makes sixteen bytes of a stage's row from the two aligned sixteens that hold them, eight such
        // pieces of every second stage, into the places where TMA would put them.
        const int loader = warp - kFewWarps - 1, group = loader >> 3, thread = (loader & 7) * 32 + lane;
        const int piece = thread & 7, row_in = thread >> 3, col = col0 + piece * 8;
        bool ok = true;
        int s = group;
        uint32_t phase = 0;
        for (int i = group; i < mine; i += 2)
        {
            ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(ptx::smem_u32(&bar_empty[s]), phase ^ 1u, p.wait_limit));
            if (!ok)
                break;
            const uint32_t sW = smem_base + (uint32_t)(s * p.stage_bytes);
#pragma unroll
            for (int m = 0; m < 2; m++)
            {
                uint4 lo[4], hi[4];
                int64_t at[4];
#pragma unroll
                for (int j = 0; j < 4; j++)
                {
                    const int k = (first + i) * kFewStageK + row_in + 32 * j;
                    at[j]       = k < p.C && col < p.W ? (((int64_t)batch * p.C + k) * p.W + col) * 2 : -1;
                    lo[j] = hi[j] = make_uint4(0, 0, 0, 0);
                    const int64_t aligned = at[j] & ~(int64_t)15;
                    if (at[j] >= 0 && aligned + 32 <= p.w_bytes)
                    {
                        lo[j] = *reinterpret_cast<const uint4*>(p.w[m] + aligned);
                        hi[j] = *reinterpret_cast<const uint4*>(p.w[m] + aligned + 16);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
                {
                    const int row = row_in + 32 * j;
                    uint4 v       = shifted_piece(lo[j], hi[j], (int)(at[j] & 15));
                    if (at[j] >= 0 && (at[j] & ~(int64_t)15) + 32 > p.w_bytes)
                    {
                        // the matrix's last elements
                        uint16_t e[8];
#pragma unroll
                        for (int c = 0; c < 8; c++)
                            e[c] = at[j] + 2 * c < p.w_bytes ? *reinterpret_cast<const uint16_t*>(p.w[m] + at[j] + 2 * c) : (uint16_t)0;
                        v = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
                    }
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sW + (uint32_t)(m * 16384 + row * 128 + ((piece ^ (row & 7)) << 4))), "r"(v.x),
                                 "r"(v.y), "r"(v.z), "r"(v.w)
                                 : "memory");
                }
            }
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive(ptx::smem_u32(&bar_full[s]));
            s += 2;
            if (s >= p.num_stages)
            {
                s -= p.num_stages;
                phase ^= 1u;
            }
        }
        if (!ok && lane == 0)
            atomicOr(p.status, TB200_DEV_TIMEOUT);
    }
    else
    {
        const int piece0 = (warp & 3) * 2;    // this warp's sixteen columns: two 16-byte pieces of a 128-byte row
        const int q = lane >> 3, r = lane & 7;
        const uint32_t aW = (uint32_t)((warp >> 2) * 16384 + ((q >> 1) * 8 + r) * 128) + (uint32_t)(((piece0 + (q & 1)) ^ r) << 4);
        bool ok = true;
        int s = 0;
        uint32_t phase = 0;
        for (int i = 0; i < mine; i++)
        {
            ok = ptx::mbar_wait_bounded(ptx::smem_u32(&bar_full[s]), phase, p.wait_limit) &&
                 (!SHIFT || ptx::mbar_wait_bounded(ptx::smem_u32(&bar_rows[s]), phase, p.wait_limit));
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            const uint32_t sW = smem_base + (uint32_t)(s * p.stage_bytes), sX = sW + kFewWBytes;
            float accum[NT][4];
#pragma unroll
            for (int j = 0; j < NT; j++)
                accum[j][0] = accum[j][1] = accum[j][2] = accum[j][3] = 0.f;
#pragma unroll
            for (int c = 0; c < 4; c++)    // 32 rows of K
            {
                uint32_t a0[4], a1[4];
                ldsm4t(sW + aW + (uint32_t)(c * 4096), a0);
                ldsm4t(sW + aW + (uint32_t)(c * 4096 + 2048), a1);
#pragma unroll
                for (int j = 0; j < NT; j++)
                {
                    uint32_t b[4];
                    ldsm4(sX + (uint32_t)((c >> 1) * 8 * NT * 128 + j * 1024 + r * 128) + (uint32_t)((((c & 1) * 4 + q) ^ r) << 4), b);
                    few_mma<BF16>(accum[j], a0, b[0], b[1]);
                    few_mma<BF16>(accum[j], a1, b[2], b[3]);
                }
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    total[j][e] += accum[j][e];
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive(ptx::smem_u32(&bar_empty[s]));
            if (++s == p.num_stages)
            {
                s = 0;
                phase ^= 1u;
            }
        }
        if (!ok && lane == 0)
        {
            atomicOr(p.status, TB200_DEV_TIMEOUT);
            gave_up = 1;
        }
    }

    // ---- sums to shared memory, over the ring (every copy has landed and been read, unless a wait gave up: then the results do
    // not count, and the ring is left alone)
    __syncthreads();
    float* const red     = reinterpret_cast<float*>(smem_raw + (smem_base - ptx::smem_u32(smem_raw)));
    const bool timed_out = gave_up != 0;
    if (warp < kFewWarps && !timed_out)
    {
        const int g = lane >> 2, t = lane & 3, c = warp * 16 + g;    // gate columns 0-63, up projection's 64-127
#pragma unroll
        for (int j = 0; j < NT; j++)
        {
            red[(j * 8 + 2 * t) * kFewRedLd + c]         = total[j][0];
            red[(j * 8 + 2 * t + 1) * kFewRedLd + c]     = total[j][1];
            red[(j * 8 + 2 * t) * kFewRedLd + c + 8]     = total[j][2];
            red[(j * 8 + 2 * t + 1) * kFewRedLd + c + 8] = total[j][3];
        }
    }
    if (p.splits > 1)
        ptx::cluster_sync();
    else
        __syncthreads();
    // a thread stays with its column; the cluster's blocks share the rows out
    const int rows = min(p.H - row0, 8 * NT), c = tid % kFewCols;
    constexpr int kStep = 32 * kFewWarps / kFewCols;
    for (int n = (int)rank * kStep + tid / kFewCols; n < rows && tid < 32 * kFewWarps && col0 + c < p.W && !timed_out; n += p.splits * kStep)
    {
        float v[2];
#pragma unroll
        for (int m = 0; m < 2; m++)
        {
            const float* at = red + n * kFewRedLd + m * kFewCols + c;
            float sum       = 0.f;
            if (p.splits > 1)
            {
                const uint32_t local = ptx::smem_u32(at);
                float x[8];    // all on their way before the first is added
#pragma unroll
                for (int r = 0; r < 8; r++)
                {
                    x[r] = 0.f;
                    if (r < p.splits)
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[r]) : "r"(ptx::map_to_cta(local, (uint32_t)r)) : "memory");
                }
#pragma unroll
                for (int r = 0; r < 8; r++)
                    sum += x[r];
            }
            else
                sum = *at;
            v[m] = sum;
        }
        store_fp(p.out, ((int64_t)batch * p.H + row0 + n) * p.W + col0 + c, p.out_dt, act_value(p.act, v[0]) * v[1]);
    }
    if (p.splits > 1)
        ptx::cluster_sync();    // nobody leaves while another block may still read its sums
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

tb200_status encode3d(tb200_ctx* ctx, CUtensorMap* m, const Matrix& x, bool bf16, uint32_t box_outer)
{
    const EncodeTiled enc = reinterpret_cast<EncodeTiled>(tensor_map_encode_fn());
    if (!enc)
        return fail(ctx, TB200_INTERNAL, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3]    = { (cuuint64_t)x.inner, (cuuint64_t)x.outer, (cuuint64_t)x.batches };
    const cuuint64_t strides[2] = { (cuuint64_t)x.pitch * 2, (cuuint64_t)x.pitch * (cuuint64_t)x.outer * 2 };
    const cuuint32_t box[3]     = { 64, box_outer, 1 };
    const cuuint32_t estr[3]    = { 1, 1, 1 };
    const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(x.data), dims, strides, box,
                           estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(ctx, TB200_INTERNAL, "tensor map of a gated product rejected (CUresult %d)", (int)r);
    return TB200_OK;
}

typedef void (*FewKern)(const FewParams);

template <bool BF16, bool SHIFT>
FewKern pick(int nt)
{
    return nt == 1 ? gated_rows_kernel<BF16, 1, SHIFT> : nt == 2 ? gated_rows_kernel<BF16, 2, SHIFT> : gated_rows_kernel<BF16, 4, SHIFT>;
}

}    // namespace

tb200_status gated_rows_launch(tb200_ctx* ctx, const PairProduct& q)
{
    FewParams p;
    memset(&p, 0, sizeof(p));
    const bool bf16 = q.dt == TB200_BF16;
    const int nt    = q.rows <= 8 ? 1 : q.rows <= 16 ? 2 : 4;
    const bool shift = q.b[0].pitch % 8 != 0;    // rows that TMA cannot address
    tb200_status st  = shift ? TB200_OK : encode3d(ctx, &p.tmG, q.b[0], bf16, 64);
    if (st == TB200_OK && !shift)
        st = encode3d(ctx, &p.tmU, q.b[1], bf16, 64);
    p.w[0]    = reinterpret_cast<const uint8_t*>(q.b[0].data);
    p.w[1]    = reinterpret_cast<const uint8_t*>(q.b[1].data);
    p.w_bytes = q.b[0].batches * q.b[0].outer * q.b[0].inner * 2;
    if (st == TB200_OK)
        st = encode3d(ctx, &p.tmX, q.a, bf16, (uint32_t)(8 * nt));
    if (st != TB200_OK)
        return st;
    p.W = q.cols; p.C = (int)q.K; p.H = q.rows; p.act = q.act; p.out = q.out[0]; p.out_dt = q.out_dt[0];
    p.wait_limit   = ctx->wait_limit_cycles;
    p.status       = ctx->d_status;
    p.stages_total = (p.C + kFewStageK - 1) / kFewStageK;
    p.stage_bytes  = kFewWBytes + nt * 8 * kFewStageK * 2;
    const int64_t tiles = (p.W + kFewCols - 1) / kFewCols, yb = (p.H + 8 * nt - 1) / (8 * nt);
    // K over a cluster while the blocks do not fill the SMs and a block keeps two stages
    p.splits = 1;
    while (p.splits < 8 && p.stages_total / (2 * p.splits) >= 2 && tiles * yb * q.NB * p.splits * (shift ? 2 : 1) < ctx->num_sms + (shift ? 1 : 0))
        p.splits *= 2;
    p.per_split       = (p.stages_total + p.splits - 1) / p.splits;
    p.num_stages      = std::max(2, std::min(std::min(kFewMaxStages, p.per_split), (shift ? 200 : 104) * 1024 / p.stage_bytes));
    if (shift)
        p.num_stages &= ~1;    // a group of loaders keeps to its stages
    const size_t red  = (size_t)8 * nt * kFewRedLd * sizeof(float);
    const size_t smem = std::max((size_t)p.num_stages * p.stage_bytes, red) + 1024;
    const FewKern kern = bf16 ? (shift ? pick<true, true>(nt) : pick<true, false>(nt)) : shift ? pick<false, true>(nt) : pick<false, false>(nt);
    st = raise_smem_limit(ctx, (shift ? 140 : 168) + nt / 2 * 2 + (bf16 ? 1 : 0), reinterpret_cast<const void*>(kern), (int)smem);
    if (st != TB200_OK)
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned)(tiles * p.splits), (unsigned)yb, (unsigned)q.NB);
    cfg.blockDim           = dim3((unsigned)few_threads(shift));
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
    return post_launch(ctx, "gated_rows_f16");
}

}    // namespace ffn
}    // namespace tb200
