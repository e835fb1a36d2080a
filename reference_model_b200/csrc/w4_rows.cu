// Products with 4-bit weights, up to 64 rows: the weights are read once, straight from their bytes, and multiplied on the warp-level
// matrix instruction (m16n8k16) with the output's columns as its sixteen rows and eight rows of `a` as its columns.  A 128-row
// tensor-core tile would be padding, and CUDA cores cannot keep up: at the memory's rate an SM receives 46 weights a clock, which
// leaves 2.8 lane instructions for each.
//
// q - z (element minus zero point) is a whole number of at most 15, exact in fp16 and bf16; products of those with a's elements are exact in fp32,
// where the instruction adds them.  The scale multiplies the fp32 sum of a group: no weight is ever rounded.  fp32 rows go as three
// bf16 rows each (24 bits taken apart), whose results are added at the end.
//
// A nibble becomes a number by one bit operation and one subtraction for two of them: (word & 000F000F) ^ 43084308 is the bf16 pair
// 128 + 8 + q (fp16: 1024 + 8 + q from 64086408), minus 136 + z.  A word holds eight elements of K and the instruction does not mind the order
// of K, so word t of a 32-element run feeds thread t of a quad twice; a's elements are paired to match ((0,4), (1,5), ...) by
// byte permutes of one 16-byte read.
//
// A block takes 128 matrix rows (64 of each for the gated product) and a piece of K; eight warps take 16 rows each and all of the piece, one
// thread feeds a ring of 256-element stages by TMA (128-byte swizzle: both operands are read from shared memory without bank
// conflicts).  Blocks of a cluster share K out while the grid does not fill the SMs; their sums meet in shared memory, in order.
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

constexpr int kRowsWarps   = 8;
constexpr int kRowsThreads = 32 * (kRowsWarps + 1);    // and the TMA warp
constexpr int kRowsTile    = 128;                      // matrix rows of a block
constexpr int kRowsStageK  = 256;                      // elements of K in a stage: 128 bytes of weights a row
constexpr int kRowsWBytes  = kRowsTile * 128;
constexpr int kRowsGroups  = 32;                       // groups whose scales a block holds at a time
constexpr int kRowsMaxStages = 6;
constexpr int kRowsRedLd   = kRowsTile + 4;            // row pitch of the sums in shared memory: a warp's stores meet 32 banks

struct RowsParams
{
    CUtensorMap tmW0, tmW1;    // bytes [W][pitch], box 128 x 128 (gated: 128 x 64 of each)
    CUtensorMap tmX;           // [rows][C] 16-bit, box 64 x 8 NT
    const void* scale[2];
    const int8_t* zero[2];
    tb200_dtype scale_dt[2];
    int W, C, rows;            // rows of `a`
    int parts;                 // 16-bit rows that make a row of `a`: 1, or 3 for fp32
    int group, act;
    int stages_total;          // stages of K
    int splits, per_split;     // blocks that share K, stages of each
    int num_stages, stage_bytes;
    int super;                 // stages whose groups' scales fit kRowsGroups
    void* out;
    tb200_dtype out_dt;
    long long wait_limit;
    int* status;
};

template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight elements to four pairs (0,4), (1,5), (2,6), (3,7), minus their zero point; `base` holds 136 + z (fp16: 1032 + z) twice.
template <bool BF16>
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t base, uint32_t (&p)[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++)
    {
        const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) ^ (BF16 ? 0x43084308u : 0x64086408u);
        if (BF16)
        {
            const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&base));
            p[i]                   = *reinterpret_cast<const uint32_t*>(&d);
        }
        else
        {
            const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&base));
            p[i]            = *reinterpret_cast<const uint32_t*>(&d);
        }
    }
}

__device__ __forceinline__ uint4 lds128(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

template <bool BF16, int NT, int MATS>
__global__ void __launch_bounds__(kRowsThreads) w4_rows_kernel(const __grid_constant__ RowsParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[kRowsMaxStages];
    __shared__ __align__(8) uint64_t bar_empty[kRowsMaxStages];
    __shared__ float scales[kRowsGroups][kRowsTile];
    __shared__ uint32_t bases[kRowsGroups][kRowsTile];
    __shared__ int gave_up;

    constexpr int kPer       = kRowsTile / MATS;    // columns of the output
    const int tid            = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank      = p.splits > 1 ? ptx::cluster_ctarank() : 0;
    const int tile           = (int)(blockIdx.x / (unsigned)p.splits);
    const int col0           = tile * kPer;
    const int x0             = blockIdx.y * 8 * NT;    // first 16-bit row
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const int first          = (int)rank * p.per_split;
    const int mine           = max(0, min(p.per_split, p.stages_total - first));

    if (tid == 0)
    {
        for (int s = 0; s < p.num_stages; s++)
        {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), kRowsWarps);
        }
        ptx::fence_barrier_init();
        ptx::prefetch_tmap(&p.tmW0);
        ptx::prefetch_tmap(&p.tmX);
        if (MATS == 2)
            ptx::prefetch_tmap(&p.tmW1);
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

    if (warp == kRowsWarps)
    {
        if (lane == 0)
        {
            bool ok = true;
            int i   = 0;
            for (; i < mine; i++)
            {
                const int s = i % p.num_stages;
                if (!ptx::mbar_wait_bounded(ptx::smem_u32(&bar_empty[s]), ((uint32_t)(i / p.num_stages) & 1u) ^ 1u, p.wait_limit))
                {
                    ok = false;
                    break;
                }
                const uint32_t full = ptx::smem_u32(&bar_full[s]);
                const uint32_t sW   = smem_base + (uint32_t)(s * p.stage_bytes), sX = sW + kRowsWBytes;
                ptx::mbar_arrive_expect_tx(full, (uint32_t)p.stage_bytes);
                const int b = (first + i) * 128, k = (first + i) * kRowsStageK;
                ptx::tma_load_2d(sW, &p.tmW0, full, b, col0);
                if (MATS == 2)
                    ptx::tma_load_2d(sW + kPer * 128, &p.tmW1, full, b, col0);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    ptx::tma_load_2d(sX + (uint32_t)(j * 8 * NT * 128), &p.tmX, full, k + j * 64, x0);
            }
            if (!ok)
            {
                atomicOr(p.status, TB200_DEV_TIMEOUT);
                // copies in flight land before the block leaves
                for (int j = max(0, i - p.num_stages); j < i; j++)
                    ptx::mbar_wait_bounded(ptx::smem_u32(&bar_full[j % p.num_stages]), (uint32_t)(j / p.num_stages) & 1u, p.wait_limit);
            }
        }
    }
    else
    {
        const int g = lane >> 2, t = lane & 3;
        const int wrow = warp * 16 + g;    // and wrow + 8
        // column n of the instruction is row perm(n) of the tile of eight: neighbouring lanes' reads then meet different banks
        const int xr = (g >> 1) + (g & 1) * 4;
        float accum[NT][4];
#pragma unroll
        for (int j = 0; j < NT; j++)
            accum[j][0] = accum[j][1] = accum[j][2] = accum[j][3] = 0.f;
        bool ok       = true;
        bool bad_zero = false;
        int next_load = 0;    // stage at which the next batch of scales is due
        int g0        = 0;    // first group held
        int gi        = 0;    // the current run's group, counted from g0
        int left      = 0;    // elements until its end
        float s_lo = 0.f, s_hi = 0.f;
        uint32_t b_lo = 0, b_hi = 0;
        for (int i = 0; i < mine; i++)
        {
            const int k0 = (first + i) * kRowsStageK;
            if (i == next_load)
            {
                // scales and zero points of the next `super` stages; nobody may still read the ones before
                ptx::named_barrier_and(1, 32 * kRowsWarps, true);
                g0               = k0 / p.group;
                const int kend   = min(p.C, (first + min(mine - i, p.super) + i) * kRowsStageK);
                const int ngroup = kend > k0 ? (kend - 1) / p.group - g0 + 1 : 0;
                for (int e = tid; e < ngroup * kRowsTile; e += 32 * kRowsWarps)
                {
                    const int gg = e / kRowsTile, r = e % kRowsTile;
                    const int mat = MATS == 2 ? r / kPer : 0, col = col0 + (MATS == 2 ? r % kPer : r);
                    float s = 0.f;
                    int z   = 0;
                    if (col < p.W)
                    {
                        const int64_t at = (int64_t)(g0 + gg) * p.W + col;
                        s                = load_fp(p.scale[mat], at, p.scale_dt[mat]);
                        z                = p.zero[mat] ? (int)p.zero[mat][at] : 0;
                        if (z < -8 || z > 7)
                        {
                            bad_zero = true;
                            z        = 0;
                        }
                    }
                    scales[gg][r] = s;
                    bases[gg][r]  = BF16 ? pack2((float)(136 + z), (float)(136 + z), true) : pack2((float)(1032 + z), (float)(1032 + z), false);
                }
                next_load += p.super;
                ptx::named_barrier_and(1, 32 * kRowsWarps, true);
                gi   = 0;
                left = (int)((int64_t)(g0 + 1) * p.group - k0);
                s_lo = scales[0][wrow];
                s_hi = scales[0][wrow + 8];
                b_lo = bases[0][wrow];
                b_hi = bases[0][wrow + 8];
            }
            const int s = i % p.num_stages;
            if (ok)
                ok = ptx::mbar_wait_bounded(ptx::smem_u32(&bar_full[s]), (uint32_t)(i / p.num_stages) & 1u, p.wait_limit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                continue;    // the barriers around the scales are still met
            const uint32_t sW = smem_base + (uint32_t)(s * p.stage_bytes), sX = sW + kRowsWBytes;
            const uint32_t aW = sW + (uint32_t)(wrow * 128 + t * 4), swz = (uint32_t)(wrow & 7) << 4;
            const uint32_t aX = sX + (uint32_t)(xr * 128), xswz = (uint32_t)(xr & 7) << 4;
            const int runs    = min(8, (p.C - k0 + 31) / 32);
#pragma unroll
            for (int c = 0; c < 8; c++)
            {
                if (c < runs)
                {
                    const uint32_t w_lo = lds32(aW + (((uint32_t)c << 4) ^ swz)), w_hi = lds32(aW + 1024 + (((uint32_t)c << 4) ^ swz));
                    uint32_t lo[4], hi[4];
                    unpack8<BF16>(w_lo, b_lo, lo);
                    unpack8<BF16>(w_hi, b_hi, hi);
#pragma unroll
                    for (int j = 0; j < NT; j++)
                    {
                        const uint4 x = lds128(aX + (uint32_t)((c >> 1) * 8 * NT * 128 + j * 1024) + ((uint32_t)(((c & 1) * 4 + t) << 4) ^ xswz));
                        mma<BF16>(accum[j], lo[0], hi[0], lo[1], hi[1], __byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632));
                        mma<BF16>(accum[j], lo[2], hi[2], lo[3], hi[3], __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
                    }
                    left -= 32;
                    if (left <= 0)
                    {
                        // end of a group: its sum under its scale
#pragma unroll
                        for (int j = 0; j < NT; j++)
                        {
                            total[j][0] = fmaf(s_lo, accum[j][0], total[j][0]);
                            total[j][1] = fmaf(s_lo, accum[j][1], total[j][1]);
                            total[j][2] = fmaf(s_hi, accum[j][2], total[j][2]);
                            total[j][3] = fmaf(s_hi, accum[j][3], total[j][3]);
                            accum[j][0] = accum[j][1] = accum[j][2] = accum[j][3] = 0.f;
                        }
                        left = p.group;
                        gi   = min(gi + 1, kRowsGroups - 1);
                        s_lo = scales[gi][wrow];
                        s_hi = scales[gi][wrow + 8];
                        b_lo = bases[gi][wrow];
                        b_hi = bases[gi][wrow + 8];
                    }
                }
            }
            if ((i + 1 == next_load || i + 1 == mine) && left < p.group)
            {
                // a group that the next batch of scales, another block or nobody continues
#pragma unroll
                for (int j = 0; j < NT; j++)
                {
                    total[j][0] = fmaf(s_lo, accum[j][0], total[j][0]);
                    total[j][1] = fmaf(s_lo, accum[j][1], total[j][1]);
                    total[j][2] = fmaf(s_hi, accum[j][2], total[j][2]);
                    total[j][3] = fmaf(s_hi, accum[j][3], total[j][3]);
                    accum[j][0] = accum[j][1] = accum[j][2] = accum[j][3] = 0.f;
                }
            }
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive(ptx::smem_u32(&bar_empty[s]));
        }
        if (!ok && lane == 0)
        {
            atomicOr(p.status, TB200_DEV_TIMEOUT);
            gave_up = 1;
        }
        if (bad_zero)
            atomicOr(p.status, TB200_DEV_UNPREDICTABLE);
    }

    // ---- the block's sums to shared memory, over the ring (every copy has landed and been read, unless a wait gave up: then
    // the results do not count, and the ring is left alone)
    __syncthreads();
    float* const red     = reinterpret_cast<float*>(smem_raw + (smem_base - ptx::smem_u32(smem_raw)));
    const bool timed_out = gave_up != 0;
    if (warp < kRowsWarps && !timed_out)
    {
        const int g = lane >> 2, t = lane & 3, r = warp * 16 + g;
#pragma unroll
        for (int j = 0; j < NT; j++)
        {
            // instruction columns 2t and 2t + 1 are rows t and t + 4 of the tile of eight
            red[(j * 8 + t) * kRowsRedLd + r]         = total[j][0];
            red[(j * 8 + t + 4) * kRowsRedLd + r]     = total[j][1];
            red[(j * 8 + t) * kRowsRedLd + r + 8]     = total[j][2];
            red[(j * 8 + t + 4) * kRowsRedLd + r + 8] = total[j][3];
        }
    }
    if (p.splits > 1)
        ptx::cluster_sync();
    else
        __syncthreads();
    // results: row n of the block's (parts added), output column c; the cluster's blocks share them out
    const int first_row = x0 / p.parts;
    const int nrows     = min(p.rows - first_row, 8 * NT / p.parts);
    const int items     = nrows * kPer;
    for (int e = (int)rank * kRowsThreads + tid; e < items && !timed_out; e += p.splits * kRowsThreads)
    {
        const int n = e / kPer, c = e % kPer;
        if (col0 + c >= p.W)
            continue;
        float v[MATS];
#pragma unroll
        for (int m = 0; m < MATS; m++)
        {
            float sum = 0.f;
            for (int part = p.parts - 1; part >= 0; part--)
            {
                const float* at = red + (n * p.parts + part) * kRowsRedLd + m * kPer + c;
                if (p.splits > 1)
                {
                    const uint32_t local = ptx::smem_u32(at);
                    for (int r = 0; r < p.splits; r++)
                    {
                        float x;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(ptx::map_to_cta(local, (uint32_t)r)) : "memory");
                        sum += x;
                    }
                }
                else
                    sum += *at;
            }
            v[m] = sum;
        }
        const float y = MATS == 2 ? act_value(p.act, v[0]) * v[MATS - 1] : v[0];
        store_fp(p.out, (int64_t)(first_row + n) * p.W + col0 + c, p.out_dt, y);
    }
    if (p.splits > 1)
        ptx::cluster_sync();    // nobody leaves while another block may still read its sums
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

tb200_status encode2d(tb200_ctx* ctx, CUtensorMap* m, CUtensorMapDataType dt, size_t es, const void* data, int64_t inner, int64_t outer, int64_t pitch,
                      uint32_t box_inner, uint32_t box_outer)
{
    const EncodeTiled enc = reinterpret_cast<EncodeTiled>(tensor_map_encode_fn());
    if (!enc)
        return fail(ctx, TB200_INTERNAL, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2]    = { (cuuint64_t)inner, (cuuint64_t)outer };
    const cuuint64_t strides[1] = { (cuuint64_t)pitch * es };
    const cuuint32_t box[2]     = { box_inner, box_outer };
    const cuuint32_t estr[2]    = { 1, 1 };
    const CUresult r = enc(m, dt, 2, const_cast<void*>(data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(ctx, TB200_INTERNAL, "tensor map of a 4-bit product rejected (CUresult %d)", (int)r);
    return TB200_OK;
}

typedef void (*RowsKern)(const RowsParams);

template <bool BF16, int MATS>
RowsKern pick(int nt)
{
    return nt == 1 ? w4_rows_kernel<BF16, 1, MATS> : nt == 2 ? w4_rows_kernel<BF16, 2, MATS> : nt == 3 ? w4_rows_kernel<BF16, 3, MATS>
           : nt == 4 ? w4_rows_kernel<BF16, 4, MATS>                                                   : w4_rows_kernel<BF16, 8, MATS>;
}

}    // namespace

// x: the rows in 16 bits (bf16 parts of fp32 rows), `x_pitch` elements apart, 16-byte aligned; the weights' pitch is a multiple of 16.
tb200_status w4_rows_launch(tb200_ctx* ctx, const W4Problem& q, const void* x, int64_t x_pitch, int parts, bool bf16)
{
    RowsParams p;
    memset(&p, 0, sizeof(p));
    const int xrows = (int)q.M * parts;
    int nt          = (std::min(xrows, 64) + 7) / 8;
    if (parts == 3)
        nt = nt == 1 ? 1 : 3;    // whole rows of `a` to a block: one tile holds two, three tiles hold eight
    else
        nt = nt <= 4 ? nt : 8;
    const int rows_block = parts == 3 ? (nt == 1 ? 2 : 8) : 8 * nt;
    const int kPer       = kRowsTile / q.mats;
    const size_t stage   = kRowsWBytes + (size_t)nt * 8 * 512;
    tb200_status st = encode2d(ctx, &p.tmW0, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.w[0].data, q.w[0].pitch, q.W, q.w[0].pitch, 128, (uint32_t)kPer);
    if (st == TB200_OK && q.mats == 2)
        st = encode2d(ctx, &p.tmW1, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.w[1].data, q.w[1].pitch, q.W, q.w[1].pitch, 128, (uint32_t)kPer);
    if (st == TB200_OK)
        st = encode2d(ctx, &p.tmX, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x, q.C, xrows, x_pitch, 64, (uint32_t)(8 * nt));
    if (st != TB200_OK)
        return st;
    for (int m = 0; m < 2; m++)
    {
        p.scale[m]    = q.w[m].scale;
        p.zero[m]     = q.w[m].zero;
        p.scale_dt[m] = q.w[m].scale_dt;
    }
    p.W = q.W; p.C = q.C; p.rows = (int)q.M; p.parts = parts;
    p.group = q.group; p.act = q.act; p.out = q.out; p.out_dt = q.out_dt;
    p.wait_limit   = ctx->wait_limit_cycles;
    p.status       = ctx->d_status;
    p.stages_total = (q.C + kRowsStageK - 1) / kRowsStageK;
    p.stage_bytes  = (int)stage;
    // stages whose groups fit: one more group than whole ones may be touched
    p.super = (int)std::max<int64_t>(1, std::min<int64_t>(1 << 23, ((int64_t)(kRowsGroups - 2) * q.group) / kRowsStageK));
    const int64_t tiles = (q.W + kPer - 1) / kPer;
    const int64_t yb    = (q.M + rows_block - 1) / rows_block;
    // K over a cluster while the blocks do not fill two per SM and a block keeps two stages
    p.splits = 1;
    while (p.splits < 8 && p.stages_total / (2 * p.splits) >= 2 && tiles * yb * p.splits < ctx->num_sms)
        p.splits *= 2;
    p.per_split  = (p.stages_total + p.splits - 1) / p.splits;
    p.num_stages = std::max(2, std::min(kRowsMaxStages, std::min(p.per_split, (int)((72 * 1024) / stage))));
    const size_t red  = (size_t)8 * nt * kRowsRedLd * sizeof(float);
    const size_t smem = std::max(p.num_stages * stage, red) + 1024;
    const RowsKern kern = q.mats == 2 ? (bf16 ? pick<true, 2>(nt) : pick<false, 2>(nt)) : (bf16 ? pick<true, 1>(nt) : pick<false, 1>(nt));
    const int size_id   = nt <= 4 ? nt - 1 : 4;
    st = raise_smem_limit(ctx, 136 + size_id * 4 + (bf16 ? 2 : 0) + q.mats - 1, reinterpret_cast<const void*>(kern), (int)smem);
    if (st != TB200_OK)
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned)(tiles * p.splits), (unsigned)yb);
    cfg.blockDim           = dim3(kRowsThreads);
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
        return fail(ctx, TB200_INTERNAL, "launch of a 4-bit product failed: %s", cudaGetErrorString(le));
    return post_launch(ctx, q.mats == 2 ? "gated_w4_rows" : "matmul_w4_rows");
}

}    // namespace ffn
}    // namespace tb200
