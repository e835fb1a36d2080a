// Products with 4-bit weights, up to 32 rows (64 of fp32's parts): the weights are read once, straight from their bytes, and multiplied on the warp-level
// matrix instruction (m16n8k16) with the output's columns as its sixteen rows and eight rows of `a` as its columns.  A 128-row
// tensor-core tile would be padding, and CUDA cores cannot keep up: at the memory's rate an SM receives 46 weights a clock, which
// leaves 2.8 lane instructions for each.
//
// q - z (element minus zero point) is a whole number of at most 15, exact in fp16 and bf16; products of those with a's elements are exact in fp32,
// where the instruction adds them.  The scale multiplies the fp32 sum of a group: no weight is ever rounded.  fp32 rows go as three
// bf16 rows each (24 bits taken apart), whose results are added at the end.
//
// A nibble becomes a number by one bit operation and one multiply-add for two of them: (word & 000F000F) ^ 43084308 is the bf16 pair
// 128 + 8 + q (fp16: 1024 + 8 + q from 64086408), minus 136 + z.  A word holds eight elements of K and the instruction does not mind the order
// of K, so word t of a 32-element run feeds thread t of a quad twice; a's elements are paired to match ((0,4), (1,5), ...) by
// byte permutes of one 16-byte read.
//
// Work is cut into stages of 128 matrix rows (64 of each matrix for the gated product) by 256 elements of K; every block takes the same
// number of consecutive stages, whatever tile they belong to, so that all SMs end together (whole tiles over 148 SMs left up to
// half of them idle).  A tile that several blocks share goes through fp32 sums in scratch: the block whose stages complete it adds them
// up, in block order, so results do not depend on which one that is.
// Eight warps take 32 rows each and one half of every stage (with more rows of `a`, 16 and all of it).  One thread feeds a ring of stages
// by TMA (weights and rows of `a` with 128-byte swizzle, so that both are read from shared memory without bank conflicts; scales and zero points
// as they lie: threads that fetched them cost 5 us a call).
//
// Measured, bf16, one row, group 128 with zero points: 8192 x 8192 15.4 us (35 MB, 2.3 TB/s), gated 4096 x 16384 24.3 us (2.9 TB/s); 24 rows,
// 4096 x 10250 fp16 21.9 us; 2048 x 1000 6.5 us.  What bounds it: no single thing.  Instructions, 78 to 100 for 1024 weights, are 5 to 6 us of issue time for
// the first, 9 to 11 for the second, 3 to 3.5 for the third (45 % of the issue slots and 39 % of the integer pipe over the whole kernel).  Shared memory:
// with three tiles of eight rows each of eight warps reads all of `a` for its sixteen matrix rows, 98 KB a stage beside 16 KB of weights, about 4 us, and
// permutes it again.  Latencies at either end, paid for 4 to 14 stages a block: 1.4 us from the start to the first stage, 1.5 to 4 us
// from a shared tile's last sums to its results.
#pragma once
#include <cuda.h>
#include <type_traits>

#include "ffn.h"
#include "ffn_math.cuh"
#include "ptx_sm100.cuh"
#include "w4_unpack.cuh"

namespace tb200
{
namespace ffn
{

constexpr int kRowsWarps   = 8;
constexpr int kRowsThreads = 32 * (kRowsWarps + 2);    // and the TMA warp, and one that looks at the zero points
constexpr int kRowsTile    = 128;                      // matrix rows of a block
constexpr int kRowsStageK  = 256;                      // elements of K in a stage: 128 bytes of weights a row
constexpr int kRowsWBytes  = kRowsTile * 128;
constexpr int kRowsMaxStages = 6;
constexpr int kRowsRedLd   = kRowsTile + 4;            // row pitch of the sums in shared memory: a warp's stores meet 32 banks

struct RowsParams
{
    CUtensorMap tmW0, tmW1;    // bytes [W][pitch], box 128 x 128 (gated: 128 x 64 of each)
    CUtensorMap tmX;           // [rows][C] 16-bit, box 64 x 8 NT
    // Scales and zero points [groups][W], boxes of a tile's columns x the runs of a stage.  Where W elements are not whole sixteens of bytes
    // (flat): one row of groups x W, a box for each run that starts at the sixteen below its first element.
    CUtensorMap tmS[2], tmZ[2];
    tb200_dtype scale_dt[2];
    int has_zero[2];
    int s_off[2], z_off[2];    // of a stage's scales and zero points in the ring
    int s_step[2], z_step[2];  // bytes from one run's to the next
    int s_flat[2], z_flat[2];  // elements of sixteen bytes, or 0
    int z_words[2];            // of a run's zero points
    int W, C, rows;            // rows of `a`
    int parts;                 // 16-bit rows that make a row of `a`: 1, or 3 for fp32
    int group, act;
    int stages_total;          // stages of a tile
    int units_total, per_block;    // stages of all tiles, of a block
    int num_stages, stage_bytes, loaded_bytes;
    float* partial;                // [blocks][2][8 NT][kRowsTile]: sums of a block's first and last tile
    int* counts;                   // [tiles]: stages that have arrived; zero between launches
    int unit;                  // 32-element pieces of a run that shares a group: 1, 2 or 4
    uint32_t units_group;      // runs of a group
    void* out;
    tb200_dtype out_dt;
    long long wait_limit;
    int* status;
};

template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

// What a warp needs to know of its matrix: where a run's scales and zero points are, for its rows
struct RowsRun
{
    uint32_t scale, zero;    // shared addresses of the first run's, at the lane's first row
    int scale_step, zero_step;    // bytes from one run to the next
    uint32_t first, W;            // flat: where the first run's group has the tile's first column; its box begins at the sixteen bytes below
    uint32_t scale_mask, zero_mask;    // elements of sixteen bytes, less one, where flat
    tb200_dtype dt;
    bool has_zero;
};

// Scales of rows +0, +8, +16, +24, and minus their zero point: -(136 + z) twice as bf16 (steps of 1 from 128 on), -(1032 + z) as fp16 (steps
// of 1 from 1024 on).  A zero point that is none of -8 .. 7 is reported by the warp that looks for it; the product is then not one.
template <bool BF16, int MT, bool FLAT>
__device__ __forceinline__ void run_scales(const RowsRun& r, int i, float (&scale)[2 * MT], uint32_t (&base)[2 * MT])
{
    uint32_t at = r.scale + (uint32_t)(i * r.scale_step), zat = r.zero + (uint32_t)(i * r.zero_step);
    if (FLAT)
    {
        at += ((r.first + (uint32_t)i * r.W) & r.scale_mask) * (r.dt == TB200_FP32 ? 4 : 2);
        zat += (r.first + (uint32_t)i * r.W) & r.zero_mask;
    }
    if (r.dt == TB200_FP32)
    {
#pragma unroll
        for (int q = 0; q < 2 * MT; q++)
            scale[q] = __uint_as_float(lds32(at + (uint32_t)(q * 32)));
    }
    else
    {
#pragma unroll
        for (int q = 0; q < 2 * MT; q++)
        {
            uint16_t h;
            asm volatile("ld.shared.b16 %0, [%1];" : "=h"(h) : "r"(at + (uint32_t)(q * 16)));
            scale[q] = r.dt == TB200_BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
        }
    }
#pragma unroll
    for (int q = 0; q < 2 * MT; q++)
    {
        int z = 0;
        if (r.has_zero)
            asm volatile("ld.shared.s8 %0, [%1];" : "=r"(z) : "r"(zat + (uint32_t)(q * 8)));
        base[q] = unpack_base<BF16>(z);
    }
}

// One warp's part of a stage: eight 32-element pieces of 16 matrix rows, or four of 32 (MT 1 or 2 sixteens), against all rows of `a`; runs of
// UNIT pieces share a group.  `runs`: the row of scales that each run takes, four bits each.
template <bool BF16, int NT, int MT, int UNIT, bool FLAT>
__device__ __forceinline__ void stage_part(float (&total)[MT][NT][4], uint32_t sW, uint32_t sX, const uint32_t (&offW)[8 / MT],
                                           const uint32_t (&offX)[2], const RowsRun& run, uint32_t runs)
{
#pragma unroll
    for (int r = 0; r < 8 / MT / UNIT; r++)
    {
        float scale[2 * MT];
        uint32_t base[2 * MT];
        run_scales<BF16, MT, FLAT>(run, (int)(runs >> (4 * r) & 15), scale, base);
        float accum[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int j = 0; j < NT; j++)
                accum[m][j][0] = accum[m][j][1] = accum[m][j][2] = accum[m][j][3] = 0.f;
#pragma unroll
        for (int c = r * UNIT; c < (r + 1) * UNIT; c++)
        {
            uint32_t w[2 * MT][4];
#pragma unroll
            for (int q = 0; q < 2 * MT; q++)
                unpack8<BF16>(lds32(sW + offW[c] + (uint32_t)(q * 1024)), base[q], w[q]);
#pragma unroll
            for (int j = 0; j < NT; j++)
            {
                const uint4 x     = lds128(sX + offX[c & 1] + (uint32_t)((c >> 1) * 8 * NT * 128 + j * 1024));
                const uint32_t x0 = __byte_perm(x.x, x.z, 0x5410), x1 = __byte_perm(x.x, x.z, 0x7632), x2 = __byte_perm(x.y, x.w, 0x5410),
                               x3 = __byte_perm(x.y, x.w, 0x7632);
#pragma unroll
                for (int m = 0; m < MT; m++)
                {
                    mma<BF16>(accum[m][j], w[2 * m][0], w[2 * m + 1][0], w[2 * m][1], w[2 * m + 1][1], x0, x1);
                    mma<BF16>(accum[m][j], w[2 * m][2], w[2 * m + 1][2], w[2 * m][3], w[2 * m + 1][3], x2, x3);
                }
            }
        }
        // the run's sum under its scale
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int j = 0; j < NT; j++)
            {
                total[m][j][0] = fmaf(scale[2 * m], accum[m][j][0], total[m][j][0]);
                total[m][j][1] = fmaf(scale[2 * m], accum[m][j][1], total[m][j][1]);
                total[m][j][2] = fmaf(scale[2 * m + 1], accum[m][j][2], total[m][j][2]);
                total[m][j][3] = fmaf(scale[2 * m + 1], accum[m][j][3], total[m][j][3]);
            }
    }
}

// Rows of the matrix that a warp takes, in sixteens, and blocks to an SM.  Few rows of `a`: 32 matrix rows share every read and permutation of a's
// elements.  More: sixteen, whose sums leave registers for two blocks, and the matrix instructions take as long as the rest.
constexpr int rows_mt(int nt)
{
    return nt <= 2 ? 2 : 1;
}
constexpr int rows_blocks_sm(int nt)
{
    return nt <= 4 ? 2 : 1;
}

template <bool BF16, int NT, int MATS, bool FLAT>
__global__ void __launch_bounds__(kRowsThreads, rows_blocks_sm(NT)) w4_rows_kernel(const __grid_constant__ RowsParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[kRowsMaxStages];
    __shared__ __align__(8) uint64_t bar_empty[kRowsMaxStages];
    __shared__ int completes[2];

    constexpr int kPer       = kRowsTile / MATS;    // columns of the output
    constexpr int MT         = rows_mt(NT);
    const int tid            = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const ring      = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    float* const red         = reinterpret_cast<float*>(ring + p.num_stages * p.stage_bytes);    // sums of a tile
    const int S = p.stages_total, begin = (int)blockIdx.x * p.per_block, end = min(p.units_total, begin + p.per_block);

    if (tid == 0)
    {
        for (int s = 0; s < p.num_stages; s++)
        {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), kRowsWarps + 1);
        }
        ptx::fence_barrier_init();
        ptx::prefetch_tmap(&p.tmW0);
        ptx::prefetch_tmap(&p.tmX);
        if (MATS == 2)
            ptx::prefetch_tmap(&p.tmW1);
        ptx::dep_launch_trigger();
        // the ring's first weights on their way to L2, where a write by the kernel before would still find them
        for (int u = begin, i = 0; u < end && i < p.num_stages; u++, i++)
        {
            ptx::prefetch_2d(&p.tmW0, u % S * 128, u / S * kPer);
            if (MATS == 2)
                ptx::prefetch_2d(&p.tmW1, u % S * 128, u / S * kPer);
        }
    }
    __syncthreads();
    // everything a kernel before this one may have written is read behind this wait
    ptx::dep_launch_wait();

    const int units = p.unit == 4 ? 2 : p.unit == 2 ? 4 : 8;    // runs of a stage
    const int tile0 = begin / S, stage0 = begin - tile0 * S;

    if (warp == kRowsWarps)
    {
        if (lane == 0)
        {
            bool ok = true;
            int i = 0, s = 0, tile = tile0, k = stage0;
            uint32_t phase = 0;
            for (; i < end - begin; i++)
            {
                if (!ptx::mbar_wait_bounded(ptx::smem_u32(&bar_empty[s]), phase ^ 1u, p.wait_limit))
                {
                    ok = false;
                    break;
                }
                const uint32_t full = ptx::smem_u32(&bar_full[s]);
                const uint32_t sW   = smem_base + (uint32_t)(s * p.stage_bytes), sX = sW + kRowsWBytes;
                ptx::mbar_arrive_expect_tx(full, (uint32_t)p.loaded_bytes);
                ptx::tma_load_2d(sW, &p.tmW0, full, k * 128, tile * kPer);
                if (MATS == 2)
                    ptx::tma_load_2d(sW + kPer * 128, &p.tmW1, full, k * 128, tile * kPer);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    ptx::tma_load_2d(sX + (uint32_t)(j * 8 * NT * 128), &p.tmX, full, k * kRowsStageK + j * 64, 0);
                const int group = (int)((uint32_t)(k * units) / p.units_group);    // of the stage's first run
#pragma unroll
                for (int m = 0; m < MATS; m++)
                {
                    auto load = [&](const CUtensorMap* map, int off, int step, int flat) {
                        if (!FLAT || !flat)
                        {
                            ptx::tma_load_2d(sW + (uint32_t)off, map, full, tile * kPer, group);
                            return;
                        }
                        // a box behind the last element reads as zeros
                        for (int r = 0; r < units; r++)
                        {
                            const int64_t at = min((int64_t)(group + r) * p.W + tile * kPer, (int64_t)0x7ffffff0);    // (may pass the last group)
                            ptx::tma_load_2d(sW + (uint32_t)(off + r * step), map, full, (int)(at & ~(int64_t)(flat - 1)), 0);
                        }
                    };
                    load(&p.tmS[m], p.s_off[m], p.s_step[m], p.s_flat[m]);
                    if (p.has_zero[m])
                        load(&p.tmZ[m], p.z_off[m], p.z_step[m], p.z_flat[m]);
                }
                if (++k == S)
                {
                    k = 0;
                    tile++;
                }
                if (++s == p.num_stages)
                {
                    s = 0;
                    phase ^= 1u;
                }
            }
            if (!ok)
                atomicOr(p.status, TB200_DEV_TIMEOUT);
            // Copies in flight land before the block leaves, whichever role may have given up on them.  (A block whose roles all go on waits
            // for them anyway.)
            for (int j = max(0, i - p.num_stages); j < i; j++)
                ptx::mbar_wait_bounded(ptx::smem_u32(&bar_full[j % p.num_stages]), (uint32_t)(j / p.num_stages) & 1u, ptx::kDrainCycles);
        }
    }
    else if (warp > kRowsWarps)
    {
        // REQUIRE: zero points are 4-bit numbers, -8 .. 7 (what lies outside the matrix reads as 0)
        bool ok = true;
        uint32_t bad = 0, phase = 0;
        for (int u = begin, s = 0; u < end && ok; u++)
        {
            ok = ptx::mbar_wait_bounded(ptx::smem_u32(&bar_full[s]), phase, p.wait_limit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
#pragma unroll
            for (int m = 0; m < MATS; m++)
                for (int e = lane; p.has_zero[m] && e < units * p.z_words[m]; e += 32)
                {
                    // (flat: with some of the neighbouring groups')
                    const int r = e / p.z_words[m], c = e - r * p.z_words[m];
                    const uint32_t z = lds32(smem_base + (uint32_t)(s * p.stage_bytes + p.z_off[m] + r * p.z_step[m] + 4 * c));
                    bad |= __vcmpgts4(z, 0x07070707u) | __vcmplts4(z, 0xF8F8F8F8u);
                }
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
            atomicOr(p.status, TB200_DEV_TIMEOUT);
        if (bad)
            atomicOr(p.status, TB200_DEV_UNPREDICTABLE);
    }
    else
    {
        const int g = lane >> 2, t = lane & 3;
        const int group = MT == 2 ? warp & 3 : warp;    // of 16 MT matrix rows
        const int half  = MT == 2 ? warp >> 2 : 0;      // of a stage: 32-element pieces 4 half .. 4 half + 3, or all eight
        const int wrow  = group * 16 * MT + g;          // and wrow + 8 (+ 16, + 24)
        // column n of the instruction is row perm(n) of the tile of eight: neighbouring lanes' reads then meet different banks
        const int xr = (g >> 1) + (g & 1) * 4;
        uint32_t offW[8 / MT], offX[2];
#pragma unroll
        for (int c = 0; c < 8 / MT; c++)
            offW[c] = (uint32_t)(wrow * 128 + t * 4) + (uint32_t)((((half * 4 + c) ^ g) & 7) << 4);
#pragma unroll
        for (int c = 0; c < 2; c++)
            offX[c] = (uint32_t)(half * 2 * 8 * NT * 128 + xr * 128) + (uint32_t)(((c * 4 + t) ^ xr) << 4);
        const int values = p.rows * p.parts * kRowsTile;
        // results of a tile whose sums are in `red`
        auto results = [&](int col0) {
            // a thread stays with its column
            const int c = tid % kPer;
            if (col0 + c >= p.W)
                return;
            constexpr int kStep = 32 * kRowsWarps / kPer;
            const int64_t out   = (int64_t)(tid / kPer) * p.W + col0 + c;
            const float* at     = red + tid / kPer * p.parts * kRowsRedLd + c;
#pragma unroll 4
            for (int r = tid / kPer, i = 0; r < p.rows; r += kStep, i++)
            {
                float v[MATS];
#pragma unroll
                for (int m = 0; m < MATS; m++)
                {
                    const float* const x = at + (int64_t)i * kStep * p.parts * kRowsRedLd + m * kPer;
                    v[m]                 = p.parts == 3 ? x[2 * kRowsRedLd] + x[kRowsRedLd] + x[0] : x[0];    // the smallest first
                }
                store_fp(p.out, out + (int64_t)i * kStep * p.W, p.out_dt, MATS == 2 ? act_value(p.act, v[0]) * v[MATS - 1] : v[0]);
            }
        };
        constexpr int kSlot = 8 * NT * kRowsTile;
        bool ok = true;
        int s = 0, tile = tile0, k = stage0;
        uint32_t phase = 0;
        const int mat = MATS == 2 ? wrow / kPer : 0, mrow = wrow - mat * kPer;    // row of its matrix in the tile
        RowsRun run;
        run.dt         = p.scale_dt[mat];
        run.has_zero   = p.has_zero[mat] != 0;
        run.scale_step = p.s_step[mat];
        run.zero_step  = p.z_step[mat];
        run.W          = (uint32_t)p.W;
        run.scale_mask = p.s_flat[mat] ? (uint32_t)p.s_flat[mat] - 1 : 0;
        run.zero_mask  = p.z_flat[mat] ? (uint32_t)p.z_flat[mat] - 1 : 0;
        run.first      = 0;
        const uint32_t s_off = (uint32_t)(p.s_off[mat] + mrow * (run.dt == TB200_FP32 ? 4 : 2)), z_off = (uint32_t)(p.z_off[mat] + mrow);
        const uint32_t full0 = ptx::smem_u32(&bar_full[0]), empty0 = ptx::smem_u32(&bar_empty[0]);
        for (int u = begin; u < end;)
        {
            const int n = min(end - u, S - k);    // stages of this tile
            float total[MT][NT][4];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int j = 0; j < NT; j++)
                    total[m][j][0] = total[m][j][1] = total[m][j][2] = total[m][j][3] = 0.f;
            auto stages = [&](auto pieces) {
                constexpr int UNIT = decltype(pieces)::value, kRuns = 8 / UNIT;
                // rows of scales that this part's runs take: one each, or fewer where a group holds several runs
                const uint32_t own = half ? 0x76543210u >> (2 * kRuns) : 0x76543210u;
                for (int i = 0; i < n; i++)
                {
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(full0 + 8 * s, phase, p.wait_limit));
                    if (!ok)
                        break;
                    const uint32_t sW = smem_base + (uint32_t)(s * p.stage_bytes);
                    run.scale         = sW + s_off;
                    run.zero          = sW + z_off;
                    uint32_t runs     = own;
                    if (FLAT)
                        run.first = (uint32_t)((k + i) * kRuns) / p.units_group * run.W + (uint32_t)(tile * kPer);
                    if (p.units_group > 1)
                    {
                        const uint32_t u0 = (uint32_t)((k + i) * kRuns), g0 = u0 / p.units_group;
                        runs              = 0;
#pragma unroll
                        for (int r = 0; r < kRuns / MT; r++)
                            runs |= ((u0 + (own >> (4 * r) & 15)) / p.units_group - g0) << (4 * r);
                    }
                    stage_part<BF16, NT, MT, UNIT, FLAT>(total, sW, sW + kRowsWBytes, offW, offX, run, runs);
                    __syncwarp();
                    if (lane == 0)
                        ptx::mbar_arrive(empty0 + 8 * s);
                    if (++s == p.num_stages)
                    {
                        s = 0;
                        phase ^= 1u;
                    }
                }
            };
            if (ok)
            {
                if (p.unit == 4)
                    stages(std::integral_constant<int, 4>());
                else if (p.unit == 2)
                    stages(std::integral_constant<int, 2>());
                else
                    stages(std::integral_constant<int, 1>());
            }
            // the eight warps go on together; after a wait that gave up they only count their stages, so that the counts end at zero
            ok = ptx::named_barrier_and(1, 32 * kRowsWarps, ok);
            const int col0 = tile * kPer;
            if (ok)
            {
                // the first half's sums, then the second's on top
#pragma unroll
                for (int pass = 0; pass < MT; pass++)
                {
                    if (half == pass)
                    {
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int j = 0; j < NT; j++)
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                {
                                    // instruction columns 2t and 2t + 1 are rows t and t + 4 of the tile of eight
                                    float* const at = red + (j * 8 + t + (e & 1) * 4) * kRowsRedLd + wrow + m * 16 + (e >> 1) * 8;
                                    *at             = pass ? *at + total[m][j][e] : total[m][j][e];
                                }
                    }
                    ptx::named_barrier_and(1, 32 * kRowsWarps, true);
                }
            }
            if (n == S)
            {
                if (ok)
                    results(col0);
            }
            else if (ok)
            {
                float4* const mine = reinterpret_cast<float4*>(p.partial + ((int64_t)blockIdx.x * 2 + (u == begin ? 0 : 1)) * kSlot);
                for (int e = tid; e < values / 4; e += 32 * kRowsWarps)
                    __stcg(mine + e, *reinterpret_cast<const float4*>(red + e / (kRowsTile / 4) * kRowsRedLd + e % (kRowsTile / 4) * 4));
            }
            ptx::named_barrier_and(1, 32 * kRowsWarps, true);    // `red` is free again
            u += n;
            k = 0;
            tile++;
        }
        // tiles shared with other blocks, at most the first and the last: whoever brings the last stages adds the sums up, in block order
        const int n_first = min(end - begin, S - stage0), tile_last = (end - 1) / S, n_last = end - tile_last * S;
        const bool share_first = n_first < S, share_last = tile_last > tile0 && n_last < S;
        if (tid == 0)
        {
            __threadfence();    // the block's sums, which the barrier above has put before this
            const int first = share_first ? atomicAdd(p.counts + tile0, n_first) : 0, last = share_last ? atomicAdd(p.counts + tile_last, n_last) : 0;
            completes[0]    = share_first && first + n_first == S;
            completes[1]    = share_last && last + n_last == S;
            if (completes[0])
                p.counts[tile0] = 0;    // for the next launch
            if (completes[1])
                p.counts[tile_last] = 0;
            __threadfence();
        }
        ptx::named_barrier_and(1, 32 * kRowsWarps, true);
#pragma unroll
        for (int which = 0; which < 2; which++)
        {
            if (!completes[which] || !ok)
                continue;
            const int shared = which ? tile_last : tile0;
            const int lo = shared * S / p.per_block, hi = (shared * S + S - 1) / p.per_block;
            // the tile is the first of every block but maybe `lo`, which may have come from the one before
            const int slot_lo = lo * p.per_block >= shared * S ? 0 : 1;
            const float4* const first = reinterpret_cast<const float4*>(p.partial + ((int64_t)lo * 2 + slot_lo) * kSlot);
            if (values <= 2 * 32 * kRowsWarps && hi - lo > 2)
            {
                // few sums from many blocks: the threads share out the blocks too (one thread's loads, four blocks at a time, were most of
                // the call where 28 blocks had a stage each of one tile)
                const int quads = values / 4, parts = 32 * kRowsWarps / quads, quad = tid % quads, part = tid / quads;
                float4 v        = make_float4(0.f, 0.f, 0.f, 0.f);
                if (part < parts)
                {
#pragma unroll 4
                    for (int block = lo + part; block <= hi; block += parts)
                    {
                        const float4 x = __ldcg(block == lo ? first + quad : reinterpret_cast<const float4*>(p.partial + (int64_t)block * 2 * kSlot) + quad);
                        v.x += x.x;
                        v.y += x.y;
                        v.z += x.z;
                        v.w += x.w;
                    }
                }
                float4* const shared_sums = reinterpret_cast<float4*>(red);    // 256 of them: no more than `red` holds
                shared_sums[tid]          = v;
                ptx::named_barrier_and(1, 32 * kRowsWarps, true);
                v = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < parts && tid < quads; k++)
                {
                    const float4 x = shared_sums[k * quads + tid];
                    v.x += x.x;
                    v.y += x.y;
                    v.z += x.z;
                    v.w += x.w;
                }
                ptx::named_barrier_and(1, 32 * kRowsWarps, true);
                if (tid < quads)
                    *reinterpret_cast<float4*>(red + tid / (kRowsTile / 4) * kRowsRedLd + tid % (kRowsTile / 4) * 4) = v;
                ptx::named_barrier_and(1, 32 * kRowsWarps, true);
                results(shared * kPer);
                ptx::named_barrier_and(1, 32 * kRowsWarps, true);
                continue;
            }
            constexpr int kAtOnce = 4;    // loads of a thread on their way together
            for (int e0 = tid; e0 < values / 4; e0 += 32 * kRowsWarps * kAtOnce)
            {
                float4 v[kAtOnce];
#pragma unroll
                for (int e = 0; e < kAtOnce; e++)
                {
                    const int at = e0 + e * 32 * kRowsWarps;
                    v[e]         = at < values / 4 ? __ldcg(first + at) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll 4
                for (int block = lo + 1; block <= hi; block++)
                {
                    const float4* const next = reinterpret_cast<const float4*>(p.partial + (int64_t)block * 2 * kSlot);
#pragma unroll
                    for (int e = 0; e < kAtOnce; e++)
                    {
                        const int at   = e0 + e * 32 * kRowsWarps;
                        const float4 x = at < values / 4 ? __ldcg(next + at) : make_float4(0.f, 0.f, 0.f, 0.f);
                        v[e].x += x.x;
                        v[e].y += x.y;
                        v[e].z += x.z;
                        v[e].w += x.w;
                    }
                }
#pragma unroll
                for (int e = 0; e < kAtOnce; e++)
                {
                    const int at = e0 + e * 32 * kRowsWarps;
                    if (at < values / 4)
                        *reinterpret_cast<float4*>(red + at / (kRowsTile / 4) * kRowsRedLd + at % (kRowsTile / 4) * 4) = v[e];
                }
            }
            ptx::named_barrier_and(1, 32 * kRowsWarps, true);
            results(shared * kPer);
            ptx::named_barrier_and(1, 32 * kRowsWarps, true);
        }
        if (!ok && lane == 0)
            atomicOr(p.status, TB200_DEV_TIMEOUT);
    }
}

typedef void (*RowsKern)(const RowsParams);

// (more than 32 rows are fp32's parts, in bf16)
template <bool BF16, int MATS, bool FLAT>
RowsKern pick(int nt)
{
    if constexpr (BF16)
    {
        if (nt == 6)
            return w4_rows_kernel<BF16, 6, MATS, FLAT>;
        if (nt == 8)
            return w4_rows_kernel<BF16, 8, MATS, FLAT>;
    }
    return nt == 1   ? w4_rows_kernel<BF16, 1, MATS, FLAT>
           : nt == 2 ? w4_rows_kernel<BF16, 2, MATS, FLAT>
           : nt == 3 ? w4_rows_kernel<BF16, 3, MATS, FLAT>
           : nt == 4 ? w4_rows_kernel<BF16, 4, MATS, FLAT>
                     : nullptr;
}

// w4_rows_f16.cu, w4_rows_bf16.cu: the kernel for `nt` tiles of eight rows
RowsKern w4_rows_kernel_f16(int nt, int mats, bool flat);
RowsKern w4_rows_kernel_bf16(int nt, int mats, bool flat);

}    // namespace ffn
}    // namespace tb200
