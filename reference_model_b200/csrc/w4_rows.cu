// Host side of the products with 4-bit weights and few rows (w4_rows.cuh): tensor maps, shares, launch.
#include <algorithm>
#include <cstring>

#include "w4_rows.cuh"

namespace tb200
{
namespace ffn
{
namespace
{

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

// [rows][inner] elements of es bytes, rows `pitch` elements apart (a multiple of 16 bytes), as they lie
tb200_status encode_plain(tb200_ctx* ctx, CUtensorMap* m, size_t es, const void* data, int64_t inner, int64_t rows, int64_t pitch, uint32_t box_inner, uint32_t box_rows)
{
    const EncodeTiled enc = reinterpret_cast<EncodeTiled>(tensor_map_encode_fn());
    if (!enc)
        return fail(ctx, TB200_INTERNAL, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2]    = { (cuuint64_t)inner, (cuuint64_t)rows };
    const cuuint64_t strides[1] = { (cuuint64_t)pitch * es };
    const cuuint32_t box[2]     = { box_inner, box_rows };
    const cuuint32_t estr[2]    = { 1, 1 };
    const CUresult r = enc(m, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : es == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                           const_cast<void*>(data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(ctx, TB200_INTERNAL, "tensor map of a 4-bit product's scales rejected (CUresult %d)", (int)r);
    return TB200_OK;
}

// elements, up to whole sixteens of bytes
int64_t round_up16(int64_t n, size_t es)
{
    const int64_t per = 16 / (int64_t)es;
    return (n + per - 1) / per * per;
}

int tiles_of_eight(int64_t xrows)
{
    const int nt = (int)((xrows + 7) / 8);
    return nt == 5 ? 6 : nt == 7 ? 8 : nt;
}

}    // namespace

// Blocks are resident two to an SM (one with more rows, whose sums take the registers), all at once.
int64_t w4_rows_blocks(const tb200_ctx* ctx, int64_t xrows)
{
    return (int64_t)ctx->num_sms * rows_blocks_sm(tiles_of_eight(xrows));
}

size_t w4_rows_partial_bytes(const tb200_ctx* ctx, int64_t xrows)
{
    return (size_t)w4_rows_blocks(ctx, xrows) * 2 * 8 * tiles_of_eight(xrows) * kRowsTile * sizeof(float);
}

// x: the rows in 16 bits (bf16 parts of fp32 rows), `x_pitch` elements apart, 16-byte aligned; the weights' pitch is a multiple of 16;
// at most 32 of them (64 of the parts).  partial: w4_rows_partial_bytes.
tb200_status w4_rows_launch(tb200_ctx* ctx, const W4Problem& q, const void* x, int64_t x_pitch, int parts, bool bf16, float* partial)
{
    RowsParams p;
    memset(&p, 0, sizeof(p));
    const int xrows    = (int)q.M * parts;
    const int nt       = tiles_of_eight(xrows);
    const int kPer     = kRowsTile / q.mats;
    const int tiles    = (q.W + kPer - 1) / kPer;
    if (tiles > ctx->ffn_counts)
    {
        if (ctx->capturing)
            return fail(ctx, TB200_ERROR, "counters of 4-bit products would have to grow during capture; evaluate once eagerly first");
        release_block(ctx, ctx->ffn_count);
        ctx->ffn_count    = nullptr;
        ctx->ffn_counts   = 0;
        const int want    = std::max(tiles, 4096);
        void* block       = nullptr;
        TB200_CUDA_CHECK(ctx, cudaMalloc(&block, (size_t)want * sizeof(int)));
        ctx->ffn_count = reinterpret_cast<int*>(block);
        TB200_CUDA_CHECK(ctx, cudaMemsetAsync(block, 0, (size_t)want * sizeof(int), ctx->stream));
        ctx->ffn_counts = want;
    }
    tb200_status st = encode2d(ctx, &p.tmW0, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.w[0].data, q.w[0].pitch, q.W, q.w[0].pitch, 128, (uint32_t)kPer);
    if (st == TB200_OK && q.mats == 2)
        st = encode2d(ctx, &p.tmW1, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q.w[1].data, q.w[1].pitch, q.W, q.w[1].pitch, 128, (uint32_t)kPer);
    if (st == TB200_OK)
        st = encode2d(ctx, &p.tmX, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x, q.C, xrows, x_pitch, 64, (uint32_t)(8 * nt));
    if (st != TB200_OK)
        return st;
    // runs that share a group in every matrix column: as long as divides the group (one that holds a whole row may be cut anywhere)
    p.unit        = q.group >= q.C || q.group % 128 == 0 ? 4 : q.group % 64 == 0 ? 2 : 1;
    p.units_group = q.group >= q.C ? 0x7fffffffu : (uint32_t)(q.group / (32 * p.unit));
    const int units      = 8 / p.unit;
    const int64_t groups = ((int64_t)q.C + q.group - 1) / q.group;
    size_t stage         = kRowsWBytes + (size_t)nt * 8 * 512, loaded = stage;    // its place in the ring, what is copied there
    for (int m = 0; m < q.mats; m++)
    {
        const size_t es = dtype_size(q.w[m].scale_dt);
        p.scale_dt[m]   = q.w[m].scale_dt;
        p.has_zero[m]   = q.w[m].zero ? 1 : 0;
        auto operand = [&](CUtensorMap* map, size_t size, const void* data, int* off, int* step, int* flat) {
            const bool whole = (size_t)q.W * size % 16 == 0;
            *flat            = whole ? 0 : (int)(16 / size);
            *off             = (int)stage;
            // (a box of its own starts at a multiple of 128 bytes)
            *step = whole ? (int)(kPer * size) : (int)((kPer * size + 16 + 127) / 128 * 128);
            stage += (size_t)units * *step;
            loaded += (size_t)units * (kPer * size + (whole ? 0 : 16));
            return whole ? encode_plain(ctx, map, size, data, q.W, groups, q.W, (uint32_t)kPer, (uint32_t)units)
                         : encode_plain(ctx, map, size, data, groups * q.W, 1, round_up16(groups * q.W, size), (uint32_t)(kPer + 16 / size), 1);
        };
        st = operand(&p.tmS[m], es, q.w[m].scale, &p.s_off[m], &p.s_step[m], &p.s_flat[m]);
        if (st == TB200_OK && q.w[m].zero)
            st = operand(&p.tmZ[m], 1, q.w[m].zero, &p.z_off[m], &p.z_step[m], &p.z_flat[m]);
        if (st != TB200_OK)
            return st;
        p.z_words[m] = (kPer + (p.z_flat[m] ? 16 : 0)) / 4;
    }
    stage = (stage + 1023) & ~(size_t)1023;
    p.W = q.W; p.C = q.C; p.rows = (int)q.M; p.parts = parts;
    p.group = q.group; p.act = q.act; p.out = q.out; p.out_dt = q.out_dt;
    p.wait_limit   = ctx->wait_limit_cycles;
    p.status       = ctx->d_status;
    p.partial      = partial;
    p.counts       = ctx->ffn_count;
    p.stages_total = (q.C + kRowsStageK - 1) / kRowsStageK;
    p.stage_bytes  = (int)stage;
    p.loaded_bytes = (int)loaded;
    p.units_total = tiles * p.stages_total;
    const int64_t most = w4_rows_blocks(ctx, xrows);
    p.per_block        = (int)((p.units_total + most - 1) / most);
    const int blocks   = (p.units_total + p.per_block - 1) / p.per_block;
    const size_t red   = (size_t)8 * nt * kRowsRedLd * sizeof(float);
    const size_t room  = (rows_blocks_sm(nt) == 2 ? 113 : 226) * 1024 - (red + 2048);
    p.num_stages       = std::max(2, std::min(kRowsMaxStages, (int)(room / stage)));
    const size_t smem  = p.num_stages * stage + red + 1024;
    const bool flat     = p.s_flat[0] || p.z_flat[0] || p.s_flat[1] || p.z_flat[1];
    const RowsKern kern = bf16 ? w4_rows_kernel_bf16(nt, q.mats, flat) : w4_rows_kernel_f16(nt, q.mats, flat);
    const int size_id   = nt <= 4 ? nt - 1 : nt / 2 + 1;
    if (!kern)
        return fail(ctx, TB200_INTERNAL, "no kernel for %d rows against 4-bit weights", xrows);
    st = raise_smem_limit(ctx, 192 + size_id * 8 + (flat ? 4 : 0) + (bf16 ? 2 : 0) + q.mats - 1, reinterpret_cast<const void*>(kern), (int)smem);
    if (st != TB200_OK)
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned)blocks);
    cfg.blockDim           = dim3(kRowsThreads);
    cfg.dynamicSmemBytes   = smem;
    cfg.stream             = ctx->stream;
    cudaLaunchAttribute at[1];
    at[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs    = at;
    cfg.numAttrs = ctx->launch_overlap ? 1 : 0;
    timer_begin(ctx);
    const cudaError_t le = cudaLaunchKernelEx(&cfg, kern, p);
    timer_end(ctx);
    if (le != cudaSuccess)
        return fail(ctx, TB200_INTERNAL, "launch of a 4-bit product failed: %s", cudaGetErrorString(le));
    return post_launch(ctx, q.mats == 2 ? "gated_w4_rows" : "matmul_w4_rows");
}

}    // namespace ffn
}    // namespace tb200
