// Entry points of the feed-forward operators: argument rules, workspaces, and which kernels serve a call.
#include <algorithm>
#include <cstring>
#include <exception>

#include "ffn.h"

using namespace tb200;
using namespace tb200::ffn;

namespace
{

// Nothing throws across the C boundary: host memory that runs out ends in a status.
template <typename F>
tb200_status guarded(tb200_ctx* ctx, F body)
{
    try
    {
        return body();
    }
    catch (const std::exception& e)
    {
        (void)e;
        return ctx ? fail(ctx, TB200_INTERNAL, "out of host memory") : TB200_INTERNAL;
    }
}

// Carves a call's workspace out of the context's scratch: first the sizes, then the addresses.
struct Carver
{
    uint8_t* base = nullptr;
    size_t used   = 0;
    void* take(size_t bytes)
    {
        void* p = base ? base + used : nullptr;
        used += (bytes + 255) & ~(size_t)255;
        return p;
    }
};

int64_t round_up(int64_t v, int64_t to)
{
    return (v + to - 1) / to * to;
}

// A 16-bit operand as the tensor maps want it, rows a multiple of 16 bytes apart: as it lies, or copied into `pad`.
Matrix operand(const void* data, int64_t inner, int64_t outer, int64_t batches, void* pad)
{
    Matrix m = { data, inner, outer, batches, inner };
    if (inner % 8 != 0)
    {
        m.data  = pad;
        m.pitch = round_up(inner, 8);
    }
    return m;
}

size_t pad_bytes(int64_t inner, int64_t rows)
{
    return inner % 8 != 0 ? (size_t)rows * round_up(inner, 8) * 2 : 0;
}

void pad(RowCopies* copies, const void* data, const Matrix& m)
{
    if (m.data != data)
        copies->add(data, const_cast<void*>(m.data), m.outer * m.batches, m.inner * 2, m.inner * 2, m.pitch * 2);
}

#define TB200_TRY(expr)                     \
    do                                      \
    {                                       \
        const tb200_status st__ = (expr);   \
        if (st__ != TB200_OK)               \
            return st__;                    \
    } while (0)

// Rows up to which the kernels that stream the weights past a few rows serve; with more, 128-row tiles of the tensor cores are quicker for all their
// padding (4-bit 4096 x 4096: 24 rows 11.7 against 13.0 us, 33 rows 14.6 against 13.1; 16-bit gated 2048 x 8192: 32 rows 14.3 against
// 16.8, 33 rows 25.6 against 16.9).  fp32 rows against 4-bit weights, whose alternative is a pass over fp32 values: 64 of their parts.
constexpr int64_t kFewRows = 32, kFewParts = 64;

// 16-bit gated product on the tensor cores
tb200_status gated_pair(tb200_ctx* ctx, const GatedProblem& q)
{
    const bool few = q.H <= kFewRows && q.NB <= 65535;    // (that kernel takes the matrices as they lie)
    Carver size, at;
    for (int pass = 0; pass < 2; pass++)
    {
        Carver& c     = pass ? at : size;
        void* const a = c.take(pad_bytes(q.C, q.NB * q.H));
        void* const g = c.take(few ? 0 : pad_bytes(q.W, (int64_t)q.NB * q.C));
        void* const u = c.take(few ? 0 : pad_bytes(q.W, (int64_t)q.NB * q.C));
        if (!pass)
        {
            if (size.used)
                TB200_TRY(ensure_scratch(ctx, size.used));
            at.base = reinterpret_cast<uint8_t*>(ctx->scratch);
            continue;
        }
        PairProduct k;
        memset(&k, 0, sizeof(k));
        k.dt   = q.dt;
        k.kind = PAIR_GATED;
        k.b_mn = true;
        k.a    = operand(q.a, q.C, q.H, q.NB, a);
        k.b[0] = operand(q.gate, q.W, q.C, q.NB, g);
        k.b[1] = operand(q.up, q.W, q.C, q.NB, u);
        if (few)
        {
            k.b[0] = { q.gate, q.W, q.C, q.NB, q.W };
            k.b[1] = { q.up, q.W, q.C, q.NB, q.W };
        }
        RowCopies copies;
        pad(&copies, q.a, k.a);
        pad(&copies, q.gate, k.b[0]);
        pad(&copies, q.up, k.b[1]);
        TB200_TRY(row_copies_launch(ctx, copies));
        k.rows      = (int)q.H;
        k.cols      = q.W;
        k.K         = q.C;
        k.phases    = 1;
        k.NB        = q.NB;
        k.results   = 1;
        k.act       = q.act;
        k.out[0]    = q.out;
        k.out_dt[0] = k.out_dt[1] = q.out_dt;
        k.ld        = q.W;
        k.name      = "gated_pair_f16";
        TB200_TRY(few ? gated_rows_launch(ctx, k) : pair_launch(ctx, k));
    }
    return TB200_OK;
}

// Its gradients: dG and dU into scratch, then one product for grad_a and one for both weights'.  Both are rounded to the operands' type, whatever type a
// gradient has: two numbers each would double the MMAs of two thirds of the pass (1105 us at 4096 x 4096 x 8192), and half a step of each element counts
// for less in a sum over many.  In FP16 they are held under a power of two where their size calls for one, which a second launch sees to.
tb200_status gated_backward_pair(tb200_ctx* ctx, const GatedProblem& q)
{
    const int64_t Wp  = round_up(q.W, 16);
    const size_t half = (size_t)q.NB * q.H * Wp * 2;    // bytes of dG
    Carver size, at;
    for (int pass = 0; pass < 2; pass++)
    {
        Carver& c           = pass ? at : size;
        void* const pa      = c.take(pad_bytes(q.C, q.NB * q.H));
        void* const pg      = c.take(pad_bytes(q.W, (int64_t)q.NB * q.C));
        void* const pu      = c.take(pad_bytes(q.W, (int64_t)q.NB * q.C));
        uint8_t* const dg   = reinterpret_cast<uint8_t*>(c.take(2 * half));
        const bool f16      = q.dt == TB200_FP16;
        float* const peaks  = reinterpret_cast<float*>(c.take(f16 ? (size_t)pair_peaks(ctx) * sizeof(float) : 0));
        float* const undo   = reinterpret_cast<float*>(c.take(f16 ? sizeof(float) : 0));
        if (!pass)
        {
            TB200_TRY(ensure_scratch(ctx, size.used));
            at.base = reinterpret_cast<uint8_t*>(ctx->scratch);
            continue;
        }
        const Matrix a = operand(q.a, q.C, q.H, q.NB, pa), gate = operand(q.gate, q.W, q.C, q.NB, pg), up = operand(q.up, q.W, q.C, q.NB, pu);
        RowCopies copies;
        pad(&copies, q.a, a);
        pad(&copies, q.gate, gate);
        pad(&copies, q.up, up);
        TB200_TRY(row_copies_launch(ctx, copies));
        PairProduct k;
        memset(&k, 0, sizeof(k));
        k.dt      = q.dt;
        k.kind    = PAIR_GRAD;
        k.b_mn    = true;
        k.a       = a;
        k.b[0]    = gate;
        k.b[1]    = up;
        k.rows    = (int)q.H;
        k.cols    = q.W;
        k.K       = q.C;
        k.phases  = 1;
        k.NB      = q.NB;
        k.results = 2;
        k.act     = q.act;
        k.dout    = q.dout;
        k.out[0]  = dg;
        k.out[1]  = dg + half;
        k.out_dt[0] = k.out_dt[1] = q.dt;
        k.ld      = Wp;
        k.name    = "gated_backward_pair_f16";
        k.peaks   = f16 ? peaks : nullptr;
        TB200_TRY(pair_launch(ctx, k));
        if (f16)
        {
            k.peaks = nullptr;
            k.seen  = peaks;
            k.undo  = undo;
            TB200_TRY(pair_launch(ctx, k));
        }
        const Matrix d = { dg, q.W, q.H, 2 * (int64_t)q.NB, Wp };
        if (q.da)
        {
            memset(&k, 0, sizeof(k));
            k.dt        = q.dt;
            k.kind      = PAIR_PLAIN;
            k.a         = d;
            k.b[0]      = gate;
            k.b[1]      = up;
            k.rows      = (int)q.H;
            k.cols      = q.C;
            k.K         = q.W;
            k.phases    = 2;
            k.NB        = q.NB;
            k.results   = 1;
            k.out[0]    = q.da;
            k.out_dt[0] = q.da_dt;
            k.undo      = f16 ? undo : nullptr;
            k.ld        = q.C;
            k.name      = "gated_backward_pair_f16";
            TB200_TRY(pair_launch(ctx, k));
        }
        if (q.dgate || q.dup)
        {
            memset(&k, 0, sizeof(k));
            k.dt      = q.dt;
            k.kind    = PAIR_PLAIN;
            k.a_mn    = true;
            k.b_mn    = true;
            k.a       = a;
            k.b[0]    = d;
            k.rows    = q.C;
            k.cols    = q.W;
            k.K       = q.H;
            k.phases  = 1;
            k.NB      = q.NB;
            k.results = q.dgate && q.dup ? 2 : 1;
            k.beside  = q.da != nullptr;
            if (!q.dgate)
                k.b[0].data = dg + half;
            k.b[0].batches = (int64_t)q.NB * k.results;
            k.out[0]    = q.dgate ? q.dgate : q.dup;
            k.out_dt[0] = q.dgate ? q.dgate_dt : q.dup_dt;
            k.out[1]    = k.results == 2 ? q.dup : nullptr;
            k.out_dt[1] = q.dup_dt;
            k.undo      = f16 ? undo : nullptr;
            k.ld        = q.W;
            k.name      = "gated_backward_pair_f16";
            TB200_TRY(pair_launch(ctx, k));
        }
    }
    return TB200_OK;
}

// fp32: both projections into scratch, G's batches and then U's, in one launch where the weights are one matrix each
tb200_status projections_f32(tb200_ctx* ctx, const GatedProblem& q, float* gu)
{
    const float *a = reinterpret_cast<const float*>(q.a), *gate = reinterpret_cast<const float*>(q.gate), *up = reinterpret_cast<const float*>(q.up);
    if (q.NB == 1)
        return sgemm_f32_two_launch(ctx, a, gate, up, gu, gu + q.H * q.W, (int)q.H, q.C, q.W);
    TB200_TRY(sgemm_f32_launch(ctx, a, gate, gu, q.NB, (int)q.H, q.C, q.W));
    return sgemm_f32_launch(ctx, a, up, gu + (int64_t)q.NB * q.H * q.W, q.NB, (int)q.H, q.C, q.W);
}

// fp32: one row past streamed weights; more as the two projections by the fp32 product, then a pass over them
tb200_status gated_f32(tb200_ctx* ctx, const GatedProblem& q)
{
    if (q.H == 1 && q.NB <= 65535)
        return gated_rows_f32_launch(ctx, q);
    const int64_t n = q.NB * q.H * q.W;
    TB200_TRY(ensure_scratch(ctx, (size_t)n * 8));
    float* const gu = reinterpret_cast<float*>(ctx->scratch);
    TB200_TRY(projections_f32(ctx, q, gu));
    TB200_TRY(gate_f32_launch(ctx, gu, gu + n, reinterpret_cast<float*>(q.out), n, q.act));
    return post_launch(ctx, "gated_f32", 0);
}

// Its gradients: the fp32 product takes its second operand as [K][columns], so what lies the other way is transposed into scratch.
tb200_status gated_backward_f32(tb200_ctx* ctx, const GatedProblem& q)
{
    const int64_t rows = q.NB * q.H, n = rows * q.W, weights = (int64_t)q.C * q.W;
    const bool weights_too = q.dgate || q.dup;
    Carver c;
    float *g = nullptr, *u = nullptr, *both = nullptr, *bt = nullptr, *at = nullptr;
    for (int pass = 0; pass < 2; pass++)
    {
        g    = reinterpret_cast<float*>(c.take((size_t)n * 8));
        u    = g + n;
        both = reinterpret_cast<float*>(c.take(q.da ? (size_t)n * 8 : 0));
        bt   = reinterpret_cast<float*>(c.take(q.da ? (size_t)q.NB * weights * 8 : 0));
        at   = reinterpret_cast<float*>(c.take(weights_too ? (size_t)rows * q.C * 4 : 0));
        if (!pass)
        {
            TB200_TRY(ensure_scratch(ctx, c.used));
            c      = Carver();
            c.base = reinterpret_cast<uint8_t*>(ctx->scratch);
        }
    }
    const float *a = reinterpret_cast<const float*>(q.a), *gate = reinterpret_cast<const float*>(q.gate), *up = reinterpret_cast<const float*>(q.up);
    Transposes t;
    if (q.da)
    {
        t.add(gate, bt, q.NB, q.C, q.W, 2 * weights);
        t.add(up, bt + weights, q.NB, q.C, q.W, 2 * weights);
    }
    if (weights_too)
        t.add(a, at, q.NB, q.H, q.C, q.H * q.C);
    TB200_TRY(transposes_f32_launch(ctx, t));
    TB200_TRY(projections_f32(ctx, q, g));
    TB200_TRY(grad_f32_launch(ctx, g, u, reinterpret_cast<const float*>(q.dout), q.da ? both : nullptr, rows, q.W, q.act));
    if (q.da)
        TB200_TRY(sgemm_f32_launch(ctx, both, bt, reinterpret_cast<float*>(q.da), q.NB, (int)q.H, 2 * q.W, q.C));
    if (weights_too)
    {
        float *const dgate = reinterpret_cast<float*>(q.dgate), *const dup = reinterpret_cast<float*>(q.dup);
        if (dgate && dup && q.NB == 1)
            TB200_TRY(sgemm_f32_two_launch(ctx, at, g, u, dgate, dup, q.C, (int)q.H, q.W));
        else if (dgate || dup)
        {
            if (dgate)
                TB200_TRY(sgemm_f32_launch(ctx, at, g, dgate, q.NB, q.C, (int)q.H, q.W));
            if (dup)
                TB200_TRY(sgemm_f32_launch(ctx, at, u, dup, q.NB, q.C, (int)q.H, q.W));
        }
    }
    return post_launch(ctx, "gated_backward_f32", 0);
}

// 4-bit weights: few rows multiply whole numbers and scale the sums; more take the weights' values in a's type, as a tile needs them.  Many fp32
// rows go through fp32 values laid out in scratch.
tb200_status w4_launch(tb200_ctx* ctx, const W4Problem& q)
{
    const bool f32      = q.dt == TB200_FP32;
    const int parts     = f32 ? 3 : 1;
    const int64_t xpitch = round_up(q.C, 8);
    const int64_t wpitch = round_up((q.C + 1) / 2, 16);
    const bool few       = f32 ? q.M * parts <= kFewParts : q.M <= kFewRows;
    const bool copy_x    = !f32 && q.C % 8 != 0;
    const int64_t n      = q.M * q.W;
    Carver c;
    void *x = nullptr, *w[2] = {}, *proj[2] = {}, *partial = nullptr;
    for (int pass = 0; pass < 2; pass++)
    {
        x = c.take(few && f32 ? (size_t)q.M * 3 * xpitch * 2 : copy_x ? (size_t)q.M * xpitch * 2 : 0);
        for (int i = 0; i < q.mats; i++)
        {
            w[i]    = c.take(!few && f32 ? (size_t)q.C * q.W * 4 : q.w[i].pitch % 16 ? (size_t)q.W * wpitch : 0);
            proj[i] = c.take(!few && f32 && q.mats == 2 ? (size_t)n * 4 : 0);
        }
        partial = c.take(few ? w4_rows_partial_bytes(ctx, q.M * parts) : 0);
        if (!pass)
        {
            if (c.used)
                TB200_TRY(ensure_scratch(ctx, c.used));
            c      = Carver();
            c.base = reinterpret_cast<uint8_t*>(ctx->scratch);
        }
    }
    if (!few && f32)
    {
        TB200_TRY(w4_dense_launch(ctx, q.w, q.mats, q.C, q.W, q.group, w));
        for (int i = 0; i < q.mats; i++)
            TB200_TRY(sgemm_f32_launch(ctx, reinterpret_cast<const float*>(q.a), reinterpret_cast<const float*>(w[i]),
                                       reinterpret_cast<float*>(q.mats == 2 ? proj[i] : q.out), 1, (int)q.M, q.C, q.W));
        if (q.mats == 2)
            TB200_TRY(gate_f32_launch(ctx, reinterpret_cast<const float*>(proj[0]), reinterpret_cast<const float*>(proj[1]), reinterpret_cast<float*>(q.out), n,
                                      q.act));
        return post_launch(ctx, q.mats == 2 ? "gated_w4_f32" : "matmul_w4_f32", 0);
    }
    W4Problem r = q;
    RowCopies copies;
    for (int i = 0; i < q.mats; i++)
        if (q.w[i].pitch % 16)
        {
            copies.add(q.w[i].data, w[i], q.W, (q.C + 1) / 2, q.w[i].pitch, wpitch);
            r.w[i].data  = reinterpret_cast<const uint8_t*>(w[i]);
            r.w[i].pitch = wpitch;
        }
    if (f32)
        copies.add(q.a, x, q.M, (int64_t)q.C * 4, (int64_t)q.C * 4, xpitch * 2, true);
    else if (copy_x)
        copies.add(q.a, x, q.M, (int64_t)q.C * 2, (int64_t)q.C * 2, xpitch * 2);
    TB200_TRY(row_copies_launch(ctx, copies));
    if (few)
        return w4_rows_launch(ctx, r, f32 || copy_x ? x : q.a, f32 || copy_x ? xpitch : q.C, parts, f32 || q.dt == TB200_BF16,
                              reinterpret_cast<float*>(partial));
    PairProduct k;
    memset(&k, 0, sizeof(k));
    k.dt        = q.dt;
    k.kind      = q.mats == 2 ? PAIR_GATED : PAIR_PLAIN;
    k.a         = operand(q.a, q.C, q.M, 1, x);
    k.w4        = r.w;
    k.group     = q.group;
    k.rows      = (int)q.M;
    k.cols      = q.W;
    k.K         = q.C;
    k.phases    = 1;
    k.NB        = 1;
    k.results   = 1;
    k.act       = q.act;
    k.out[0]    = q.out;
    k.out_dt[0] = k.out_dt[1] = q.out_dt;
    k.ld        = q.W;
    k.name      = q.mats == 2 ? "gated_w4_pair" : "matmul_w4_pair";
    return pair_launch(ctx, k);
}

// A sum over nothing is zero in every type.
tb200_status write_zeros(tb200_ctx* ctx, const tb200_tensor* t)
{
    if (t && t->bytes)
        TB200_CUDA_CHECK(ctx, cudaMemsetAsync(t->data, 0, t->bytes, ctx->stream));
    return TB200_OK;
}

tb200_status w4_entry(tb200_ctx* ctx, const char* op, const tb200_tensor* a, const tb200_w4* const* mats, int nmats, int activation,
                      tb200_tensor* output)
{
    const std::string why = check_w4(op, a, mats, nmats, activation, output);
    TB200_ERROR_IF(ctx, !why.empty(), "%s", why.c_str());
    if (numel(output) == 0)
        return TB200_OK;
    cache_note_write(ctx, output->data, output->bytes);
    if (a->shape[2] == 0)
        return write_zeros(ctx, output);
    W4Problem q;
    memset(&q, 0, sizeof(q));
    q.dt     = a->dtype;
    q.out_dt = output->dtype;
    q.a      = a->data;
    q.M      = (int64_t)a->shape[0] * a->shape[1];
    q.C      = a->shape[2];
    q.W      = output->shape[2];
    q.group  = mats[0]->group;
    q.mats   = nmats;
    q.act    = activation;
    q.out    = output->data;
    for (int i = 0; i < nmats; i++)
    {
        q.w[i].data     = reinterpret_cast<const uint8_t*>(mats[i]->data->data);
        q.w[i].pitch    = mats[i]->data->shape[1];
        q.w[i].scale    = mats[i]->scale->data;
        q.w[i].scale_dt = mats[i]->scale->dtype;
        q.w[i].zero     = mats[i]->zero ? reinterpret_cast<const int8_t*>(mats[i]->zero->data) : nullptr;
    }
    // (scales of any width are read as one row, whose elements have 32-bit coordinates)
    const int64_t groups = ((int64_t)q.C + q.group - 1) / q.group;
    const bool tiled     = ctx->policy == 0 && tiles_reach(1, q.M, q.C, q.W, false) && groups * q.W < (1LL << 31) - 256;
    return tiled ? w4_launch(ctx, q) : w4_direct_launch(ctx, q);
}

GatedProblem gated_problem(const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up, int activation)
{
    GatedProblem q;
    memset(&q, 0, sizeof(q));
    const bool shared = gate->shape[0] == 1;    // one matrix: the batches' rows are rows of one product
    q.dt   = a->dtype;
    q.a    = a->data;
    q.gate = gate->data;
    q.up   = up->data;
    q.NB   = shared ? 1 : a->shape[0];
    q.H    = shared ? (int64_t)a->shape[0] * a->shape[1] : a->shape[1];
    q.C    = a->shape[2];
    q.W    = gate->shape[2];
    q.act  = activation;
    return q;
}

}    // namespace

extern "C" tb200_status tb200_matmul_w4(tb200_ctx* ctx, const tb200_tensor* a, const tb200_w4* b, tb200_tensor* output)
{
    if (!ctx)
        return TB200_ERROR;
    TB200_ENTER(ctx);
    return guarded(ctx, [&] { return w4_entry(ctx, "matmul_w4", a, &b, 1, 0, output); });
}

extern "C" tb200_status tb200_matmul_gated_w4(tb200_ctx* ctx, const tb200_tensor* a, const tb200_w4* gate, const tb200_w4* up,
                                              int32_t activation, tb200_tensor* output)
{
    if (!ctx)
        return TB200_ERROR;
    TB200_ENTER(ctx);
    const tb200_w4* mats[2] = { gate, up };
    return guarded(ctx, [&] { return w4_entry(ctx, "matmul_gated_w4", a, mats, 2, activation, output); });
}

extern "C" tb200_status tb200_matmul_gated(tb200_ctx* ctx, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up,
                                           int32_t activation, tb200_tensor* output)
{
    if (!ctx)
        return TB200_ERROR;
    TB200_ENTER(ctx);
    return guarded(ctx, [&]() -> tb200_status {
        const std::string why = check_gated("matmul_gated", a, gate, up, activation, output, "output");
        TB200_ERROR_IF(ctx, !why.empty(), "%s", why.c_str());
        const std::string out_why = check_gated_output("matmul_gated", a, gate, up, output);
        TB200_ERROR_IF(ctx, !out_why.empty(), "%s", out_why.c_str());
        if (numel(output) == 0)
            return TB200_OK;
        cache_note_write(ctx, output->data, output->bytes);
        if (a->shape[2] == 0)
            return write_zeros(ctx, output);
        GatedProblem q = gated_problem(a, gate, up, activation);
        q.out          = output->data;
        q.out_dt       = output->dtype;
        if (ctx->policy == 0 && tiles_reach(q.NB, q.H, q.C, q.W, false))
            return q.dt == TB200_FP32 ? gated_f32(ctx, q) : gated_pair(ctx, q);
        return gated_direct_launch(ctx, q);
    });
}

extern "C" tb200_status tb200_matmul_gated_backward(tb200_ctx* ctx, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up,
                                                    const tb200_tensor* grad_output, int32_t activation, tb200_tensor* grad_a,
                                                    tb200_tensor* grad_gate, tb200_tensor* grad_up)
{
    if (!ctx)
        return TB200_ERROR;
    TB200_ENTER(ctx);
    return guarded(ctx, [&]() -> tb200_status {
        const std::string why = check_gated("matmul_gated_backward", a, gate, up, activation, grad_output, "grad_output");
        TB200_ERROR_IF(ctx, !why.empty(), "%s", why.c_str());
        const std::string grad_why = check_gated_grads("matmul_gated_backward", a, gate, up, grad_output, grad_a, grad_gate, grad_up);
        TB200_ERROR_IF(ctx, !grad_why.empty(), "%s", grad_why.c_str());
        tb200_tensor* grads[3] = { grad_a, grad_gate, grad_up };
        for (tb200_tensor* g : grads)
            if (g && g->bytes)
                cache_note_write(ctx, g->data, g->bytes);
        if (numel(a) == 0 || numel(gate) == 0)
        {
            for (tb200_tensor* g : grads)
            {
                const tb200_status st = write_zeros(ctx, g);
                if (st != TB200_OK)
                    return st;
            }
            return TB200_OK;
        }
        GatedProblem q = gated_problem(a, gate, up, activation);
        q.dout         = grad_output->data;
        if (grad_a)
        {
            q.da    = grad_a->data;
            q.da_dt = grad_a->dtype;
        }
        if (grad_gate)
        {
            q.dgate    = grad_gate->data;
            q.dgate_dt = grad_gate->dtype;
        }
        if (grad_up)
        {
            q.dup    = grad_up->data;
            q.dup_dt = grad_up->dtype;
        }
        if (ctx->policy == 0 && tiles_reach(q.NB, q.H, q.C, q.W, true))
            return q.dt == TB200_FP32 ? gated_backward_f32(ctx, q) : gated_backward_pair(ctx, q);
        const size_t each     = (size_t)q.NB * q.H * q.W * sizeof(float);
        const tb200_status st = ensure_scratch(ctx, 2 * each);
        if (st != TB200_OK)
            return st;
        float* const dg = reinterpret_cast<float*>(ctx->scratch);
        return gated_backward_direct_launch(ctx, q, dg, dg + each / sizeof(float));
    });
}
