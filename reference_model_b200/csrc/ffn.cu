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

size_t aligned(size_t bytes)
{
    return (bytes + 255) & ~(size_t)255;
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
    return w4_direct_launch(ctx, q);
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
        const size_t each     = aligned((size_t)q.NB * q.H * q.W * sizeof(float));
        const tb200_status st = ensure_scratch(ctx, 2 * each);
        if (st != TB200_OK)
            return st;
        float* const dg = reinterpret_cast<float*>(ctx->scratch);
        return gated_backward_direct_launch(ctx, q, dg, reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ctx->scratch) + each));
    });
}
