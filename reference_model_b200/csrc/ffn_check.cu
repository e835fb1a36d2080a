// Argument rules of the feed-forward operators.  Host code without a CUDA call, so that it can be tested without a GPU.
#include "ffn.h"

#include <cstdarg>
#include <cstdio>

namespace tb200
{
namespace ffn
{
namespace
{

std::string say(const char* fmt, ...)
{
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return buf;
}

bool overlap(const tb200_tensor* x, const tb200_tensor* y)
{
    if (!x || !y || !x->bytes || !y->bytes)
        return false;
    const uintptr_t a = reinterpret_cast<uintptr_t>(x->data), b = reinterpret_cast<uintptr_t>(y->data);
    return a < b + y->bytes && b < a + x->bytes;
}

bool activation_known(int act)
{
    return act >= TB200_ACT_SILU && act <= TB200_ACT_SIGMOID;
}

}    // namespace

std::string check_w4(const char* op, const tb200_tensor* a, const tb200_w4* const* mats, int nmats, int activation, const tb200_tensor* output)
{
    if (!a || !output)
        return say("%s: null operand", op);
    for (int i = 0; i < nmats; i++)
        if (!mats[i] || !mats[i]->data || !mats[i]->scale)
            return say("%s: null operand", op);
    if (a->rank != 3 || output->rank != 3)
        return say("%s: a and output must be rank 3", op);
    if (!a->contiguous || !output->contiguous)
        return say("%s: zero-copy views are accepted only as the CONV2D input; this operand must be contiguous", op);
    if (!dtype_is_float(a->dtype))
        return say("%s: a must be FP16, BF16 or FP32", op);
    if (output->dtype != a->dtype && output->dtype != TB200_FP32)
        return say("%s: output dtype must be a's or FP32", op);
    const int N = a->shape[0], H = a->shape[1], C = a->shape[2], W = output->shape[2];
    if (output->shape[0] != N || output->shape[1] != H)
        return say("%s: output must have a's first two dimensions", op);
    if (nmats == 2 && !activation_known(activation))
        return say("%s: unknown activation %d", op, activation);
    for (int i = 0; i < nmats; i++)
    {
        const tb200_tensor *d = mats[i]->data, *s = mats[i]->scale, *z = mats[i]->zero;
        const int group = mats[i]->group;
        if (d->dtype != TB200_INT8 && d->dtype != TB200_UINT8)
            return say("%s: 4-bit weights are bytes (INT8 or UINT8 tensors)", op);
        if (d->rank != 2 || s->rank != 2 || (z && z->rank != 2))
            return say("%s: 4-bit weights, their scales and zero points must be rank 2", op);
        if (!d->contiguous || !s->contiguous || (z && !z->contiguous))
            return say("%s: zero-copy views are accepted only as the CONV2D input; this operand must be contiguous", op);
        if (d->shape[0] != W)
            return say("%s: the weights must have a row for each of the output's %d columns", op, W);
        if (d->shape[1] < C / 2 + C % 2)
            return say("%s: a weight row of %d bytes does not hold %d elements", op, d->shape[1], C);
        if (group < 1 || (group % 32 != 0 && group < C))
            return say("%s: a group must be a multiple of 32 elements, or hold a whole row", op);
        const int groups = (int)(((int64_t)C + group - 1) / group);
        if (!dtype_is_float(s->dtype))
            return say("%s: scales must be FP16, BF16 or FP32", op);
        if (s->shape[0] != groups || s->shape[1] != W)
            return say("%s: scales must be [%d,%d]", op, groups, W);
        if (z && (z->dtype != TB200_INT8 || z->shape[0] != groups || z->shape[1] != W))
            return say("%s: zero points must be INT8 [%d,%d]", op, groups, W);
        if (overlap(output, d) || overlap(output, s) || overlap(output, z))
            return say("%s: the output overlaps an operand", op);
    }
    if (nmats == 2 && mats[0]->group != mats[1]->group)
        return say("%s: both matrices must have the same group", op);
    if (overlap(output, a))
        return say("%s: the output overlaps an operand", op);
    return std::string();
}

std::string check_gated(const char* op, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up, int activation,
                        const tb200_tensor* like_out, const char* like_name)
{
    if (!a || !gate || !up || !like_out)
        return say("%s: null operand", op);
    if (a->rank != 3 || gate->rank != 3 || up->rank != 3 || like_out->rank != 3)
        return say("%s: operands must be rank 3", op);
    if (!a->contiguous || !gate->contiguous || !up->contiguous || !like_out->contiguous)
        return say("%s: zero-copy views are accepted only as the CONV2D input; this operand must be contiguous", op);
    if (!dtype_is_float(a->dtype))
        return say("%s: operands must be FP16, BF16 or FP32", op);
    if (gate->dtype != a->dtype || up->dtype != a->dtype)
        return say("%s: operand dtypes differ", op);
    const int N = a->shape[0], H = a->shape[1], C = a->shape[2], W = gate->shape[2];
    if (gate->shape[0] != N && gate->shape[0] != 1)
        return say("%s: the weights must have one matrix, or one for each of a's %d batches", op, N);
    if (gate->shape[1] != C)
        return say("%s: gate.shape[1] should match a.shape[2]", op);
    for (int i = 0; i < 3; i++)
        if (up->shape[i] != gate->shape[i])
            return say("%s: gate and up must have the same shape", op);
    if (like_out->shape[0] != N || like_out->shape[1] != H || like_out->shape[2] != W)
        return say("%s: %s must be [%d,%d,%d]", op, like_name, N, H, W);
    if (!activation_known(activation))
        return say("%s: unknown activation %d", op, activation);
    return std::string();
}

std::string check_gated_output(const char* op, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up, const tb200_tensor* output)
{
    if (output->dtype != a->dtype && output->dtype != TB200_FP32)
        return say("%s: output dtype must be a's or FP32", op);
    if (overlap(output, a) || overlap(output, gate) || overlap(output, up))
        return say("%s: the output overlaps an operand", op);
    return std::string();
}

// Indexes step past the last element, by less than a tile; tiles, of 128 rows and 64 columns of a gated product (128 of another) at least, are
// counted in 32 bits with room for a grid's step.
bool tiles_reach(int64_t batches, int64_t rows, int64_t C, int64_t W, bool gradients)
{
    auto tiles = [](int64_t n, int64_t size) { return (double)((n + size - 1) / size); };
    const double most = 1 << 30;
    return rows <= (1 << 30) && C <= (1 << 30) && W <= (1 << 29) && batches * tiles(rows, 128) * tiles(W, 64) <= most &&
           (!gradients || (batches * tiles(rows, 128) * tiles(C, 128) <= most && 2 * batches * tiles(C, 128) * tiles(W, 128) <= most));
}

std::string check_gated_grads(const char* op, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up, const tb200_tensor* dout,
                              const tb200_tensor* da, const tb200_tensor* dgate, const tb200_tensor* dup)
{
    if (dout->dtype != a->dtype)
        return say("%s: the output's gradient must have the operands' dtype", op);
    const tb200_tensor* g[3]    = { da, dgate, dup };
    const tb200_tensor* like[3] = { a, gate, up };
    const char* names[3]        = { "grad_a", "grad_gate", "grad_up" };
    const tb200_tensor* in[4]   = { a, gate, up, dout };
    if (!da && !dgate && !dup)
        return say("%s: no gradient is asked for", op);
    for (int i = 0; i < 3; i++)
    {
        if (!g[i])
            continue;
        if (!g[i]->contiguous)
            return say("%s: zero-copy views are accepted only as the CONV2D input; this operand must be contiguous", op);
        if (g[i]->dtype != a->dtype && g[i]->dtype != TB200_FP32)
            return say("%s: %s must have the operands' dtype or FP32", op, names[i]);
        bool same = g[i]->rank == 3;
        for (int k = 0; same && k < 3; k++)
            same = g[i]->shape[k] == like[i]->shape[k];
        if (!same)
            return say("%s: %s must have its operand's shape", op, names[i]);
        for (int k = 0; k < 4; k++)
            if (overlap(g[i], in[k]))
                return say("%s: %s overlaps an operand", op, names[i]);
        for (int k = 0; k < i; k++)
            if (overlap(g[i], g[k]))
                return say("%s: two gradients overlap", op);
    }
    return std::string();
}

}    // namespace ffn
}    // namespace tb200
