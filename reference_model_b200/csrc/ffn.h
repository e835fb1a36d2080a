// Feed-forward operators: MATMUL with 4-bit weights, the gated product of two projections and its backward pass.  Argument rules
// (host only, no CUDA call) and what the kernels of ffn_*.cu take.
#pragma once
#include <cstdint>
#include <string>

#include "common.h"

namespace tb200
{
namespace ffn
{

// One 4-bit matrix: rows of bytes (two elements each), scales and zero points [groups][W]
struct W4Mat
{
    const uint8_t* data;
    int64_t pitch;    // bytes from one row to the next
    const void* scale;
    const int8_t* zero;    // or null
    tb200_dtype scale_dt;
};

struct W4Problem
{
    tb200_dtype dt, out_dt;
    const void* a;    // [M][C]
    int64_t M;
    int C, W, group, mats;    // mats 2: the gated product of the two
    W4Mat w[2];
    int act;
    void* out;    // [M][W]
};

struct GatedProblem
{
    tb200_dtype dt, out_dt;
    const void *a, *gate, *up;    // a [NB][H][C], weights [NB][C][W]
    int NB;
    int64_t H;
    int C, W, act;
    void* out;           // forward: [NB][H][W]
    const void* dout;    // backward: [NB][H][W], and the gradients that are asked for (any may be null)
    void *da, *dgate, *dup;
    tb200_dtype da_dt, dgate_dt, dup_dt;
};

// ---- argument rules: a message, empty when the call stands
std::string check_w4(const char* op, const tb200_tensor* a, const tb200_w4* const* mats, int nmats, int activation, const tb200_tensor* output);
std::string check_gated(const char* op, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up, int activation,
                        const tb200_tensor* like_out, const char* like_name);
std::string check_gated_output(const char* op, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up, const tb200_tensor* output);
std::string check_gated_grads(const char* op, const tb200_tensor* a, const tb200_tensor* gate, const tb200_tensor* up, const tb200_tensor* dout,
                              const tb200_tensor* da, const tb200_tensor* dgate, const tb200_tensor* dup);

// ---- ffn_direct.cu: one thread per result, any type and size
tb200_status w4_direct_launch(tb200_ctx* ctx, const W4Problem& q);
tb200_status gated_direct_launch(tb200_ctx* ctx, const GatedProblem& q);
// dg, du: fp32 scratch [NB][H][W] each
tb200_status gated_backward_direct_launch(tb200_ctx* ctx, const GatedProblem& q, float* dg, float* du);

}    // namespace ffn
}    // namespace tb200
