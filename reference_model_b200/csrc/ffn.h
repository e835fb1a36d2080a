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

// whether the tiled kernels' 32-bit indexes serve a product of these sizes (or its gradients)
bool tiles_reach(int64_t batches, int64_t rows, int64_t C, int64_t W, bool gradients);

// ---- ffn_direct.cu: one thread per result, any type and size
tb200_status w4_direct_launch(tb200_ctx* ctx, const W4Problem& q);
tb200_status gated_direct_launch(tb200_ctx* ctx, const GatedProblem& q);
// dg, du: fp32 scratch [NB][H][W] each
tb200_status gated_backward_direct_launch(tb200_ctx* ctx, const GatedProblem& q, float* dg, float* du);

// ---- ffn_pair.cu: 16-bit products on CTA pairs
// [batches][outer][inner] elements, rows `pitch` elements apart (a multiple of 8), 16-byte aligned
struct Matrix
{
    const void* data;
    int64_t inner, outer, batches, pitch;
};
enum PairKind : int
{
    PAIR_PLAIN = 0,
    PAIR_GATED = 1,    // f(A B0) (A B1)
    PAIR_GRAD  = 2     // dG and dU of the same from the output's gradient
};
struct PairProduct
{
    tb200_dtype dt;    // of the operands, FP16 or BF16
    PairKind kind;
    bool a_mn, b_mn;   // K across the operand's rows instead of along them
    Matrix a, b[2];
    int rows, cols;
    int64_t K;
    int phases;        // 2: K runs over a's first NB batches against b[0], then over the next NB against b[1]
    int NB;
    int results;       // PAIR_PLAIN, 2: b[0]'s batches NB .. 2 NB - 1 give out[1]
    int act;
    const void* dout;
    void* out[2];
    tb200_dtype out_dt[2];
    int64_t ld;        // elements from one result row to the next
    const W4Mat* w4;   // in b's place: 4-bit matrices, rows a multiple of 16 bytes apart (PAIR_PLAIN and PAIR_GATED, NB and phases 1)
    int group;
    bool beside;       // reads nothing that the launch of this kind directly before it writes: the two may run side by side
    float* peaks;        // PAIR_GRAD in FP16: where the launch leaves what its values reach (pair_peaks of them)
    const float* seen;   // ... a second launch of the same product, which looks at them and evaluates again where they call for a power of two,
    float* undo;         // ... and leaves what takes it back; PAIR_PLAIN: what results are multiplied by (or null)
    const char* name;
};
tb200_status pair_launch(tb200_ctx* ctx, const PairProduct& q);
int64_t pair_peaks(const tb200_ctx* ctx);

// ---- gated_rows.cu: PAIR_GATED with K across b's rows and few rows of a (weights read once)
tb200_status gated_rows_launch(tb200_ctx* ctx, const PairProduct& q);

// ---- gated_rows_f32.cu: the fp32 gated product of one row
tb200_status gated_rows_f32_launch(tb200_ctx* ctx, const GatedProblem& q);

// ---- w4_rows.cu: up to 32 16-bit rows against 4-bit weights
// (64, where they are parts of fp32 rows.)
// x: a's rows in 16 bits, `x_pitch` elements apart (a multiple of 8), 16-byte aligned; fp32 rows as three bf16 rows each (parts 3,
// bf16).  The weights' pitch is a multiple of 16 bytes.
tb200_status w4_rows_launch(tb200_ctx* ctx, const W4Problem& q, const void* x, int64_t x_pitch, int parts, bool bf16, float* partial);
size_t w4_rows_partial_bytes(const tb200_ctx* ctx, int64_t xrows);

// ---- ffn_small.cu: copies
// rows of `inner` bytes, `in_pitch` apart, to rows `pitch` (a multiple of 16) apart with zeros behind them; split: fp32 rows to three bf16 rows each
// whose sum they are.  Up to eight copies in a launch.
struct RowCopy
{
    const uint8_t* in;
    uint8_t* out;
    int64_t inner, in_pitch, pitch, bytes;    // bytes: of the whole operand
    int word, split;
};
struct RowCopies
{
    RowCopy copy[8];
    int64_t items[8];    // of sixteen result bytes, up to and with each copy
    int n = 0;
    void add(const void* in, void* out, int64_t rows, int64_t inner, int64_t in_pitch, int64_t pitch, bool split = false);
};
tb200_status row_copies_launch(tb200_ctx* ctx, const RowCopies& q);
// fp32 values [C][W] of one or two 4-bit matrices
tb200_status w4_dense_launch(tb200_ctx* ctx, const W4Mat* w, int mats, int C, int W, int group, void* const* out);
tb200_status gate_f32_launch(tb200_ctx* ctx, const float* g, const float* u, float* out, int64_t n, int act);
// g and u hold dG and dU afterwards, `both` (or null) the two side by side
tb200_status grad_f32_launch(tb200_ctx* ctx, float* g, float* u, const float* d, float* both, int64_t rows, int W, int act);
// [batches][R][C] to [batches][C][R], results `out_batch` elements apart; up to three in a launch
struct Transpose
{
    const float* in;
    float* out;
    int64_t R, C, out_batch;
};
struct Transposes
{
    Transpose job[3];
    int64_t tiles[3];    // up to and with each
    int n = 0;
    void add(const float* in, float* out, int64_t batches, int64_t R, int64_t C, int64_t out_batch);
};
tb200_status transposes_f32_launch(tb200_ctx* ctx, const Transposes& q);
}    // namespace ffn
}    // namespace tb200
