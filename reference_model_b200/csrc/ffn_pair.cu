// 16-bit products of the feed-forward operators on CTA pairs (tcgen05 cta_group::2): the gated product of two projections, the
// gradients of its projections, the plain products of the backward pass, and both forms with 4-bit weights.
//
// A pair owns a 256-row tile of 256 accumulator columns.  Each CTA loads its own 128 rows of A and its own 128 columns of B per 64
// elements of K; the tensor cores of both read B from both.  For the gated product the first CTA's 128 columns are the gate's and
// the second's the same 128 columns of the up projection: one pass over A serves both, a thread of the epilogue finds G in
// accumulator column j and U in column 128 + j of its own row, and neither projection leaves the chip.  The other products
// take 256 neighbouring columns.  Either operand may have K along its rows (the tile's K runs are contiguous) or across them
// (gradients of weights: a^T x dG reads both as they lie).  grad_a is one product over both projections: K runs over dG against
// the gate, then over dU against the up projection, in the same accumulator.
// Tiles go in groups of `group_m` rows of tiles, rows fastest: a wave's tiles then share few columns of B and the group's A stays
// in L2 while B streams by once per group.
// Sums are fp32 in tensor memory; results are rounded once, where they are stored.
//
// 4-bit weights (W4): the ring's stages receive a chunk's nibbles (4 KB where its values take 16), and three groups of four warps make the values in
// their place, a thread a row of 64 elements, chunk by chunk in turn; the tensor cores wait for those as for A's bytes.  Laid out in
// memory by a pass before, the values cost 10 us for 4096 x 4096; made here they pass through shared memory once more (a chunk takes a
// pair 690 cycles instead of 520), which evens out at about 2000 rows.  Two groups were 10 to 20 % slower.  The gated product carries what the
// rounding of a value left as a second 16-bit number and a second MMA: rounded once, two projections' weights put 1.6 times the
// output's own rounding into the result (100 x 2048 x 8192: 17.4 us so, 21.6 with both; 1000 rows 62 and 88).
//
// Measured: gated 4096 x 4096 x 8192 bf16 344 us (1600 TFLOP/s, the rate of the library's product for a short time; power holds the
// clock down when it goes on), backward of the same 1105 us (1490); 777 x 4096 x 4096 with 4-bit weights 35 us (750: 64 of 74 pairs, a quarter of the rows
// padding; tensor pipe 61 % busy); gated 788 x 1000 x 1416 fp16 14.5 us, its backward at 394 x 1024 x 2048 34 us (chains of launches
// of a few chunks: latencies of set-up, first copies, epilogue and exchange).
#include <algorithm>
#include <cstring>
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
namespace
{

constexpr int kEpiWarps = 8;
constexpr int kRawBytes    = 128 * 32;            // 128 rows x 64 elements of 4-bit weights
constexpr int kChunk    = 16384;                  // 128 rows (or columns) x 64 elements of K

// Pairs of CTAs (PAIR) with tiles of 256 rows and 256 accumulator columns, or CTAs by themselves with 128 x 128; one CTA to an SM.
// W4: 4-bit weights; LOW: their values as two 16-bit numbers each.
template <bool PAIR, bool W4 = false, bool LOW = false>
struct Shape
{
    static constexpr int kGroups  = !W4 ? 0 : LOW ? 2 : 3;                   // of four warps that make the values
    static constexpr int kThreads = 64 + 32 * (kEpiWarps + 4 * kGroups);     // TMA warp, MMA warp, epilogue, and those
    static constexpr int kStages = LOW ? 4 : PAIR && !W4 ? 3 : 6;
    static_assert(!W4 || kStages % kGroups == 0, "a group keeps to its stages");
    static constexpr int kCtas = PAIR ? 2 : 1;
    static constexpr int kRows = 128 * kCtas, kCols = PAIR ? 256 : 128;    // of a tile
    static constexpr int kSub  = PAIR && !W4 ? 2 : 1;                      // chunks per stage
    static constexpr int kStage = (LOW ? 3 : 2 * kSub) * kChunk;           // each CTA holds 128 rows of A and 128 columns of B
    // (with the static part all of an SM's: a CTA that waits for tensor memory never shares an SM with another kernel's that holds some)
    static constexpr int kSmem  = 208 * 1024;
    static_assert(kStages * kStage + 1024 <= kSmem, "the ring fits");
    static constexpr int kTmemCols = 2 * kCols;
    static constexpr int kRedLd    = kCols + 4;    // row pitch of a tile's sums in shared memory: a warp's stores meet every bank
};

enum : int
{
    EPI_PLAIN = 0,    // out[idx] = accumulator
    EPI_GATED = 1,    // out = f(G) U
    EPI_GRAD  = 2     // dG and dU from the output's gradient
};

struct Params
{
    CUtensorMap tmA, tmB0, tmB1;
    int rows, cols;    // of a result matrix
    int tiles_m, tiles_n, num_tiles, group_m;
    int chunks, phases;    // K chunks of a phase
    int splits;            // CTAs of a cluster that share a tile's K (CTAs by themselves only)
    int NB;                // batches of A's and B's own
    int beside;
    int act, bf16;
    tb200_dtype out_dt;
    uint32_t idesc;
    uint64_t a_desc_hi, b_desc_hi;
    void *out0, *out1;     // results [NB][rows][ld]; plain products: batch NB + n goes to out1
    tb200_dtype out1_dt;
    int64_t ld;
    int vec;               // whole 16-element runs of a result's row may be stored 32 bytes at a time (2), 16 (1), or not (0)
    int even;              // whole pairs of elements in every row, at 4-byte addresses
    const void* dout;      // [NB][rows][cols]
    int dout_vec;          // its rows may be read 16 bytes at a time
    // 4-bit weights: tmB0 and tmB1 are [W][pitch] bytes, boxes of 32 bytes
    const void* scale[2];
    const int8_t* zero[2];
    tb200_dtype scale_dt[2];
    int K, groups;
    uint32_t group32;      // of 32 elements
    // The power of two under which fp16 holds dG and dU (range_scale).  Gradients, first launch: where each warp leaves the largest it has met;
    // second: those, and where the other products find what takes the power back.
    float* peaks;
    const float* seen;
    float* undo;
    long long wait_limit;
    int* status;
};

// fp16 has five bits of exponent: from 65520 on dG and dU would be infinite, and below 2^-14 they lose places.  Where the largest of a call is outside of
// what fp16 holds well, all are held under the power of two that brings it to 2^14 .. 2^15, and the products' fp32 sums are divided by it again, which
// rounds nothing.  Values below 2^-39 of the largest become 0 (2^-17 where no power is taken and the largest is near 2^-8).
__device__ __forceinline__ float range_scale(float peak)
{
    if (!(peak >= 65520.f || (peak > 0.f && peak < 0x1p-8f)))
        return 1.f;
    const int exponent = max((int)(__float_as_uint(peak) >> 23) - 127, -106);
    return __uint_as_float((uint32_t)(14 - exponent + 127) << 23);
}

// (what is not finite stays so under any power)
__device__ __forceinline__ void note_peak(float& peak, float x)
{
    const float v = fabsf(x);
    peak          = v <= 3.402823466e38f ? fmaxf(peak, v) : peak;
}

struct Tile
{
    int idx, m0, n0;
};

template <int EPI, bool PAIR>
__device__ __forceinline__ Tile decode(const Params& p, int tile)
{
    const int per = p.tiles_m * p.tiles_n;
    Tile t;
    t.idx         = tile / per;
    const int r   = tile - t.idx * per;
    const int grp = r / (p.group_m * p.tiles_n), first = grp * p.group_m;
    const int gm  = min(p.group_m, p.tiles_m - first);
    const int rr  = r - first * p.tiles_n;
    t.m0          = (first + rr % gm) * Shape<PAIR>::kRows;
    t.n0          = rr / gm * (EPI == EPI_PLAIN ? Shape<PAIR>::kCols : Shape<PAIR>::kCols / 2);
    return t;
}

// Sixteen neighbouring results of a row.
__device__ __forceinline__ void store_run(void* base, int64_t at, tb200_dtype dt, int n, int vec, const float (&v)[16])
{
    if (dt == TB200_FP32)
    {
        float* o = reinterpret_cast<float*>(base) + at;
        if (n == 16 && vec == 2)
        {
#pragma unroll
            for (int i = 0; i < 16; i += 8)
                ptx::st_global_v8(o + i, __float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]),
                                  __float_as_uint(v[i + 4]), __float_as_uint(v[i + 5]), __float_as_uint(v[i + 6]), __float_as_uint(v[i + 7]));
        }
        else if (n == 16 && vec == 1)
        {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4*>(o + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (i < n)
                    o[i] = v[i];
        }
        return;
    }
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        h[i] = pack2(v[2 * i], v[2 * i + 1], dt == TB200_BF16);
    uint16_t* o = reinterpret_cast<uint16_t*>(base) + at;
    if (n == 16 && vec == 2)
        ptx::st_global_v8(o, h[0], h[1], h[2], h[3], h[4], h[5], h[6], h[7]);
    else if (n == 16 && vec == 1)
    {
        *reinterpret_cast<uint4*>(o)     = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(o + 8) = make_uint4(h[4], h[5], h[6], h[7]);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i < n)
                o[i] = (uint16_t)((i & 1) ? (h[i >> 1] >> 16) : (h[i >> 1] & 0xffffu));
    }
}

template <int ACT>
__device__ __forceinline__ void gate_run(const uint32_t (&g)[16], const uint32_t (&u)[16], float (&o)[16])
{
#pragma unroll
    for (int i = 0; i < 16; i++)
        o[i] = act_value_16<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]);
}

template <int ACT>
__device__ __forceinline__ void gate_run_32(const uint32_t (&g)[16], const uint32_t (&u)[16], float (&o)[16])
{
#pragma unroll
    for (int i = 0; i < 16; i++)
        o[i] = act_value_32<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]);
}

template <int ACT>
__device__ __forceinline__ void grad_run(const uint32_t (&g)[16], const uint32_t (&u)[16], const float (&d)[16], float scale, float (&dg)[16], float (&du)[16])
{
#pragma unroll
    for (int i = 0; i < 16; i++)
    {
        float value, slope;
        act_slope_16<ACT>(__uint_as_float(g[i]), value, slope);
        dg[i] = d[i] * slope * __uint_as_float(u[i]) * scale;    // (the slope is 1.13 at most: in fp32 only the product itself can overflow)
        du[i] = d[i] * value * scale;
    }
}

// Sixteen neighbouring columns of a row of the tile, all sums there: results, activated and multiplied, or the two gradients.  The
// warp's lanes are 32 rows of the tile and call together: rows that may not be stored sixteen bytes at a time go through `stage` (32 x 17 words
// of the warp's own) and out sixteen neighbouring columns of two rows at a time (a row a lane, one element at a time, touched 32 sectors with every
// store: gradients of 6 x 280 x 2758 took 150 us).
template <int EPI>
__device__ __forceinline__ void finish_run(const Params& p, const Tile& t, int row, int run, const uint32_t (&g)[16], const uint32_t (&u)[16], float* stage,
                                           float scale, float& peak)
{
    const int m = t.m0 + row, col = t.n0 + run, n = min(16, p.cols - col);
    const bool valid = m < p.rows, together = p.vec == 0;
    if (!valid && !together)
        return;
    const int batch    = t.idx < p.NB ? t.idx : t.idx - p.NB;
    const int64_t orow = ((int64_t)batch * p.rows + m) * p.ld;
    auto emit          = [&](void* out, tb200_dtype dt, const float (&v)[16]) {
        if (!together)
        {
            store_run(out, orow + col, dt, n, p.vec, v);
            return;
        }
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 16; i++)
            stage[lane * 17 + i] = v[i];
        __syncwarp();
        if (p.even && dt != TB200_FP32)
        {
            // two elements at a time, four rows
#pragma unroll 4
            for (int i = 0; i < 8; i++)
            {
                const int r = 4 * i + (lane >> 3), c = (lane & 7) * 2;
                if (m - lane + r < p.rows && c < n)
                    *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(out) + orow + (int64_t)(r - lane) * p.ld + col + c) =
                        pack2(stage[r * 17 + c], stage[r * 17 + c + 1], dt == TB200_BF16);
            }
        }
        else
        {
#pragma unroll 4
            for (int i = 0; i < 16; i++)
            {
                const int r = 2 * i + (lane >> 4), c = lane & 15;
                if (m - lane + r < p.rows && c < n)
                    store_fp(out, orow + (int64_t)(r - lane) * p.ld + col + c, dt, stage[r * 17 + c]);
            }
        }
        __syncwarp();
    };
    if (EPI == EPI_PLAIN)
    {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++)
            v[i] = __uint_as_float(g[i]) * scale;
        emit(t.idx < p.NB ? p.out0 : p.out1, t.idx < p.NB ? p.out_dt : p.out1_dt, v);
    }
    else if (EPI == EPI_GATED)
    {
        float v[16];
        if (p.out_dt == TB200_FP32)
        {
            switch (p.act)
            {
                case TB200_ACT_SILU: gate_run_32<TB200_ACT_SILU>(g, u, v); break;
                case TB200_ACT_GELU: gate_run_32<TB200_ACT_GELU>(g, u, v); break;
                case TB200_ACT_GELU_TANH: gate_run_32<TB200_ACT_GELU_TANH>(g, u, v); break;
                case TB200_ACT_RELU: gate_run_32<TB200_ACT_RELU>(g, u, v); break;
                default: gate_run_32<TB200_ACT_SIGMOID>(g, u, v); break;
            }
        }
        else
        {
            switch (p.act)
            {
                case TB200_ACT_SILU: gate_run<TB200_ACT_SILU>(g, u, v); break;
                case TB200_ACT_GELU: gate_run<TB200_ACT_GELU>(g, u, v); break;
                case TB200_ACT_GELU_TANH: gate_run<TB200_ACT_GELU_TANH>(g, u, v); break;
                case TB200_ACT_RELU: gate_run<TB200_ACT_RELU>(g, u, v); break;
                default: gate_run<TB200_ACT_SIGMOID>(g, u, v); break;
            }
        }
        emit(p.out0, p.out_dt, v);
    }
    else
    {
        float d[16], dg[16], du[16];
        const uint16_t* const s = reinterpret_cast<const uint16_t*>(p.dout) + ((int64_t)batch * p.rows + m) * p.cols + col;
        if (valid && n == 16 && p.dout_vec)
        {
            const uint4 lo = *reinterpret_cast<const uint4*>(s), hi = *(reinterpret_cast<const uint4*>(s) + 1);
            const uint32_t w[8] = { lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w };
#pragma unroll
            for (int i = 0; i < 8; i++)
            {
                const float2 f = unpack2(w[i], p.bf16 != 0);
                d[2 * i]       = f.x;
                d[2 * i + 1]   = f.y;
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < 16; i++)
                d[i] = valid && i < n ? unpack2(s[i], p.bf16 != 0).x : 0.f;
        }
        switch (p.act)
        {
            case TB200_ACT_SILU: grad_run<TB200_ACT_SILU>(g, u, d, scale, dg, du); break;
            case TB200_ACT_GELU: grad_run<TB200_ACT_GELU>(g, u, d, scale, dg, du); break;
            case TB200_ACT_GELU_TANH: grad_run<TB200_ACT_GELU_TANH>(g, u, d, scale, dg, du); break;
            case TB200_ACT_RELU: grad_run<TB200_ACT_RELU>(g, u, d, scale, dg, du); break;
            default: grad_run<TB200_ACT_SIGMOID>(g, u, d, scale, dg, du); break;
        }
        if (p.peaks)
        {
#pragma unroll
            for (int i = 0; i < 16; i++)
            {
                note_peak(peak, dg[i]);
                note_peak(peak, du[i]);
            }
        }
        emit(p.out0, p.out_dt, dg);
        emit(p.out1, p.out_dt, du);
    }
}

__device__ __forceinline__ void store_quad(void* base, int64_t at, tb200_dtype dt, int n, int vec, const float (&v)[4])
{
    if (n == 4 && vec > 0)
    {
        if (dt == TB200_FP32)
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(base) + at) =
                make_uint2(pack2(v[0], v[1], dt == TB200_BF16), pack2(v[2], v[3], dt == TB200_BF16));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n)
            store_fp(base, at + i, dt, v[i]);
}

// The same for four columns, whichever thread has them.
template <int EPI>
__device__ __forceinline__ void finish_quad(const Params& p, const Tile& t, int row, int run, const float (&g)[4], const float (&u)[4], float scale, float& peak)
{
    const int m = t.m0 + row, col = t.n0 + run, n = min(4, p.cols - col);
    const int batch    = t.idx < p.NB ? t.idx : t.idx - p.NB;
    const int64_t orow = ((int64_t)batch * p.rows + m) * p.ld + col;
    if (EPI == EPI_PLAIN)
    {
        const float v[4] = { g[0] * scale, g[1] * scale, g[2] * scale, g[3] * scale };
        store_quad(t.idx < p.NB ? p.out0 : p.out1, orow, t.idx < p.NB ? p.out_dt : p.out1_dt, n, p.vec, v);
    }
    else if (EPI == EPI_GATED)
    {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = (p.out_dt == TB200_FP32 ? act_value_32(p.act, g[i]) : act_value_16(p.act, g[i])) * u[i];
        store_quad(p.out0, orow, p.out_dt, n, p.vec, v);
    }
    else
    {
        const int64_t at = ((int64_t)batch * p.rows + m) * p.cols + col;
        float dg[4], du[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            const float d = i < n ? load_fp(p.dout, at + i, p.bf16 ? TB200_BF16 : TB200_FP16) : 0.f;
            float value, slope;
            act_slope_16(p.act, g[i], value, slope);
            dg[i] = d * slope * u[i] * scale;
            du[i] = d * value * scale;
            if (p.peaks)
            {
                note_peak(peak, dg[i]);
                note_peak(peak, du[i]);
            }
        }
        store_quad(p.out0, orow, p.out_dt, n, p.vec, dg);
        store_quad(p.out1, orow, p.out_dt, n, p.vec, du);
    }
}

// Elements as bits, by one instruction into their register, so that the thread goes on without them (a conversion, or a choice between two
// loads' results, waited for each here: 2100 cycles a chunk).
__device__ __forceinline__ void load_bits(uint32_t& v, const uint8_t* at, bool wide)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.b32 %0, [%1];\n\t@!q ld.global.u16 %0, [%1];\n\t}"
                 : "=r"(v)
                 : "l"(at), "r"((int)wide));
}

__device__ __forceinline__ void load_zero(int& v, const int8_t* at, bool any)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\tmov.b32 %0, 0;\n\t@q ld.global.s8 %0, [%1];\n\t}" : "=r"(v) : "l"(at), "r"((int)any));
}

// A row's 64 elements of 4-bit weights (two sixteens of bytes) as 16-bit values in a chunk of B: 128 bytes, swizzled.  Values are rounded to the
// operands' type, once: by scales of that type (SAME) as they are, by others in fp32.  TAIL: `left` elements up to the end of K.
// LOW: a chunk further, what the rounding left (exactly, for SAME): a value is then as good as never rounded.
template <bool BF16, bool SAME, bool TAIL, bool LOW>
__device__ __forceinline__ void expand_row(const uint4 (&raw)[2], const uint32_t (&bits)[2], tb200_dtype scale_dt, const int (&zero)[2], int left, uint32_t dst, int row)
{
#pragma unroll
    for (int h = 0; h < 2; h++)
    {
        const uint32_t w[4] = { raw[h].x, raw[h].y, raw[h].z, raw[h].w };
        const uint32_t base = unpack_base<BF16>(zero[h]), s2 = bits[h] * 0x10001u;
        const float scale   = SAME ? 0.f : bits_fp(bits[h], scale_dt);
        // a value that overflows has no second number (infinity less infinity; SAME is not called where one may)
        const uint32_t keep = fabsf(scale) * 15.f < (BF16 ? 3.38e38f : 65504.f) ? 0xffffffffu : 0u;
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            uint32_t v[4], o[4];
            unpack8<BF16>(w[i], base, v);
            o[0] = __byte_perm(v[0], v[1], 0x5410);
            o[1] = __byte_perm(v[2], v[3], 0x5410);
            o[2] = __byte_perm(v[0], v[1], 0x7632);
            o[3] = __byte_perm(v[2], v[3], 0x7632);
            uint32_t low[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                const uint32_t whole = o[j];
                if (SAME)
                {
                    o[j] = BF16 ? fma2_bf16(whole, s2, 0x80008000u) : fma2_f16(whole, s2, 0x80008000u);
                    if (LOW)
                        low[j] = BF16 ? fma2_bf16(whole, s2, o[j] ^ 0x80008000u) : fma2_f16(whole, s2, o[j] ^ 0x80008000u);
                }
                else
                {
                    const float2 f = unpack2(whole, BF16);
                    const float x = f.x * scale, y = f.y * scale;
                    o[j]          = pack2(x, y, BF16);
                    if (LOW)
                    {
                        const float2 h = unpack2(o[j], BF16);
                        low[j]         = keep & pack2(x - h.x, y - h.y, BF16);
                    }
                }
            }
            if (TAIL)
            {
                // behind the end lies whatever the row holds there, under a scale that may not be finite
#pragma unroll
                for (int j = 0; j < 4; j++)
                {
                    const int at = h * 32 + i * 8 + j * 2;
                    o[j]         = at + 1 < left ? o[j] : at < left ? o[j] & 0xffffu : 0u;
                    if (LOW)
                        low[j] = at + 1 < left ? low[j] : at < left ? low[j] & 0xffffu : 0u;
                }
            }
            if (LOW)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)(kChunk + (((h * 4 + i) ^ (row & 7)) << 4))), "r"(low[0]), "r"(low[1]),
                             "r"(low[2]), "r"(low[3])
                             : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)(((h * 4 + i) ^ (row & 7)) << 4)), "r"(o[0]), "r"(o[1]), "r"(o[2]),
                         "r"(o[3])
                         : "memory");
        }
    }
}

template <int EPI, bool A_MN, bool B_MN, bool PAIR, bool W4 = false>
__global__ void __launch_bounds__((Shape<PAIR, W4, W4 && EPI == EPI_GATED>::kThreads), 1) ffn_pair_kernel(const __grid_constant__ Params p)
{
    static_assert(W4 || EPI == EPI_PLAIN || B_MN, "both projections' matrices have K across their rows");
    constexpr bool LOW    = W4 && EPI == EPI_GATED;
    using S               = Shape<PAIR, W4, LOW>;
    constexpr int kSub    = S::kSub, kStage = S::kStage, kHalf = S::kCols / 2, kStages = S::kStages, kThreads = S::kThreads;
    extern __shared__ uint8_t smem_raw[];
    // identical layout in both CTAs of a pair: remote signals address a barrier by its offset
    __shared__ __align__(8) uint64_t bar_full[kStages];     // used in the first CTA: bytes of both CTAs (4-bit weights: values in place)
    __shared__ __align__(8) uint64_t bar_empty[kStages];    // per CTA: stage consumed by the MMAs
    __shared__ __align__(8) uint64_t bar_tmem_full[2];         // per CTA: accumulator buffer complete
    __shared__ __align__(8) uint64_t bar_tmem_empty[2];        // first CTA: buffer drained by both CTAs' epilogues
    __shared__ __align__(8) uint64_t bar_ready;                // first CTA: tensor memory taken in both
    __shared__ __align__(8) uint64_t bar_drain;                // first CTA: MMAs in flight when the issuer gives up
    __shared__ __align__(8) uint64_t bar_raw[W4 ? kStages : 1];         // per CTA: 4-bit weights and rows of A of the stage
    __shared__ int gave_up;                                    // a role of this CTA or of the pair's other one
    __shared__ long long stages_issued;                        // per CTA: stages whose copies were asked for
    __shared__ uint32_t tmem_base_holder;
    __shared__ float stages[kEpiWarps][32 * 17];    // of the epilogue's warps

    const int warp           = threadIdx.x >> 5;
    const int lane           = threadIdx.x & 31;
    const uint32_t rank      = PAIR ? ptx::cluster_ctarank() : 0;
    const int cluster_id     = PAIR ? blockIdx.x / 2 : blockIdx.x / (unsigned)p.splits;
    const int num_clusters   = PAIR ? gridDim.x / 2 : gridDim.x / (unsigned)p.splits;
    const int share          = !PAIR && p.splits > 1 ? (int)ptx::cluster_ctarank() : 0;    // of K
    const int chunk0         = share * (p.chunks * p.phases) / p.splits;
    const int total          = (share + 1) * (p.chunks * p.phases) / p.splits - chunk0;    // chunks of this CTA (pair)
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    float* const red         = reinterpret_cast<float*>(smem_raw + (smem_base - ptx::smem_u32(smem_raw)));    // a share's sums of a tile

    float scale = 1.f, peak = 0.f;
    if (EPI == EPI_GRAD && p.seen)
    {
        // The second launch: nothing is left to do where the first one's values are held well (394 x 1024 x 2048: 2.5 us of 34.8).
        constexpr int kWarps = kThreads / 32;
        float* const most    = &stages[0][0];
        ptx::dep_launch_wait();
        for (int i = threadIdx.x; i < (int)gridDim.x * kWarps; i += kThreads)
            peak = fmaxf(peak, __ldcg(p.seen + i));
        peak = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(peak)));    // (none is negative)
        if (lane == 0)
            most[warp] = peak;
        __syncthreads();
        for (int i = 0; i < kWarps; i++)
            peak = fmaxf(peak, most[i]);
        __syncthreads();
        scale = range_scale(peak);
        if (blockIdx.x == 0 && threadIdx.x == 0)
            *p.undo = 1.f / scale;
        if (scale == 1.f)
            return;
    }
    if (threadIdx.x == 0)
    {
        for (int s = 0; s < kStages; s++)
        {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), W4 ? 4 * S::kCtas : 1);    // a group's warps of each CTA, or copies
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
            if (W4)
                ptx::mbar_init(ptx::smem_u32(&bar_raw[s]), 1);
        }
        for (int a = 0; a < 2; a++)
        {
            ptx::mbar_init(ptx::smem_u32(&bar_tmem_full[a]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_tmem_empty[a]), S::kCtas * kEpiWarps);
        }
        ptx::mbar_init(ptx::smem_u32(&bar_drain), 1);
        ptx::mbar_init(ptx::smem_u32(&bar_ready), S::kCtas);
        gave_up       = 0;
        stages_issued = 0;
        ptx::fence_barrier_init();
        ptx::prefetch_tmap(&p.tmA);
        ptx::prefetch_tmap(&p.tmB0);
        ptx::prefetch_tmap(&p.tmB1);
        // the first weights on their way to L2, where a write by the kernel before would still find them
        if (W4 && cluster_id < p.num_tiles)
        {
            const Tile t = decode<EPI, PAIR>(p, cluster_id);
            for (int c = chunk0; c < chunk0 + min(total, kStages); c++)
            {
                ptx::prefetch_2d(EPI != EPI_PLAIN && rank ? &p.tmB1 : &p.tmB0, c * 32, EPI == EPI_PLAIN ? t.n0 + (int)rank * 128 : t.n0);
                if (EPI != EPI_PLAIN && !PAIR)
                    ptx::prefetch_2d(&p.tmB1, c * 32, t.n0);
            }
        }
        else if (EPI != EPI_PLAIN && cluster_id < p.num_tiles)
        {
            const Tile t = decode<EPI, PAIR>(p, cluster_id);
            for (int c = chunk0; c < min(p.chunks, chunk0 + min(total, kStages * kSub)); c++)
                for (int m = PAIR ? (int)rank : 0; m < (PAIR ? (int)rank + 1 : 2); m++)
                {
                    const CUtensorMap* const b = m ? &p.tmB1 : &p.tmB0;
                    for (int n = 0; n < kHalf; n += 64)
                        ptx::prefetch_3d(b, t.n0 + n, c * 64, t.idx);
                }
        }
    }
    // no signal may reach the other CTA before its barriers exist
    if (PAIR)
        ptx::cluster_sync();
    else
        __syncthreads();
    // Everything a kernel before this one may have written is read behind this wait, and nothing is written before it.  Tensor memory
    // is taken behind it too, and the next kernel let in only then: neither kernel can keep the other from columns it waits for.
    // A product beside the one before it reads what came before both: that one let this in behind its own wait, so it is there.
    if (!p.beside)
        ptx::dep_launch_wait();
    if (EPI == EPI_PLAIN && !W4 && p.undo)
        scale = __ldcg(p.undo);
    // a role that gives up says so in every CTA of the tile
    auto give_up = [&]() {
        atomicOr(p.status, TB200_DEV_TIMEOUT);
        gave_up = 1;
        if (PAIR)
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(ptx::map_to_cta(ptx::smem_u32(&gave_up), rank ^ 1u)), "r"(1) : "memory");
    };
    uint32_t tmem_base = 0;
    if (warp != 0)
    {
        if (warp == 1)
        {
            if (PAIR)
            {
                ptx::tmem_alloc_pair(ptx::smem_u32(&tmem_base_holder), S::kTmemCols);
                ptx::tmem_relinquish_pair();
            }
            else
            {
                ptx::tmem_alloc(ptx::smem_u32(&tmem_base_holder), S::kTmemCols);
                ptx::tmem_relinquish();
            }
            if (lane == 0)
            {
                if (PAIR)
                    ptx::mbar_arrive_cluster(ptx::map_to_cta(ptx::smem_u32(&bar_ready), 0));
                ptx::dep_launch_trigger();
            }
        }
        // all but the TMA warp, whose copies are on their way by now
        ptx::tc_fence_before_sync();
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 32) : "memory");
        ptx::tc_fence_after_sync();
        tmem_base = tmem_base_holder;
    }

    if (warp == 0)
    {
        // ------------------------------------------------------------------ TMA producer (both CTAs)
        if (lane == 0)
        {
            int stage      = 0;
            uint32_t phase = 0;
            bool ok        = true;
            long long issued = 0;
            for (int tile = cluster_id; tile < p.num_tiles && ok; tile += num_clusters)
            {
                const Tile t          = decode<EPI, PAIR>(p, tile);
                const int m0          = t.m0 + (int)rank * 128;
                const int n0          = EPI == EPI_PLAIN ? t.n0 + (int)rank * 128 : t.n0;    // of the CTA's 128 columns, or of each matrix's
                const int batch       = t.idx < p.NB ? t.idx : t.idx - p.NB;
                const int b_batch     = (A_MN && B_MN) ? t.idx : batch;    // gradients of weights: dG's batches, then dU's
                for (int left = total, c = chunk0; left > 0; left -= kSub)
                {
                    if (!ptx::mbar_wait_bounded(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, p.wait_limit))
                    {
                        ok = false;
                        break;
                    }
                    const int nch             = min(kSub, left);
                    const uint32_t full_local = ptx::smem_u32(&bar_full[stage]);
                    // the first CTA arms the barrier with the bytes of both CTAs; each CTA's copies report there.  4-bit weights: copies report to
                    // their own CTA, whose groups wait for them and then report.
                    if (W4)
                        ptx::mbar_arrive_expect_tx(ptx::smem_u32(&bar_raw[stage]), kChunk + kRawBytes);
                    else if (rank == 0)
                        ptx::mbar_arrive_expect_tx(full_local, (uint32_t)(nch * 2 * S::kCtas * kChunk));
                    const uint32_t full_first = W4 ? ptx::smem_u32(&bar_raw[stage]) : PAIR ? ptx::map_to_cta(full_local, 0) : full_local;
                    const uint32_t sA         = smem_base + (uint32_t)(stage * kStage);
                    const uint32_t sB         = sA + (uint32_t)(kSub * kChunk);
                    for (int j = 0; j < nch; j++, c++)
                    {
                        const int ph      = c >= p.chunks ? 1 : 0;
                        const int k       = (c - ph * p.chunks) * 64;
                        const uint32_t dA = sA + (uint32_t)(j * kChunk), dB = sB + (uint32_t)(j * kChunk);
                        auto load = [&](uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2) {
                            if (PAIR && !W4)
                                ptx::tma_load_3d_pair(dst, m, full_first, c0, c1, c2);
                            else
                                ptx::tma_load_3d(dst, m, full_first, c0, c1, c2);
                        };
                        if (A_MN)
                        {
                            load(dA, &p.tmA, m0, k, batch);
                            load(dA + 8192, &p.tmA, m0 + 64, k, batch);
                        }
                        else
                            load(dA, &p.tmA, k, m0, batch + ph * p.NB);
                        if (W4)
                        {
                            // where their values will be
                            ptx::tma_load_2d(dB, EPI != EPI_PLAIN && rank ? &p.tmB1 : &p.tmB0, full_first, c * 32, n0);
                            if (EPI != EPI_PLAIN && !PAIR)
                                ptx::tma_load_2d(dB + kRawBytes / 2, &p.tmB1, full_first, c * 32, n0);
                            continue;
                        }
                        if (EPI != EPI_PLAIN && !PAIR)
                        {
                            // one CTA holds 64 columns of each matrix
                            load(dB, &p.tmB0, n0, k, b_batch);
                            load(dB + 8192, &p.tmB1, n0, k, b_batch);
                            continue;
                        }
                        const CUtensorMap* mb = (EPI == EPI_PLAIN ? ph != 0 : rank != 0) ? &p.tmB1 : &p.tmB0;
                        if (B_MN)
                        {
                            load(dB, mb, n0, k, b_batch);
                            load(dB + 8192, mb, n0 + 64, k, b_batch);
                        }
                        else
                            load(dB, mb, k, n0, b_batch);
                    }
                    issued++;
                    if (++stage == kStages)
                    {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            stages_issued = issued;
            if (!ok)
                give_up();
        }
    }
    else if (warp == 1)
    {
        // ------------------------------------------------------------------ MMA issuer (first CTA of the pair)
        if (lane == 0 && rank == 0)
        {
            int stage      = 0;
            uint32_t phase = 0;
            int acc        = 0;
            uint32_t acc_phase = 0;
            bool ok            = true;
            // arrives in every CTA of the tile once the MMAs so far are done
            auto commit = [&](uint32_t bar) {
                if (PAIR)
                    ptx::mma_commit_pair(bar, 3);
                else
                    ptx::mma_commit(bar);
            };
            // the MMAs write both CTAs' tensor memory
            if (PAIR)
                ok = ptx::mbar_wait_bounded(ptx::smem_u32(&bar_ready), 0, p.wait_limit);
            bool ready = false;    // the stage is known to be complete
            for (int tile = cluster_id; tile < p.num_tiles && ok; tile += num_clusters)
            {
                if (!ptx::mbar_wait_bounded(ptx::smem_u32(&bar_tmem_empty[acc]), acc_phase ^ 1u, p.wait_limit))
                {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + (uint32_t)(acc * S::kCols);
                uint32_t accum        = 0;    // the first MMA of a tile overwrites the accumulator
                for (int left = total; left > 0; left -= kSub)
                {
                    if (!ready && !ptx::mbar_wait_bounded(ptx::smem_u32(&bar_full[stage]), phase, p.wait_limit))
                    {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const int nch     = min(kSub, left);
                    const uint32_t sA = smem_base + (uint32_t)(stage * kStage);
                    const uint32_t sB = sA + (uint32_t)(kSub * kChunk);
                    for (int j = 0; j < nch; j++)
                    {
                        uint64_t ad = ptx::smem_desc(p.a_desc_hi, sA + (uint32_t)(j * kChunk));
                        uint64_t bd = ptx::smem_desc(p.b_desc_hi, sB + (uint32_t)(j * kChunk));
#pragma unroll
                        for (int m = 0; m < 4; m++)
                        {
                            if (PAIR)
                                ptx::mma_f16_ss_pair(d_tmem, ad, bd, p.idesc, accum);
                            else
                                ptx::mma_f16_ss(d_tmem, ad, bd, p.idesc, accum);
                            accum = 1;
                            if (LOW)
                            {
                                if (PAIR)
                                    ptx::mma_f16_ss_pair(d_tmem, ad, bd + kChunk / 16, p.idesc, 1);
                                else
                                    ptx::mma_f16_ss(d_tmem, ad, bd + kChunk / 16, p.idesc, 1);
                            }
                            // sixteen elements of K: 32 bytes inside the swizzled row, or sixteen rows of 128 bytes
                            ad += A_MN ? 128 : 2;
                            bd += B_MN ? 128 : 2;
                            // the next stage, looked at while MMAs are queued: a look takes 110 cycles, in which the tensor cores ran dry
                            if (W4 && m == 1)
                                ready = ptx::mbar_test(ptx::smem_u32(&bar_full[stage + 1 < kStages ? stage + 1 : 0]), stage + 1 < kStages ? phase : phase ^ 1u);
                        }
                    }
                    // frees the stage in both CTAs once the MMAs above have read it
                    commit(ptx::smem_u32(&bar_empty[stage]));
                    if (++stage == kStages)
                    {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok)
                    break;
                commit(ptx::smem_u32(&bar_tmem_full[acc]));
                acc ^= 1;
                if (acc == 0)
                    acc_phase ^= 1u;
            }
            if (!ok)
                give_up();
        }
    }
    else if (W4 && warp >= 2 + kEpiWarps)
    {
        // ------------------------------------------------------------------ 4-bit weights to 16 bits (both CTAs)
        // Groups of four warps take chunks in turn, a thread a row of 64 elements.  The bytes lie where the values go, so a group has read
        // all of them before it writes.
        const int group = (warp - 2 - kEpiWarps) >> 2, row = ((warp - 2 - kEpiWarps) & 3) * 32 + lane;
        const int mat   = EPI == EPI_PLAIN ? 0 : PAIR ? (int)rank : row >> 6;
        const int shift = EPI == EPI_PLAIN ? (int)rank * 128 + row : PAIR ? row : row & 63;    // of the thread's column in the tile
        const bool same = p.scale_dt[mat] == (p.bf16 ? TB200_BF16 : TB200_FP16);
        bool ok = true, bad = false;
        int tile = cluster_id, c = chunk0 + group, stage = group;
        uint32_t phase = 0;
        int zero[2] = {}, zero_next[2] = {};
        uint32_t scale[2] = {}, scale_next[2] = {};    // bits
        // the next chunk's first group, and how many 32-element pieces of it lie before the chunk
        int first_group = 0;
        uint32_t into   = 0;
        // The next chunk's scales and zero points are on their way while this one's values are made.
        const bool wide          = p.scale_dt[mat] == TB200_FP32;
        const bool with_zero     = p.zero[mat] != nullptr;
        const uint8_t* scale_at  = nullptr;    // of the thread's column, first group
        const int8_t* zero_at    = nullptr;
        const int64_t scale_step = (int64_t)p.cols * (wide ? 4 : 2);
        const int last_group     = p.groups - 1;
        auto to_column = [&]() {
            const int col = min(decode<EPI, PAIR>(p, tile).n0 + shift, p.cols - 1);
            scale_at      = reinterpret_cast<const uint8_t*>(p.scale[mat]) + (int64_t)col * (wide ? 4 : 2);
            zero_at       = p.zero[mat] + col;
            first_group   = (int)((uint32_t)(2 * c) / p.group32);
            into          = (uint32_t)(2 * c) - (uint32_t)first_group * p.group32;
        };
        auto fetch = [&]() {
            const int g0 = min(first_group, last_group), g1 = min(first_group + (into + 1 >= p.group32 ? 1 : 0), last_group);
            load_bits(scale_next[0], scale_at + g0 * scale_step, wide);
            load_bits(scale_next[1], scale_at + g1 * scale_step, wide);
            load_zero(zero_next[0], zero_at + (int64_t)g0 * p.cols, with_zero);
            load_zero(zero_next[1], zero_at + (int64_t)g1 * p.cols, with_zero);
        };
        auto to_tile = [&]() {
            bool moved = false;
            for (; c >= chunk0 + total && tile < p.num_tiles; moved = true)
            {
                c -= total;
                tile += num_clusters;
            }
            if (moved && tile < p.num_tiles)
                to_column();
        };
        if (tile < p.num_tiles)
            to_column();
        to_tile();
        if (tile < p.num_tiles)
            fetch();
        while (tile < p.num_tiles && ok)
        {
            const int left = p.K - c * 64;
#pragma unroll
            for (int h = 0; h < 2; h++)
            {
                scale[h] = scale_next[h];
                zero[h]  = zero_next[h];
                bad |= zero[h] < -8 || zero[h] > 7;
            }
            c += S::kGroups;
            for (into += 2 * S::kGroups; into >= p.group32; into -= p.group32)
                first_group++;
            to_tile();
            if (tile < p.num_tiles)
                fetch();
            const uint32_t sB = smem_base + (uint32_t)(stage * kStage + kChunk);
            ok                = ptx::mbar_wait_bounded(ptx::smem_u32(&bar_raw[stage]), phase, p.wait_limit);
            uint4 raw[2];
#pragma unroll
            for (int h = 0; h < 2; h++)
                raw[h] = lds128(sB + (uint32_t)(row * 32 + ((h ^ ((row >> 2) & 1)) << 4)));
            ok = ptx::named_barrier_and(2 + group, 128, ok);
            if (!ok)
                break;
            const uint32_t dst = sB + (uint32_t)(row * 128);
            auto expand        = [&](auto bf16) {
                constexpr bool kBf16 = decltype(bf16)::value;
                if (left < 64)
                    expand_row<kBf16, false, true, LOW>(raw, scale, p.scale_dt[mat], zero, left, dst, row);
                else if (same && (!LOW || max(scale[0] & 0x7fffu, scale[1] & 0x7fffu) < (kBf16 ? 0x7d88u : 0x6c44u)))    // the largest number over 15
                    expand_row<kBf16, true, false, LOW>(raw, scale, p.scale_dt[mat], zero, left, dst, row);
                else
                    expand_row<kBf16, false, false, LOW>(raw, scale, p.scale_dt[mat], zero, left, dst, row);
            };
            if (p.bf16)
                expand(std::true_type());
            else
                expand(std::false_type());
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0)
            {
                if (PAIR)
                    ptx::mbar_arrive_cluster_release(ptx::map_to_cta(ptx::smem_u32(&bar_full[stage]), 0));
                else
                    ptx::mbar_arrive(ptx::smem_u32(&bar_full[stage]));
            }
            stage += S::kGroups;
            if (stage >= kStages)
            {
                stage -= kStages;
                phase ^= 1u;
            }
        }
        if (!ok && lane == 0)
            give_up();
        if (bad)
            atomicOr(p.status, TB200_DEV_UNPREDICTABLE);
    }
    else
    {
        // ------------------------------------------------------------------ epilogue warps (both CTAs)
        const int quarter = warp & 3;           // TMEM lane quarter this warp may read
        const int slot    = (warp - 2) >> 2;    // the two warps of a quarter take 16-column runs in turn
        const int row     = quarter * 32 + lane;
        float* const stage = stages[warp - 2];
        const uint32_t empty_first[2] = { PAIR ? ptx::map_to_cta(ptx::smem_u32(&bar_tmem_empty[0]), 0) : ptx::smem_u32(&bar_tmem_empty[0]),
                                          PAIR ? ptx::map_to_cta(ptx::smem_u32(&bar_tmem_empty[1]), 0) : ptx::smem_u32(&bar_tmem_empty[1]) };
        int acc            = 0;
        uint32_t acc_phase = 0;
        bool ok            = true;
        for (int tile = cluster_id; tile < p.num_tiles; tile += num_clusters)
        {
            const Tile t = decode<EPI, PAIR>(p, tile);
            ok           = ptx::mbar_wait_bounded(ptx::smem_u32(&bar_tmem_full[acc]), acc_phase, p.wait_limit);
            // the whole warp must agree before the warp-collective TMEM loads
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                break;
            ptx::tc_fence_after_sync();
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * S::kCols);
            if (!PAIR && p.splits > 1)
            {
                // this share's sums to shared memory, over the ring (its copies have landed and been multiplied)
                for (int c = slot; c < S::kCols / 16; c += 2)
                {
                    uint32_t v[16];
                    ptx::tmem_ld_32x32b_x16(taddr + (uint32_t)(c * 16), v);
                    ptx::tmem_ld_wait_x16(v);
                    uint4* const to = reinterpret_cast<uint4*>(red + row * S::kRedLd + c * 16);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        to[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            }
            else if (EPI == EPI_PLAIN)
            {
                for (int c = slot; c < S::kCols / 16; c += 2)
                {
                    if (t.n0 + c * 16 >= p.cols)
                        break;
                    uint32_t g[16];
                    ptx::tmem_ld_32x32b_x16(taddr + (uint32_t)(c * 16), g);
                    ptx::tmem_ld_wait_x16(g);
                    finish_run<EPI>(p, t, (int)rank * 128 + row, c * 16, g, g, stage, scale, peak);
                }
            }
            else
            {
                for (int c = slot; c < kHalf / 16; c += 2)
                {
                    if (t.n0 + c * 16 >= p.cols)
                        break;
                    uint32_t g[16], u[16];
                    ptx::tmem_ld_32x32b_x16(taddr + (uint32_t)(c * 16), g);
                    ptx::tmem_ld_32x32b_x16(taddr + (uint32_t)(kHalf + c * 16), u);
                    ptx::tmem_ld_wait_x16(g);
                    ptx::tmem_ld_wait_x16(u);
                    finish_run<EPI>(p, t, (int)rank * 128 + row, c * 16, g, u, stage, scale, peak);
                }
            }
            // this warp has read its part of the buffer: one arrival per warp on the first CTA's barrier
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0)
            {
                if (PAIR)
                    ptx::mbar_arrive_cluster(empty_first[acc]);
                else
                    ptx::mbar_arrive(empty_first[acc]);
            }
            acc ^= 1;
            if (acc == 0)
                acc_phase ^= 1u;
        }
        if (!ok && lane == 0)
            give_up();
    }

    if (!PAIR && p.splits > 1)
    {
        // ------------------------------------------------------------------ the shares' sums meet, in order (one tile to a cluster)
        // A share whose wait gave up holds sums that do not count; every share reaches both barriers.
        ptx::cluster_sync();
        const Tile t         = decode<EPI, PAIR>(p, cluster_id);
        constexpr int kQuads = (EPI == EPI_PLAIN ? S::kCols : kHalf) / 4;    // of a row
        const uint32_t local = ptx::smem_u32(red);
        // four neighbouring columns a thread, the shares' sums all on their way before the first is added (sixteen columns, a share at a
        // time, took 2 to 8 us)
        for (int e = share * kThreads + (int)threadIdx.x; e < 128 * kQuads; e += p.splits * kThreads)
        {
            const int r = e / kQuads, col = e % kQuads * 4;
            if (t.m0 + r >= p.rows || t.n0 + col >= p.cols)
                continue;
            auto sum = [&](int c, float (&v)[4]) {
                float4 x[8];
                const uint32_t at = local + (uint32_t)((r * S::kRedLd + c) * 4);
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (k < p.splits)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(x[k].x), "=f"(x[k].y), "=f"(x[k].z), "=f"(x[k].w)
                                     : "r"(ptx::map_to_cta(at, (uint32_t)k))
                                     : "memory");
                    else
                        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                v[0] = v[1] = v[2] = v[3] = 0.f;
#pragma unroll
                for (int k = 0; k < 8; k++)
                {
                    v[0] += x[k].x;
                    v[1] += x[k].y;
                    v[2] += x[k].z;
                    v[3] += x[k].w;
                }
            };
            float g[4], u[4] = {};
            sum(col, g);
            if (EPI != EPI_PLAIN)
                sum(kHalf + col, u);
            finish_quad<EPI>(p, t, r, col, g, u, scale, peak);
        }
        ptx::cluster_sync();    // nobody leaves while another share may still read its sums
    }

    // ---------------------------------------------------------------------- teardown
    // Neither CTA may leave (or free its TMEM) while the other can still signal it or read its shared memory.
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (EPI == EPI_GRAD && p.peaks)
    {
        peak = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(peak)));
        if (lane == 0)
            p.peaks[blockIdx.x * (kThreads / 32) + warp] = peak;
    }
    if (PAIR)
        ptx::cluster_sync();
    if (gave_up)
    {
        // A role gave up (both CTAs of a pair know by now): MMAs and copies that are on their way are waited for, whoever has issued them.
        if (warp == 1 && lane == 0 && rank == 0)
        {
            if (PAIR)
                ptx::mma_commit_pair(ptx::smem_u32(&bar_drain), 1);
            else
                ptx::mma_commit(ptx::smem_u32(&bar_drain));
            ptx::mbar_wait_bounded(ptx::smem_u32(&bar_drain), 0, ptx::kDrainCycles);
        }
        if (threadIdx.x == 0 && (W4 || rank == 0))
        {
            const long long mine = stages_issued;
            long long all        = mine;
            if (PAIR && !W4)
            {
                // One CTA may have asked for stages that the other has not.  Their barriers still count its bytes: armed for them where this
                // CTA has not armed them, less the bytes that will not come where it has.
                long long other;
                asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(other) : "r"(ptx::map_to_cta(ptx::smem_u32(&stages_issued), 1)) : "memory");
                all             = max(mine, other);
                const int per   = (total + kSub - 1) / kSub;    // stages of a tile
                for (long long i = min(mine, other); i < all; i++)
                {
                    const uint32_t full  = ptx::smem_u32(&bar_full[i % kStages]);
                    const uint32_t bytes = (uint32_t)(min(kSub, total - (int)(i % per) * kSub) * 2 * kChunk);    // of one CTA
                    if (other > mine)
                        ptx::mbar_arrive_expect_tx(full, bytes);
                    else
                        ptx::mbar_complete_tx(full, bytes);
                }
            }
            for (long long i = max(0LL, all - kStages); i < all; i++)
                ptx::mbar_wait_bounded(ptx::smem_u32(W4 ? &bar_raw[i % kStages] : &bar_full[i % kStages]), (uint32_t)(i / kStages) & 1u, ptx::kDrainCycles);
        }
        __syncthreads();
        if (PAIR)
            ptx::cluster_sync();
    }
    if (warp == 1)
    {
        ptx::tc_fence_after_sync();
        if (PAIR)
            ptx::tmem_dealloc_pair(tmem_base, S::kTmemCols);
        else
            ptx::tmem_dealloc(tmem_base, S::kTmemCols);
    }
    // whoever waits for this kernel waits for the one before it too
    if (p.beside)
        ptx::dep_launch_wait();
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A [batches][outer][inner] operand of 16-bit elements with rows `pitch` elements apart: K along its rows (boxes of 64 x 128), or
// across them (64 x 64, two for each half tile).  What lies outside reads as zero.
tb200_status encode(tb200_ctx* ctx, CUtensorMap* m, const Matrix& x, bool bf16, bool k_inner, uint32_t lines = 128)
{
    const EncodeTiled enc = reinterpret_cast<EncodeTiled>(tensor_map_encode_fn());
    if (!enc)
        return fail(ctx, TB200_INTERNAL, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3]    = { (cuuint64_t)x.inner, (cuuint64_t)x.outer, (cuuint64_t)x.batches };
    const cuuint64_t strides[2] = { (cuuint64_t)x.pitch * 2, (cuuint64_t)x.pitch * (cuuint64_t)x.outer * 2 };
    const cuuint32_t box[3]     = { 64, k_inner ? lines : 64u, 1 };
    const cuuint32_t estr[3]    = { 1, 1, 1 };
    const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(x.data), dims, strides, box,
                           estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(ctx, TB200_INTERNAL, "tensor map of a feed-forward product rejected (CUresult %d)", (int)r);
    return TB200_OK;
}

// Rows of 4-bit weights, 64 elements of `lines` of them at a time; eight threads' sixteens of bytes, one from each row, meet all banks.
tb200_status encode_raw(tb200_ctx* ctx, CUtensorMap* m, const W4Mat& w, int cols, uint32_t lines)
{
    const EncodeTiled enc = reinterpret_cast<EncodeTiled>(tensor_map_encode_fn());
    if (!enc)
        return fail(ctx, TB200_INTERNAL, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2]    = { (cuuint64_t)w.pitch, (cuuint64_t)cols };
    const cuuint64_t strides[1] = { (cuuint64_t)w.pitch };
    const cuuint32_t box[2]     = { 32, lines };
    const cuuint32_t estr[2]    = { 1, 1 };
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(w.data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(ctx, TB200_INTERNAL, "tensor map of 4-bit weights rejected (CUresult %d)", (int)r);
    return TB200_OK;
}

int run_alignment(const void* p, int64_t ld, size_t es)
{
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * (int64_t)es);
    return (bits & 31) == 0 ? 2 : (bits & 15) == 0 ? 1 : 0;
}

}    // namespace

namespace
{

typedef void (*Kern)(const Params);

template <bool PAIR>
Kern pick(const PairProduct& q, int* bit)
{
    if (q.w4)
    {
        *bit = q.kind == PAIR_GATED ? 5 : 4;
        return q.kind == PAIR_GATED ? ffn_pair_kernel<EPI_GATED, false, false, PAIR, true> : ffn_pair_kernel<EPI_PLAIN, false, false, PAIR, true>;
    }
    if (q.kind != PAIR_PLAIN && !q.a_mn && q.b_mn)
    {
        *bit = q.kind == PAIR_GATED ? 0 : 1;
        return q.kind == PAIR_GATED ? ffn_pair_kernel<EPI_GATED, false, true, PAIR> : ffn_pair_kernel<EPI_GRAD, false, true, PAIR>;
    }
    if (q.kind == PAIR_PLAIN && q.a_mn == q.b_mn)
    {
        *bit = q.a_mn ? 2 : 3;
        return q.a_mn ? ffn_pair_kernel<EPI_PLAIN, true, true, PAIR> : ffn_pair_kernel<EPI_PLAIN, false, false, PAIR>;
    }
    return nullptr;
}

template <bool PAIR>
tb200_status launch(tb200_ctx* ctx, const PairProduct& q, int splits)
{
    using S = Shape<PAIR>;    // (4-bit weights: the same but for the ring's division into stages)
    Params k;
    memset(&k, 0, sizeof(k));
    const bool bf16       = q.dt == TB200_BF16;
    const bool gated      = q.kind != PAIR_PLAIN;
    const uint32_t b_line = !PAIR && gated ? 64u : 128u;
    tb200_status st       = encode(ctx, &k.tmA, q.a, bf16, !q.a_mn);
    for (int i = 0; q.w4 && i < (gated ? 2 : 1) && st == TB200_OK; i++)
    {
        st             = encode_raw(ctx, i ? &k.tmB1 : &k.tmB0, q.w4[i], q.cols, b_line);
        k.scale[i]     = q.w4[i].scale;
        k.scale_dt[i]  = q.w4[i].scale_dt;
        k.zero[i]      = q.w4[i].zero;
    }
    if (q.w4)
    {
        if (!gated)
            k.tmB1 = k.tmB0;
        k.K       = (int)q.K;
        k.groups  = (int)((q.K + q.group - 1) / q.group);
        k.group32 = q.group >= q.K ? 1u << 30 : (uint32_t)q.group / 32;    // (a group that holds a whole row has any length)
    }
    if (st == TB200_OK && !q.w4)
        st = encode(ctx, &k.tmB0, q.b[0], bf16, !q.b_mn, b_line);
    if (st == TB200_OK && !q.w4)
        st = encode(ctx, &k.tmB1, q.b[1].data ? q.b[1] : q.b[0], bf16, !q.b_mn, b_line);
    if (st != TB200_OK)
        return st;
    const int step_n    = gated ? S::kCols / 2 : S::kCols;
    k.rows              = q.rows;
    k.cols              = q.cols;
    k.tiles_m           = (q.rows + S::kRows - 1) / S::kRows;
    k.tiles_n           = (q.cols + step_n - 1) / step_n;
    k.NB                = q.NB;
    k.beside            = q.beside ? 1 : 0;
    k.num_tiles         = k.tiles_m * k.tiles_n * q.NB * (q.results == 2 && !gated ? 2 : 1);    // (2^30 at most: tiles_reach)
    // A's rows of a group, about 32 MB, stay in L2
    const int64_t a_tile = (int64_t)S::kRows * q.K * q.phases * 2;
    k.group_m  = (int)std::max<int64_t>(1, std::min<int64_t>(k.tiles_m, (32LL << 20) / std::max<int64_t>(1, a_tile)));
    k.chunks   = (int)((q.K + 63) / 64);
    k.phases   = q.phases;
    k.splits   = splits;
    k.act      = q.act;
    k.bf16     = bf16 ? 1 : 0;
    k.out_dt   = q.out_dt[0];
    k.out1_dt  = q.out_dt[1];
    k.out0     = q.out[0];
    k.out1     = q.out[1];
    k.ld       = q.ld;
    k.vec      = q.out[0] ? run_alignment(q.out[0], q.ld, dtype_size(q.out_dt[0])) : 2;
    if (q.out[1])
        k.vec = std::min(k.vec, run_alignment(q.out[1], q.ld, dtype_size(q.out_dt[1])));
    k.even     = q.ld % 2 == 0 && q.cols % 2 == 0;
    k.dout     = q.dout;
    k.dout_vec = q.dout && run_alignment(q.dout, q.cols, 2) > 0;
    // K along the rows: 8-row groups of 128-byte swizzled rows 1024 bytes apart.  Across them: 64 columns of 64 K rows, the next 64
    // 8192 bytes behind.
    k.a_desc_hi  = q.a_mn ? ptx::make_smem_desc_hi(8192, 1024, 2) : ptx::make_smem_desc_hi(16, 1024, 2);
    k.b_desc_hi  = q.b_mn ? ptx::make_smem_desc_hi(8192, 1024, 2) : ptx::make_smem_desc_hi(16, 1024, 2);
    const uint32_t fmt = bf16 ? 1u : 0u;
    k.idesc      = ptx::make_idesc(1u, fmt, fmt, q.a_mn ? 1u : 0u, q.b_mn ? 1u : 0u, (uint32_t)S::kRows, (uint32_t)S::kCols);
    k.peaks      = q.peaks;
    k.seen       = q.seen;
    k.undo       = q.undo;
    k.wait_limit = ctx->wait_limit_cycles;
    k.status     = ctx->d_status;
    int bit      = 0;
    const Kern kern = pick<PAIR>(q, &bit);
    if (!kern)
        return fail(ctx, TB200_INTERNAL, "no kernel for this feed-forward product");
    st = raise_smem_limit(ctx, 128 + bit + (PAIR ? 0 : 48), reinterpret_cast<const void*>(kern), S::kSmem);
    if (st != TB200_OK)
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim           = dim3(!q.w4 ? S::kThreads : gated ? Shape<PAIR, true, true>::kThreads : Shape<PAIR, true>::kThreads);
    cfg.dynamicSmemBytes   = (size_t)S::kSmem;
    cfg.stream             = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = ctx->launch_overlap ? 1 : 0;
    attr[1].id               = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = PAIR ? 2 : (unsigned)splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs    = attr;
    cfg.numAttrs = PAIR || splits > 1 ? 2 : 1;
    // a tile that is shared is its cluster's only one
    cfg.gridDim  = dim3((unsigned)(PAIR         ? 2 * std::max(1, std::min(k.num_tiles, ctx->num_sms / 2))
                                   : splits > 1 ? k.num_tiles * splits
                                                : std::min(k.num_tiles, ctx->num_sms)));
    timer_begin(ctx);
    const cudaError_t le = cudaLaunchKernelEx(&cfg, kern, k);
    timer_end(ctx);
    if (le != cudaSuccess)
        return fail(ctx, TB200_INTERNAL, "launch of a feed-forward product failed: %s", cudaGetErrorString(le));
    return post_launch(ctx, q.name);
}

// How many clusters of `size` CTAs by themselves run at once
tb200_status clusters_at_once(tb200_ctx* ctx, int which, int size, int* n)
{
    if (ctx->ffn_clusters[which] == 0)
    {
        const Kern kern       = ffn_pair_kernel<EPI_PLAIN, false, false, false>;
        const tb200_status st = raise_smem_limit(ctx, 128 + 48 + 3, reinterpret_cast<const void*>(kern), Shape<false>::kSmem);
        if (st != TB200_OK)
            return st;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim            = dim3((unsigned)ctx->num_sms * size);
        cfg.blockDim           = dim3(Shape<false>::kThreads);
        cfg.dynamicSmemBytes   = (size_t)Shape<false>::kSmem;
        cudaLaunchAttribute attr[1];
        attr[0].id               = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs    = attr;
        cfg.numAttrs = 1;
        TB200_CUDA_CHECK(ctx, cudaOccupancyMaxActiveClusters(&ctx->ffn_clusters[which], kern, &cfg));
        ctx->ffn_clusters[which] = std::max(1, ctx->ffn_clusters[which]);
    }
    *n = ctx->ffn_clusters[which];
    return TB200_OK;
}

}    // namespace

// A warp of a grid each, which has no more CTAs than the device SMs (gradients' launches: no 4-bit weights).
int64_t pair_peaks(const tb200_ctx* ctx)
{
    return (int64_t)std::max(2, ctx->num_sms) * (Shape<true>::kThreads / 32);
}

tb200_status pair_launch(tb200_ctx* ctx, const PairProduct& q)
{
    // Pairs, or CTAs by themselves, K shared by up to eight: by their cycles.  A chunk of K takes a pair 520 and a CTA by itself 330, up to 700 when
    // all SMs run one, since their smaller tiles move twice the bytes for a product; with 4-bit weights, whose values pass through shared
    // memory twice, 690 and 490.  The last tile's epilogue shows, and so does the exchange of the shares' sums.
    const bool gated     = q.kind != PAIR_PLAIN;
    const int64_t copies = (int64_t)q.NB * (q.results == 2 && !gated ? 2 : 1), chunks = (q.K + 63) / 64 * q.phases;
    auto tiles = [&](int rows, int cols) { return (int64_t)((q.rows + rows - 1) / rows) * ((q.cols + cols - 1) / cols) * copies; };
    auto waves = [&](int64_t n, int64_t at_once) { return (double)((n + at_once - 1) / at_once); };
    const int64_t large = tiles(256, gated ? 128 : 256), small = tiles(128, gated ? 64 : 128);
    double best = waves(large, ctx->num_sms / 2) * (double)chunks * (!q.w4 ? 520.0 : gated ? 1100.0 : 690.0) + 4500.0;
    int splits  = 0;
    for (int s = 1, i = 0; s <= 8; s *= 2, i++)
    {
        if (s > 1 && (chunks < 4 * s || small * s > ctx->num_sms))
            break;
        const double chunk = q.w4 ? (gated ? 700.0 : 490.0) : std::max(330.0, 700.0 * (double)std::min<int64_t>(small * s, ctx->num_sms) / ctx->num_sms);
        double cost        = waves(small, ctx->num_sms) * (double)chunks * chunk + 2500.0;
        if (s > 1)
        {
            // a share does one tile; clusters of four fill 132 of 148 SMs, of eight 120 (70 x 2048 x 2048 with 4-bit weights: 18 us, 10 by fours)
            int at_once        = 0;
            const tb200_status st = clusters_at_once(ctx, i - 1, s, &at_once);
            if (st != TB200_OK)
                return st;
            cost = waves(small, at_once) * ((double)((chunks + s - 1) / s) * chunk + 2500.0) + 2500.0;
        }
        if (cost < best)
        {
            best   = cost;
            splits = s;
        }
    }
    return splits ? launch<false>(ctx, q, splits) : launch<true>(ctx, q, 1);
}

}    // namespace ffn
}    // namespace tb200
