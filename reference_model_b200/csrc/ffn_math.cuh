// Activations of the gated product, their derivatives, and rounding to the output's type.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"

namespace tb200
{
namespace ffn
{

// The logistic forms go through e = exp(-|x|): s(x) = 1 / (1 + e) or e / (1 + e) and s(x) s(-x) = e / (1 + e)^2 neither cancel nor overflow on either
// side (1 - s has no digits left from x = 17 on).  The Gaussian one goes through erfc, whose relative error stays small in the left tail where
// 1 + erf would cancel.
struct Logistic
{
    float s, product;    // s(x), s(x) s(-x)
};

__device__ __forceinline__ Logistic logistic(float x, float e, float reciprocal)
{
    return { (x < 0.f ? e : 1.f) * reciprocal, e * reciprocal * reciprocal };
}

__device__ __forceinline__ Logistic logistic(float x)
{
    const float e = expf(-fabsf(x));
    return logistic(x, e, 1.f / (1.f + e));
}

// what GELU_TANH gives to it: (1 + tanh(y)) / 2 = s(2 y)
__device__ __forceinline__ float tanh_argument(float g)
{
    return 1.5957691216057308f * (g + 0.044715f * g * g * g);
}

// Value of the activation.
template <int ACT>
__device__ __forceinline__ float act_value(float g)
{
    if (ACT == TB200_ACT_SILU)
        return g * logistic(g).s;
    if (ACT == TB200_ACT_GELU)
        return 0.5f * g * erfcf(-0.70710678118654752f * g);
    if (ACT == TB200_ACT_GELU_TANH)
        return g * logistic(tanh_argument(g)).s;
    if (ACT == TB200_ACT_RELU)
        return g < 0.f ? 0.f : g;    // a NaN stays one
    return logistic(g).s;
}

// 1 + 3 * 0.044715 g^2 of GELU_TANH's derivative.  Where s (1 - s) has long been 0 the square must not overflow beside it.
__device__ __forceinline__ float tanh_growth(float g)
{
    const float c = fminf(fabsf(g), 1e9f);
    return 1.f + 0.134145f * c * c;
}

// Value and derivative of a logistic form
template <int ACT>
__device__ __forceinline__ void logistic_slope(float g, const Logistic& l, float& value, float& slope)
{
    value = ACT == TB200_ACT_SIGMOID ? l.s : g * l.s;
    slope = ACT == TB200_ACT_SIGMOID ? l.product
            : ACT == TB200_ACT_SILU  ? l.s + g * l.product
                                     : l.s + g * l.product * 1.5957691216057308f * tanh_growth(g);
}

// Value and derivative.
template <int ACT>
__device__ __forceinline__ void act_slope(float g, float& value, float& slope)
{
    if (ACT == TB200_ACT_SILU || ACT == TB200_ACT_SIGMOID || ACT == TB200_ACT_GELU_TANH)
        logistic_slope<ACT>(g, logistic(ACT == TB200_ACT_GELU_TANH ? tanh_argument(g) : g), value, slope);
    else if (ACT == TB200_ACT_GELU)
    {
        const float p = 0.5f * erfcf(-0.70710678118654752f * g);
        value         = g * p;
        slope         = p + g * (0.39894228040143268f * expf(-0.5f * g * g));
    }
    else
    {
        value = g < 0.f ? 0.f : g;
        slope = g > 0.f ? 1.f : g <= 0.f ? 0.f : g;
    }
}

// The same for results that are rounded to 16 bits: exp by the hardware's power of two (relative error about 2^-21 |x|), quotients by its
// reciprocal, and the Gaussian's tail by a polynomial: erfc(x) = t (c0 + c1 t + ... + c7 t^7) exp(-x^2) with t = 1 / (1 + 0.44 x), the coefficients
// fitted to erfc(x) exp(x^2) / t over all x >= 0 by weighted least squares (Lawson's iteration).  Within 3.2e-8 of erfc for small x and 6.2e-6 of its value
// for all, which a bound on the difference alone does not give: f(-6) is 1e-9, and the next factor may be large.
// 4 x 197 x 1000 x 1416 fp16 with GELU: 14.5 us with these, 16.1 with the functions for fp32 values below; 700 x 1024 x 2048 bf16 with SILU 11.7 and 12.4.
__device__ __forceinline__ float erfc_positive(float x, float e)
{
    const float t = __fdividef(1.f, fmaf(0.44f, x, 1.f));
    float c       = 0.0631131908f;
    c             = fmaf(c, t, -0.244836184f);
    c             = fmaf(c, t, 0.241915805f);
    c             = fmaf(c, t, 0.0266969014f);
    c             = fmaf(c, t, 0.193881295f);
    c             = fmaf(c, t, 0.222735351f);
    c             = fmaf(c, t, 0.24824873f);
    c             = fmaf(c, t, 0.248244942f);
    return t * c * e;
}

__device__ __forceinline__ Logistic logistic_16(float x)
{
    const float e = __expf(-fabsf(x));
    return logistic(x, e, __fdividef(1.f, 1.f + e));
}

template <int ACT>
__device__ __forceinline__ float act_value_16(float g)
{
    if (ACT == TB200_ACT_SILU)
        return g * logistic_16(g).s;
    if (ACT == TB200_ACT_GELU_TANH)
        return g * logistic_16(tanh_argument(g)).s;
    if (ACT == TB200_ACT_SIGMOID)
        return logistic_16(g).s;
    if (ACT == TB200_ACT_GELU)
    {
        const float tail = 0.5f * erfc_positive(0.70710678118654752f * fabsf(g), __expf(-0.5f * g * g));
        return g * (g < 0.f ? tail : 1.f - tail);
    }
    return act_value<ACT>(g);
}

template <int ACT>
__device__ __forceinline__ void act_slope_16(float g, float& value, float& slope)
{
    if (ACT == TB200_ACT_SILU || ACT == TB200_ACT_SIGMOID || ACT == TB200_ACT_GELU_TANH)
        logistic_slope<ACT>(g, logistic_16(ACT == TB200_ACT_GELU_TANH ? tanh_argument(g) : g), value, slope);
    else if (ACT == TB200_ACT_GELU)
    {
        const float e    = __expf(-0.5f * g * g);
        const float tail = 0.5f * erfc_positive(0.70710678118654752f * fabsf(g), e);
        const float p    = g < 0.f ? tail : 1.f - tail;
        value            = g * p;
        slope            = p + g * (0.39894228040143268f * e);
    }
    else
        act_slope<ACT>(g, value, slope);
}

// Values that stay in fp32 where 16 of a thread's are made at a time: CUDA's functions, but for the quotient, which takes the hardware's reciprocal (two units
// in the last place of a number in 1 .. 2).
template <int ACT>
__device__ __forceinline__ float act_value_32(float g)
{
    if (ACT == TB200_ACT_GELU || ACT == TB200_ACT_RELU)
        return act_value<ACT>(g);
    const float x = ACT == TB200_ACT_GELU_TANH ? tanh_argument(g) : g, e = expf(-fabsf(x));
    const float s = logistic(x, e, __fdividef(1.f, 1.f + e)).s;
    return ACT == TB200_ACT_SIGMOID ? s : g * s;
}

__device__ __forceinline__ float act_value(int act, float g)
{
    switch (act)
    {
        case TB200_ACT_SILU: return act_value<TB200_ACT_SILU>(g);
        case TB200_ACT_GELU: return act_value<TB200_ACT_GELU>(g);
        case TB200_ACT_GELU_TANH: return act_value<TB200_ACT_GELU_TANH>(g);
        case TB200_ACT_RELU: return act_value<TB200_ACT_RELU>(g);
        default: return act_value<TB200_ACT_SIGMOID>(g);
    }
}

__device__ __forceinline__ void act_slope(int act, float g, float& value, float& slope)
{
    switch (act)
    {
        case TB200_ACT_SILU: act_slope<TB200_ACT_SILU>(g, value, slope); break;
        case TB200_ACT_GELU: act_slope<TB200_ACT_GELU>(g, value, slope); break;
        case TB200_ACT_GELU_TANH: act_slope<TB200_ACT_GELU_TANH>(g, value, slope); break;
        case TB200_ACT_RELU: act_slope<TB200_ACT_RELU>(g, value, slope); break;
        default: act_slope<TB200_ACT_SIGMOID>(g, value, slope); break;
    }
}

__device__ __forceinline__ float act_value_16(int act, float g)
{
    switch (act)
    {
        case TB200_ACT_SILU: return act_value_16<TB200_ACT_SILU>(g);
        case TB200_ACT_GELU: return act_value_16<TB200_ACT_GELU>(g);
        case TB200_ACT_GELU_TANH: return act_value_16<TB200_ACT_GELU_TANH>(g);
        case TB200_ACT_RELU: return act_value_16<TB200_ACT_RELU>(g);
        default: return act_value_16<TB200_ACT_SIGMOID>(g);
    }
}

__device__ __forceinline__ float act_value_32(int act, float g)
{
    switch (act)
    {
        case TB200_ACT_SILU: return act_value_32<TB200_ACT_SILU>(g);
        case TB200_ACT_GELU: return act_value_32<TB200_ACT_GELU>(g);
        case TB200_ACT_GELU_TANH: return act_value_32<TB200_ACT_GELU_TANH>(g);
        case TB200_ACT_RELU: return act_value_32<TB200_ACT_RELU>(g);
        default: return act_value_32<TB200_ACT_SIGMOID>(g);
    }
}

__device__ __forceinline__ void act_slope_16(int act, float g, float& value, float& slope)
{
    switch (act)
    {
        case TB200_ACT_SILU: act_slope_16<TB200_ACT_SILU>(g, value, slope); break;
        case TB200_ACT_GELU: act_slope_16<TB200_ACT_GELU>(g, value, slope); break;
        case TB200_ACT_GELU_TANH: act_slope_16<TB200_ACT_GELU_TANH>(g, value, slope); break;
        case TB200_ACT_RELU: act_slope_16<TB200_ACT_RELU>(g, value, slope); break;
        default: act_slope_16<TB200_ACT_SIGMOID>(g, value, slope); break;
    }
}

__device__ __forceinline__ float load_fp(const void* p, int64_t i, tb200_dtype dt)
{
    if (dt == TB200_FP32)
        return reinterpret_cast<const float*>(p)[i];
    if (dt == TB200_FP16)
        return __half2float(reinterpret_cast<const __half*>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

// The number that an element's bits stand for
__device__ __forceinline__ float bits_fp(uint32_t bits, tb200_dtype dt)
{
    return dt == TB200_FP32 ? __uint_as_float(bits) : dt == TB200_BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
}

// Results are rounded once, to nearest, where they are stored.
__device__ __forceinline__ void store_fp(void* p, int64_t i, tb200_dtype dt, float v)
{
    if (dt == TB200_FP32)
        reinterpret_cast<float*>(p)[i] = v;
    else if (dt == TB200_FP16)
        reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// The sixteen bytes from byte `by` of two neighbouring sixteens
__device__ __forceinline__ uint4 shifted_piece(const uint4& lo, const uint4& hi, int by)
{
    uint32_t w[8] = { lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w };
    if (by & 4)
    {
#pragma unroll
        for (int i = 0; i < 7; i++)
            w[i] = w[i + 1];
    }
    if (by & 8)
    {
#pragma unroll
        for (int i = 0; i < 6; i++)
            w[i] = w[i + 2];
    }
    const int bits = (by & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16)
{
    if (bf16)
    {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float2 unpack2(uint32_t w, bool bf16)
{
    if (bf16)
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

}    // namespace ffn
}    // namespace tb200
