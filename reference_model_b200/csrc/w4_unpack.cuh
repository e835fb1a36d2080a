// Nibbles of 4-bit weights to 16-bit numbers.
#pragma once
#include <cstdint>

namespace tb200
{
namespace ffn
{

__device__ __forceinline__ uint32_t fma2_bf16(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

__device__ __forceinline__ uint32_t fma2_f16(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// (w & m) ^ x in one instruction
__device__ __forceinline__ uint32_t and_xor(uint32_t w, uint32_t m, uint32_t x)
{
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(d) : "r"(w), "r"(m), "r"(x));
    return d;
}

// Eight elements to four pairs (0,4), (1,5), (2,6), (3,7), minus their zero point; `base` holds -(136 + z) twice (fp16: -(1032 + z)).
// One multiply-add by 1 takes it off (a bf16 subtraction of pairs is no instruction of its own: ncu counted five in its place).
// fp16 reads every second pair four bits higher, as 1024 + 16 (8 + q), and scales by 1/16 in the same multiply-add: one shift in place of three.
template <bool BF16>
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t base, uint32_t (&p)[4])
{
    if (BF16)
    {
#pragma unroll
        for (int i = 0; i < 4; i++)
            p[i] = fma2_bf16(and_xor(w >> (4 * i), 0x000F000Fu, 0x43084308u), 0x3F803F80u, base);
    }
    else
    {
        const uint32_t high = fma2_f16(base, 0x3C003C00u, 0x63806380u);    // 960 - (1032 + z) = -(72 + z)
        const uint32_t v    = w >> 8;
        p[0]                = fma2_f16(and_xor(w, 0x000F000Fu, 0x64086408u), 0x3C003C00u, base);
        p[1]                = fma2_f16(and_xor(w, 0x00F000F0u, 0x64806480u), 0x2C002C00u, high);
        p[2]                = fma2_f16(and_xor(v, 0x000F000Fu, 0x64086408u), 0x3C003C00u, base);
        p[3]                = fma2_f16(and_xor(v, 0x00F000F0u, 0x64806480u), 0x2C002C00u, high);
    }
}

__device__ __forceinline__ uint4 lds128(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// minus the zero point as unpack8 takes it
template <bool BF16>
__device__ __forceinline__ uint32_t unpack_base(int z)
{
    return (BF16 ? 0xC308C308u : 0xE408E408u) + (uint32_t)z * 0x10001u;
}

}    // namespace ffn
}    // namespace tb200
