// Warp-level tensor-core products with packed codes: the instruction, and a lane's codes as exact 16-bit floats in the order in
// which they leave their words cheapest.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "and_or.h"

namespace eoq {
namespace {

template <bool BF16>
__device__ __forceinline__ void mma_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the first instruction of a chain: D = A * B + 0 (the zeros are operands, not four registers to clear)
template <bool BF16>
__device__ __forceinline__ void mma_m16n8k16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// two codes, already sitting in the low bits of the two halves of v, to two exact signed 16-bit floats
template <bool BF16>
__device__ __forceinline__ uint32_t codes_to_pair(uint32_t v, uint32_t mask, uint32_t q)
{
    const uint32_t magic = BF16 ? 0x43004300u : 0x64006400u;
    const uint32_t biased = and_or(v, mask, magic), off = magic | q | (q << 16);
    uint32_t r;
    if (BF16) asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(biased), "r"(off));
    else asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(biased), "r"(off));
    return r;
}

// For fp16 the odd positions of a word are taken without a shift: (w & 0x00F000F0) | 0x6400 is 1024 + 16 code, one
// fused multiply-add (x 1/16, - 71) the signed code; the 2-bit codes likewise with 1/4, 1/16, 1/64.
template <bool BF16>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t v, uint32_t mask, uint32_t mul, uint32_t sub)
{
    static_assert(!BF16, "a bf16 mantissa has no room above bit 6");
    const uint32_t biased = and_or(v, mask, 0x64006400u);
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(biased), "r"(mul | (mul << 16)), "r"(sub | (sub << 16)));
    return r;
}

// the 16 / BITS registers of signed 16-bit float pairs of one word's codes, in the order the word gives them
template <int BITS, bool BF16>
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t (&h)[16 / BITS])
{
    if constexpr (BITS == 4) {          // register i: columns i and i + 4
        if (BF16) {
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = codes_to_pair<BF16>(w >> (4 * i), 0x000F000Fu, 7u);
        } else {
            const uint32_t u = w >> 8;
            h[0] = codes_to_pair<false>(w, 0x000F000Fu, 7u);
            h[1] = scaled_pair<false>(w, 0x00F000F0u, 0x2C00u, 0xD470u);       // (1024 + 16 c) / 16 - 71
            h[2] = codes_to_pair<false>(u, 0x000F000Fu, 7u);
            h[3] = scaled_pair<false>(u, 0x00F000F0u, 0x2C00u, 0xD470u);
        }
    } else if constexpr (BITS == 2) {   // register i: columns i and i + 8
        if (BF16) {
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = codes_to_pair<BF16>(w >> (2 * i), 0x00030003u, 1u);
        } else {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t u = w >> (8 * half);
                h[4 * half + 0] = codes_to_pair<false>(u, 0x00030003u, 1u);
                h[4 * half + 1] = scaled_pair<false>(u, 0x000C000Cu, 0x3400u, 0xDC04u);   // / 4 - 257
                h[4 * half + 2] = scaled_pair<false>(u, 0x00300030u, 0x2C00u, 0xD410u);   // / 16 - 65
                h[4 * half + 3] = scaled_pair<false>(u, 0x00C000C0u, 0x2400u, 0xCC40u);   // / 64 - 17
            }
        }
    } else if constexpr (!BF16) {       // signed bytes: u = code + 128 under 0x64 is 1024 + u; register i: columns 2i, 2i + 1
#pragma unroll
        for (int i = 0; i < 2; i++)
            h[i] = codes_to_pair<false>(__byte_perm(w ^ 0x80808080u, 0u, i ? 0x4342u : 0x4140u), 0x00FF00FFu, 128u);
    } else {
        // 128 + u needs nine significant bits, a bf16 has eight: the byte goes under 0x4B (2^23 + u as an fp32), one
        // exact subtraction gives the code, and two codes are packed into a bf16 pair (|code| <= 128: exact)
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float f0 = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540u | (2 * i))) - 8388736.0f;
            const float f1 = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540u | (2 * i + 1))) - 8388736.0f;
            const __nv_bfloat162 b = __floats2bfloat162_rn(f0, f1);
            h[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
    }
}

// the 16 registers of a lane's 32 columns of one row
template <int BITS, bool BF16>
__device__ __forceinline__ void unpack_span(const uint32_t (&w)[BITS], uint32_t (&h)[16])
{
    constexpr int kEach = 16 / BITS;
#pragma unroll
    for (int j = 0; j < BITS; j++) {
        uint32_t r[kEach];
        unpack_word<BITS, BF16>(w[j], r);
#pragma unroll
        for (int i = 0; i < kEach; i++) h[kEach * j + i] = r[i];
    }
}

}  // namespace
}  // namespace eoq
