// What the tensor-core kernels share: barriers and copies (mbarrier, TMA), tcgen05 products and tensor memory, the exact values
// of packed codes, and tensor maps.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <mutex>
#include <vector>

#include "and_or.h"

namespace eoq {
namespace {

__device__ __forceinline__ uint32_t saddr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Whether a phase is over, without waiting (a try_wait, whose answer may take until it is, would keep the warp).
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// A barrier answers each lane for itself, and where it completes meanwhile they are told different things.  One answer for the
// warp, for waits behind which the lanes vote or elect together: a lane that had gone on alone would be missing there.
__device__ __forceinline__ bool for_the_warp(bool yes) { return __all_sync(0xffffffffu, yes); }

// The last uses of a ring of n barriers, of which `used` have been made: what the copy engine still has to bring is
// there (or does not come for some ten milliseconds) before the CTA may leave its shared memory.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t used, uint32_t n)
{
    const long long t0 = clock64();
    for (uint32_t u = used > n ? used - n : 0u; u < used; u++)
        while (!bar_try(bar + 8u * (u % n), (u / n) & 1u))
            if (clock64() - t0 > 20000000ll) return;
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
// One lane of the warp, the same in every call.  The loops that issue copies and products run on all lanes and elect one
// for these instructions only: their operands then stay in the warp's uniform registers (from a branch that one lane had
// taken alone, four products and two commits took 1900 cycles).
__device__ __forceinline__ bool elect()
{
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// K-major tile with the 128-byte swizzle: rows of 128 bytes, groups of eight rows 1024 bytes apart
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) { uint32_t r; asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c)); return r; }
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) { uint32_t r; asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) { uint32_t r; asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t bfma2(uint32_t a, uint32_t b, uint32_t c) { uint32_t r; asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c)); return r; }
__device__ __forceinline__ uint32_t bsub2(uint32_t a, uint32_t b) { uint32_t r; asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) { uint32_t r; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }
__device__ __forceinline__ uint32_t dup_byte(uint32_t w, uint32_t j) { return __byte_perm(w, 0u, 0x1111u * j); }

// Code pairs in their natural order, exact, from one word (4 bits: eight codes; 2 bits: sixteen; 8 bits: four).  A byte is
// put into both halves of a register; each half keeps its own bits under the exponent of 1024 (bf16: 128), which
// makes it 1024 + 2^s code, and one fused multiply-add with a constant pair takes the shift and the offset out: three
// instructions for two codes.  A bf16 has no mantissa bit for the upper nibble, so that one comes from the word shifted
// right by four.
template <int BITS, bool BF16>
__device__ __forceinline__ void codes_exact(uint32_t w, uint32_t *h)
{
    if (BITS == 4) {
        const uint32_t u = w >> 4;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
            if (BF16) h[j] = bsub2(and_or(__byte_perm(w, u, 0x4400u + 0x1111u * j), 0x000F000Fu, 0x43004300u), 0x43074307u);
            else h[j] = hfma2(and_or(dup_byte(w, j), 0x00F0000Fu, 0x64006400u), 0x2C003C00u, 0xD470E407u);
    } else if (BITS == 2) {
        const uint32_t u = w >> 4;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            if (BF16) {
                h[2 * j] = bfma2(and_or(dup_byte(w, j), 0x000C0003u, 0x43004300u), 0x3E803F80u, 0xC204C301u);
                h[2 * j + 1] = bfma2(and_or(dup_byte(u, j), 0x000C0003u, 0x43004300u), 0x3E803F80u, 0xC204C301u);
            } else {
                const uint32_t b = dup_byte(w, j);
                h[2 * j] = hfma2(and_or(b, 0x000C0003u, 0x64006400u), 0x34003C00u, 0xDC04E401u);
                h[2 * j + 1] = hfma2(and_or(b, 0x00C00030u, 0x64006400u), 0x24002C00u, 0xCC40D410u);
            }
        }
    } else {
        const uint32_t u = w ^ 0x80808080u;          // code + 128
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
            if (BF16) {
                // 128 + u needs nine significant bits, a bf16 has eight: through fp32 (2^23 + u), exact
                const float f0 = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540u | (2 * j))) - 8388736.0f;
                const float f1 = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540u | (2 * j + 1))) - 8388736.0f;
                h[j] = pack_bf16(f0, f1);
            } else {
                h[j] = hsub2(__byte_perm(u, 0x64646464u, j ? 0x4342u : 0x4140u), 0x64806480u);
            }
        }
    }
}

// The same times the scale, rounded once: fp16 by one multiplication of the exact code; bf16 in fp32, where
// (128 + 2^s code) (scale / 2^s) - offset scale is exact in one fused multiply-add, then one rounding to the pair.
template <int BITS, bool BF16>
__device__ __forceinline__ void codes_scaled(uint32_t w, uint32_t *h, uint16_t sbits)
{
    if (!BF16) {
        codes_exact<BITS, false>(w, h);
        const uint32_t s2 = sbits | ((uint32_t)sbits << 16);
#pragma unroll
        for (int i = 0; i < 16 / BITS; i++) h[i] = hmul2(h[i], s2);
        return;
    }
    const float s = __half2float(__ushort_as_half(sbits));
    auto pair = [](uint32_t t, float m0, float c0, float m1, float c1) {
        return pack_bf16(fmaf(__uint_as_float(t << 16), m0, c0), fmaf(__uint_as_float(t & 0xFFFF0000u), m1, c1));
    };
    const uint32_t u = w >> 4;
    if (BITS == 4) {
        const float c = -135.0f * s;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) h[j] = pair(and_or(__byte_perm(w, u, 0x4400u + 0x1111u * j), 0x000F000Fu, 0x43004300u), s, c, s, c);
    } else if (BITS == 2) {
        const float q = 0.25f * s, c0 = -129.0f * s, c1 = -33.0f * s;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            h[2 * j] = pair(and_or(dup_byte(w, j), 0x000C0003u, 0x43004300u), s, c0, q, c1);
            h[2 * j + 1] = pair(and_or(dup_byte(u, j), 0x000C0003u, 0x43004300u), s, c0, q, c1);
        }
    } else {
        const uint32_t v = w ^ 0x80808080u;
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
            const float f0 = __uint_as_float(__byte_perm(v, 0x4B000000u, 0x7540u | (2 * j))) - 8388736.0f;
            const float f1 = __uint_as_float(__byte_perm(v, 0x4B000000u, 0x7540u | (2 * j + 1))) - 8388736.0f;
            h[j] = pack_bf16(f0 * s, f1 * s);
        }
    }
}

// two fp32 in a register pair
__device__ __forceinline__ uint64_t pack2(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float low2(uint64_t v) { float a, b; asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); return a; }
__device__ __forceinline__ float high2(uint64_t v) { float a, b; asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); return b; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) { uint64_t r; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                   "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
                   "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
                   "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr) : "memory");
}
// The values of a load exist after this only: they go through it, so that no use can be scheduled in front of it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}

// Position in a ring of n stages and the parity of its current lap.
struct Ring {
    uint32_t at = 0, lap = 0;
    __device__ __forceinline__ void next(uint32_t n) { if (++at == n) { at = 0; lap ^= 1u; } }
};

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn()
{
    static EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

bool map_2d(CUtensorMap &m, CUtensorMapDataType type, const void *p, uint64_t inner, uint64_t rows, uint64_t row_bytes, uint32_t box_inner,
            uint32_t box_rows, CUtensorMapSwizzle sw)
{
    const cuuint64_t dims[2] = {inner, rows}, strides[1] = {row_bytes};
    const cuuint32_t box[2] = {box_inner, box_rows}, step[2] = {1, 1};
    EncodeFn fn = encode_fn();
    return fn && fn(&m, type, 2, const_cast<void *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// CTAs of a kernel in clusters of `split` that fit on the device at once, asked once per kernel, size and shared memory.
uint32_t resident_ctas(const void *kern, uint32_t threads, size_t smem, uint32_t split)
{
    struct Known { const void *k; size_t smem; uint32_t split; int dev; uint32_t n; };
    static std::mutex mu;
    static std::vector<Known> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    std::lock_guard<std::mutex> lock(mu);
    for (const Known &k : known) if (k.k == kern && k.smem == smem && k.split == split && k.dev == dev) return k.n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) { (void)cudaGetLastError(); n = 0; }
    known.push_back(Known{kern, smem, split, dev, (uint32_t)std::max(n, 0) * split});
    return known.back().n;
}

}  // namespace
}  // namespace eoq
