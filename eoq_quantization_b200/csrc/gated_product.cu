// The gated block on the fifth-generation tensor cores, straight from packed codes:
//   forward   h[m][n] = act(g + bg) (u + bu),  g = sum over k of x[m][k] wg[n][k], u likewise
//   gradient  dx[m][k] = sum over n of dg[m][n] wg[n][k] + du[m][n] wu[n][k]   (or of one weight)
//
// Both are products of weight tiles of 256 rows, which are the A operand and live in the tensor memory of two SMs (cta_group::2,
// 128 rows each), with up to 256 tokens, which are the B operand, brought by TMA (128-byte swizzle), half to each SM: alone, an SM
// would need 64 bytes of activations a clock to keep its tensor cores busy, which is more than the L2 gives all of them.  Packed codes
// come by TMA too; producer warps turn them into code x scale, rounded to fp16 once, and store them to tensor memory, so that a
// dequantised weight touches neither global nor shared memory.  Activations are fp16, with one power of two per row where they were
// something else.
//
//   forward: a CTA's 128 rows are 64 features of the gate and the same 64 of the up projection, so that h is made where both
// sums are, on the way out.  A thread owns a row and turns 64 of its codes at a time into A's 32 columns.
//   gradient: a CTA's 128 rows are 128 columns of the weights, and the products run over the weights' rows, gate's first.  The
// codes lie the wrong way for that: a matrix load from shared memory transposes them, 16 bits (two, four or eight codes of a
// weight row) at a time, and leaves in each register the codes of two neighbouring weight rows at the same columns, half and
// half: what masking and a packed multiply-add make of it is a pair along the products' axis.  Its lanes are then sets of
// columns, not neighbouring ones; tensor memory takes them in that order, and the way out puts them back (`place`).
//
// The grid is at most as many CTA pairs as the device holds, and the work, tile after tile along the products' axis, is cut into as many
// equal runs (`plan_for`): of whole tiles, or a pair takes the end of one tile, whole ones, and the beginning of another, and nothing waits
// for a last, partly filled round.  Sums of a tile that several pairs share go to scratch; whoever comes last, by the tile's counter, adds
// them up in the order of the pairs and finishes the tile, so results do not depend on who that is.  Copies, conversion and products run on
// from one tile to the next while four warps bring the last one out; two accumulators take turns where tensor memory has room for them
// (tiles of up to 160 tokens).
//
// Measured (4 bits, fp16, back to back, codes from HBM; in brackets the products at 1688 TFLOP/s): 11008 x 4096, forward 64 rows 36 us (7.5),
// 256 65 (27), 777 131 (83), 2048 313 (219); gradient of one weight 512 rows 48 (27), 1024 70 (55), 2048 137 (109); 28672 x 8192, 2048 rows
// 1540 (1140; long runs at full power meet 1422 TFLOP/s, 1353) and 715 (570).  What bounds it: with tiles of 256 tokens the tensor pipe (79 % of
// active cycles for gradients of 1024 rows; 56 % forward at 777), beside it the producers' issue slots (70 % forward) and, where tensor memory
// holds one accumulator, the way out between two tiles; few rows: 430 clocks a block of 64, the producers' hand-over, whatever the tokens.
// Six producer sets, because a set's block takes some 2500 clocks from its codes' arrival to its operand's: four gave 650 clocks a block.
//
// A product of code and scale that fp16 has no room for makes its sums infinities or NaN: the way out looks for such, and computes a tile
// again in fp32 where the weights' scales can be why (11008 x 4096 with all scales at 20000: 64 rows 10 ms; 27 us for the look at the
// scales of a gradient that has a NaN of its own).
//
// Waits are bounded, as in the product kernel for one weight (qmm.cu): one that runs out marks the CTA, whose results become NaN,
// and sets a status word.
#include "gated.h"
#include "tensor_core.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cooperative_groups.h>

#include "activations.cuh"

namespace cg = cooperative_groups;

namespace eoq {

__device__ uint32_t g_gated_status = 0;

namespace {

constexpr uint32_t kRows = 128;            // of a weight tile
constexpr int kSets = 6;                   // producer sets of four warps, one per quadrant of tensor memory
constexpr int kWProducts = 4 * kSets, kWCodes = kWProducts + 1, kWTokens = kWProducts + 2, kWScales = kWProducts + 3, kWOut = kWProducts + 4;      // warps
constexpr uint32_t kThreads = (kWOut + 4) * 32, kTmem = 512, kOut = 8 * 2048 + 8 * 128;       // shared memory of the way out: sixteen tokens of a warp, and their maxima, twice

struct ProductArgs {
    const uint16_t *scales[2];   // [N][groups] fp16
    const void *bias[2];         // forward: [N] of bias_dtype, or null
    const float *factor;         // [M] or null
    const uint8_t *codes[2];     // [N][row_bytes]
    const uint16_t *x;           // fp16 [M][pitch] or, gradient, [weights][M][pitch]
    void *y;                     // [M][N] or, gradient, [M][K]
    Kept keep;                   // forward
    float *partial;              // [pairs][2][2][T][128]: sums of tiles that a pair's run begins (0) or ends (1) in the middle of
    uint32_t *count;             // [tiles][2], zero: parts of a tile that have arrived
    uint32_t N, K, M, T, group, groups, row_bytes, pitch;
    uint32_t tok_tiles, tiles, per_tile, per_weight, unit;         // of the grid of tiles; pieces of a tile's axis, of one weight's
    uint32_t nw, ns, nd;         // stages of packed weights and of operands, accumulators
    uint32_t at_x, at_out, at_bar;       // shared-memory offsets
    uint32_t inverse;            // group_of
    int dtype, act, bias_dtype;
    long long limit;             // clock ticks a wait may take
};

__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// at a barrier of either CTA.  What is handed over lies in tensor memory, whose order tcgen05's fences keep: without a scope of the cluster, which
// costs a fence of memory each time (920 clocks a block of 16 tokens, against 650).  A predicate, not a branch: the warp stays together.
__device__ __forceinline__ void arrive_cluster_if(uint32_t bar, bool yes)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar), "r"((uint32_t)yes) : "memory");
}
__device__ __forceinline__ void bar_arrive_if(uint32_t bar, bool yes)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar), "r"((uint32_t)yes) : "memory");
}
// a copy to this CTA whose bytes are counted by a barrier of either CTA of the pair
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
// The four products (K = 16 each) of a block, and `done` of both CTAs told when they are: one election for all five, for it is this warp's issue
// that bounds a block of few tokens (one each: 350 clocks a block).
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t done)
{
    asm volatile("{\n\t.reg .pred e, p;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
                 "setp.ne.u32 p, %4, 0;\n\tadd.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
                 "add.u64 b1, %2, 2;\n\tadd.u64 b2, %2, 4;\n\tadd.u64 b3, %2, 6;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t"
                 "@e tcgen05.mma.cta_group::2.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
                 "@e tcgen05.mma.cta_group::2.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
                 "@e tcgen05.mma.cta_group::2.kind::f16 [%0], [a3], b3, %3, 1;\n\t"
                 "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], %6;\n\t}"
                 ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(done), "h"((uint16_t)3) : "memory");
}
// arrives at this barrier of both CTAs when the products so far are done
__device__ __forceinline__ void commit_pair(uint32_t bar)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

// A wait that may sleep for a millisecond: warps that ask again and again take the issue slots of those that work.
__device__ __forceinline__ bool bar_try_long(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000000u) : "memory");
    return ok != 0;
}

// Two words of shared memory at `mark`: the CTA has given up; the kernels before this one have ended (their time does not count).  A warp
// whose wait has run out is `lost`: it runs on, but requests no copies and tells no barriers (an arrival beyond a barrier's count while a copy is
// under way would break it), so that the others' waits run out too.
struct Patience {
    uint32_t mark;
    long long limit;
    bool lost = false;
    __device__ __forceinline__ Patience(uint32_t m, long long l) : mark(m), limit(l) {}
    __device__ __forceinline__ bool stopped() const
    {
        uint32_t v;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(mark) : "memory");
        return v != 0;
    }
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity)
    {
        if (!for_the_warp(bar_try(bar, parity))) lost = slow(bar, parity, mark, limit) || lost;
    }
    static __device__ __noinline__ bool slow(uint32_t bar, uint32_t parity, uint32_t mark, long long limit)
    {
        long long t0 = clock64();
        bool gave_up = false;
        while (!gave_up && !(limit ? bar_try_long(bar, parity) : bar_try(bar, parity))) {
            const long long now = clock64();
            uint32_t stop, alone;
            asm volatile("ld.volatile.shared.v2.u32 {%0, %1}, [%2];" : "=r"(stop), "=r"(alone) : "r"(mark) : "memory");
            if (!alone && limit) t0 = now;
            // (all CTAs are there at the same time, so that their waits run out together: the status word, which stays set until it is asked
            // for, is nobody's reason to give up)
            gave_up = stop || now - t0 > limit;
        }
        gave_up = __any_sync(0xffffffffu, gave_up);
        if (gave_up) {
            asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(mark), "r"(1u) : "memory");
            *reinterpret_cast<volatile uint32_t *>(&g_gated_status) = 1u;
        }
        return gave_up;
    }
};

// What one weight copy brings, in blocks of 64 along the products' axis.
template <bool GRAD, int BITS>
struct Piece {
    static constexpr uint32_t kBytes = GRAD ? 16u * BITS : BITS == 2 ? 64u : 128u;      // of one row
    static constexpr uint32_t kAlong = GRAD ? 256u : kBytes * 8u / BITS;                 // along the products' axis
    static constexpr uint32_t kBlocks = kAlong / 64u;
    static constexpr uint32_t kStage = (GRAD ? kAlong : kRows) * kBytes;
};

// barriers, eight bytes each.  Of a pair's first CTA both use Full (its products' warp waits for both CTAs' operands) and OutEmpty.
enum { bWFull = 0, bWEmpty = 8, bFull = 16, bEmpty = 24, bOutFull = 32, bOutEmpty = 34, bTmem = 36, bDrain = 37, bMark = 38, bUsedW = 39, bTicket = 40, bEnd = 41 };
constexpr uint32_t kScales = 8u * kRows * 2u;      // of a stage of codes: forward, up to 8 groups x 128 rows; gradient, up to 4 groups x 256

__device__ __forceinline__ void ldmatrix_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// sixteen values exist from here on
__device__ __forceinline__ void use16(const uint32_t *r)
{
    asm volatile("" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]) : "memory");
}
// sixteen lanes x 32 columns: register 2 b to lane (thread / 4), column 4 b + thread % 4, register 2 b + 1 to lane 8 + thread / 4
__device__ __forceinline__ void tmem_st_16x128b(uint32_t addr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                   "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// Code pairs, one of each weight row, from the register of a transposed load; `j` counts the codes of the 16 bits.
template <int BITS>
__device__ __forceinline__ uint32_t row_pair(uint32_t w, int j)
{
    if (BITS == 4) {
        const uint32_t v = j & 2 ? w >> 8 : w;
        return j & 1 ? hfma2(and_or(v, 0x00F000F0u, 0x64006400u), 0x2C002C00u, 0xD470D470u) : hsub2(and_or(v, 0x000F000Fu, 0x64006400u), 0x64076407u);
    }
    if (BITS == 2) {       // (of the eight codes, the half that the caller has shifted down)
        if (j == 0) return hsub2(and_or(w, 0x00030003u, 0x64006400u), 0x64016401u);
        if (j == 1) return hfma2(and_or(w, 0x000C000Cu, 0x64006400u), 0x34003400u, 0xDC04DC04u);
        if (j == 2) return hfma2(and_or(w, 0x00300030u, 0x64006400u), 0x2C002C00u, 0xD410D410u);
        return hfma2(and_or(w, 0x00C000C0u, 0x64006400u), 0x24002400u, 0xCC40CC40u);
    }
    return hsub2(__byte_perm(w ^ 0x80808080u, 0x64646464u, j ? 0x4341u : 0x4240u), 0x64806480u);
}

// The column of the tile that lane `p` of quadrant `q` of tensor memory stands for.
template <bool GRAD, int BITS>
__device__ __forceinline__ uint32_t place(uint32_t q, uint32_t p)
{
    if (!GRAD) return q * 32u + p;
    if (BITS == 4) return q * 32u + 4u * (p & 7u) + (p >> 3);
    if (BITS == 2) return (q >> 1) * 64u + 8u * (p & 7u) + (q & 1u) * 4u + (p >> 3);
    return q * 32u + (p >> 4) * 16u + 2u * (p & 7u) + ((p >> 3) & 1u);
}

// Eight codes, BITS bytes, that lie together.
template <int BITS>
__device__ __forceinline__ void eight_codes(const uint8_t *from, float (&c)[8])
{
    if (BITS == 8) {
        const uint2 w = __ldg(reinterpret_cast<const uint2 *>(from));
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = (float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    } else {
        const uint32_t w = BITS == 4 ? __ldg(reinterpret_cast<const uint32_t *>(from)) : __ldg(reinterpret_cast<const uint16_t *>(from));
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = (float)((int)((w >> (BITS * i)) & ((1u << BITS) - 1u)) - ((1 << (BITS - 1)) - 1));
    }
}

// Sums of sixteen tokens again, in fp32 throughout, for weights that fp16 has no room for (beyond 65504, which takes scales above 511 for
// byte codes, 8188 for four bits): a thread goes through all codes of its row.  forward: of row n of a weight; gradient: of column n of all weights.
template <bool GRAD, int BITS>
__device__ __noinline__ void sums_in_fp32(const ProductArgs &a, uint32_t which, uint32_t n, uint32_t token, float (&v)[16])
{
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = 0.0f;
    auto add = [&](const uint16_t *x, const float (&w)[8]) {       // eight terms of each token
#pragma unroll
        for (uint32_t j = 0; j < 16; j++) {
            const uint4 q = __ldg(reinterpret_cast<const uint4 *>(x + (size_t)min(token + j, a.M - 1u) * a.pitch));
            const uint32_t p[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&p[i]));
                v[j] = fmaf(w[2 * i + 1], f.y, fmaf(w[2 * i], f.x, v[j]));
            }
        }
    };
    if constexpr (!GRAD) {
        for (uint32_t k = 0; k < a.K; k += 8u) {
            float w[8];
            eight_codes<BITS>(a.codes[which] + (size_t)n * a.row_bytes + k / 8u * BITS, w);
            const float s = __half2float(__ushort_as_half(__ldg(a.scales[which] + (size_t)n * a.groups + k / a.group)));
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] *= s;
            add(a.x + k, w);
        }
    } else {
        for (uint32_t weight = 0; weight * a.per_weight < a.per_tile; weight++)
            for (uint32_t r = 0; r < a.N; r += 8u) {
                float w[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    w[i] = 0.0f;
                    if (r + i >= a.N) continue;
                    float c[8];
                    eight_codes<BITS>(a.codes[weight] + (size_t)(r + i) * a.row_bytes + n / 8u * BITS, c);
#pragma unroll
                    for (uint32_t j = 0; j < 8; j++) if (j == n % 8u) w[i] = c[j];
                    w[i] *= __half2float(__ushort_as_half(__ldg(a.scales[weight] + (size_t)(r + i) * a.groups + n / a.group)));
                }
                add(a.x + (size_t)weight * a.M * a.pitch + r, w);
            }
    }
}

// Whether a scale of weights [w0, w1), of rows r0, r0 + step .. before r1 and groups [g0, g1), is such that a code times it may be beyond fp16.
template <int BITS>
__device__ __noinline__ bool beyond_fp16(const ProductArgs &a, uint32_t w0, uint32_t w1, uint32_t r0, uint32_t r1, uint32_t step, uint32_t g0, uint32_t g1)
{
    constexpr uint32_t kMost = BITS == 8 ? 0x5FFFu : BITS == 4 ? 0x6FFFu : 0x77FFu;        // 65504 / 128, / 8, / 2
    bool yes = false;
    for (uint32_t w = w0; w < w1; w++)
        for (uint32_t r = r0; r < r1; r += step)
            for (uint32_t g = g0; g < g1; g++) yes |= (__ldg(a.scales[w] + (size_t)r * a.groups + g) & 0x7FFFu) > kMost;
    return yes;
}

template <bool GRAD, int BITS>
__global__ void __launch_bounds__(kThreads, 1)
gated_product_kernel(const __grid_constant__ ProductArgs a, const __grid_constant__ CUtensorMap gmap, const __grid_constant__ CUtensorMap umap, const __grid_constant__ CUtensorMap xmap)
{
    using P = Piece<GRAD, BITS>;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    const uint32_t base = saddr(smem), bars = base + a.at_bar;
    auto bar = [&](uint32_t i) { return bars + 8u * i; };
    auto word = [&](uint32_t i) { return reinterpret_cast<volatile uint32_t *>(smem + a.at_bar + 8u * i); };
    Patience wait(bar(bMark), a.limit);
    const uint32_t scales_at = bars + 8u * bEnd + 8u;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
    const uint32_t rank = blockIdx.x & 1u, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t xstage = a.T * 64u, a_base = a.nd * a.T;          // half of a block's tokens; first column of A
    constexpr uint32_t kWide = GRAD ? 128u : 64u;                    // columns, or features, of a CTA's tile

    // A pair's run of pieces, and its parts of tiles.  Where its run ends inside a tile, that part comes first: then the next pair, which has the rest of
    // that tile and takes it up last but one run later, finds the other sums there and adds its own to them on the way out.  (In the run's order the sums of
    // shared tiles were added up when nothing else was left to do: 68 of 255 thousand clocks for a 11008 x 4096 gradient of 2048 rows.)
    auto run_start = [&](uint32_t p) { return (uint64_t)a.tiles * (a.per_tile / a.unit) * p / pairs * a.unit; };
    const uint64_t run0 = run_start(pair), run1 = run_start(pair + 1), cut = run1 - run1 % a.per_tile, head = cut > run0 && cut < run1 ? cut : run0;
    struct Part { uint32_t tile, p0, p1, blocks; };                  // pieces [p0, p1) of a tile, in blocks of 64
    auto part_at = [&](uint64_t at) {
        Part s;
        s.tile = (uint32_t)(at / a.per_tile);
        s.p0 = (uint32_t)(at - (uint64_t)s.tile * a.per_tile);
        s.p1 = (uint32_t)min((uint64_t)a.per_tile, s.p0 + (run1 - at));
        // forward: the last piece's blocks past the last column are left out; gradient: rows past the last one are zeros
        s.blocks = (GRAD ? s.p1 * P::kBlocks : min(s.p1 * P::kBlocks, (a.K + 63u) / 64u)) - s.p0 * P::kBlocks;
        return s;
    };
    auto go_on = [&](uint64_t &at, uint64_t &left, const Part &s) {
        left -= s.p1 - s.p0;
        at += s.p1 - s.p0;
        if (at == run1) at = run0;
    };
    // tokens fastest: the pairs that run at the same time share codes, which come from HBM, rather than activations, which the L2 holds
    auto first_row = [&](uint32_t tile) { return (tile / a.tok_tiles * 2u + rank) * kWide; };
    // k / group for groups of 32 columns and their multiples: with d = group / 16 and the inverse 2^32 / d rounded up, exact while (k / 16) d < 2^32
    auto group_of = [&](uint32_t k) { return __umulhi(k >> 4, a.inverse); };
    auto first_token = [&](uint32_t tile) { return tile % a.tok_tiles * a.T; };

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 8; i++) {
            bar_init(bar(bWFull + i), 2); bar_init(bar(bWEmpty + i), 4 * kSets);           // the copy and the scales; every producer warp
            bar_init(bar(bFull + i), 9); bar_init(bar(bEmpty + i), 1);                     // four producer warps of either CTA and the copies' bytes
        }
        for (uint32_t i = 0; i < 2; i++) { bar_init(bar(bOutFull + i), 1); bar_init(bar(bOutEmpty + i), 8); }
        bar_init(bar(bDrain), 1);
        word(bMark)[0] = word(bMark)[1] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == kWProducts) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar(bTmem)), "n"(kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    cg::this_cluster().sync();                 // both CTAs' barriers are there before either arrives at the other's
    fence_after();
    constexpr uint32_t tmem = 0;               // all 512 columns are this CTA's

    if (warp < 4 * kSets) {
        // ---- producers: codes, a block of 64 along the products' axis at a time, to the A operand in tensor memory.  The sets take the
        // blocks in turn, through all parts; every warp comes by every piece and gives it back.
        const uint32_t set = warp >> 2, q = warp & 3u, r = q * 32u + lane;
        const uint32_t lane_base = tmem + ((q * 32u) << 16) + a_base, full0 = in_cta(bar(bFull), 0u);
        Ring wr, ar;
        for (uint32_t j = 0; j < set; j++) ar.next(a.ns);
        uint32_t turn = set;                   // blocks until this set's next one
        for (uint64_t at = head, left = run1 - run0; left;) {
            const Part s = part_at(at);
            go_on(at, left, s);
            const uint32_t row0 = first_row(s.tile);
            for (uint32_t p = s.p0; p < s.p1; p++, wr.next(a.nw)) {
                static_assert(P::kBlocks <= kSets, "a set has one block of a piece, or none");
                const uint32_t have = GRAD ? P::kBlocks : min(P::kBlocks, (a.K + 63u) / 64u - p * P::kBlocks), ws = wr.at;
                const bool work = turn < have;
                wait(bar(bWFull + ws), wr.lap);
                uint32_t h[32];
                if (work) {
                    if constexpr (!GRAD) {
                        constexpr int kWords = BITS == 4 ? 8 : BITS == 2 ? 4 : 16;
                        const uint32_t row_at = base + ws * P::kStage + r * P::kBytes, sw = BITS == 2 ? (r >> 1) & 3u : r & 7u;
                        uint32_t w[kWords];
#pragma unroll
                        for (uint32_t c = 0; c < kWords / 4; c++)
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[4 * c]), "=r"(w[4 * c + 1]), "=r"(w[4 * c + 2]), "=r"(w[4 * c + 3])
                                         : "r"(row_at + (((turn * (kWords / 4) + c) ^ sw) << 4)));
                        // the groups of the block's halves, counted from the piece's first
                        const uint32_t c0 = p * P::kAlong, g0 = group_of(c0), k = c0 + turn * 64u;
                        uint16_t sc[2];
#pragma unroll
                        for (uint32_t j = 0; j < 2; j++)
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(sc[j]) : "r"(scales_at + ws * kScales + (group_of(min(k + j * 32u, a.K - 1u)) - g0) * (kRows * 2u) + r * 2u));
#pragma unroll
                        for (int c = 0; c < kWords; c++) codes_scaled<BITS, false>(w[c], h + c * (32 / kWords), c < kWords / 2 ? sc[0] : sc[1]);
                    } else {
                        constexpr int kChunks = BITS == 8 ? 2 : 1;            // 16-byte pieces of a weight row that a quadrant's 32 columns take
                        const uint32_t rows_at = base + ws * P::kStage, chunk = BITS == 4 ? q : BITS == 8 ? 2u * q : q >> 1;
                        // scales of neighbouring weight rows at this lane's columns' group
                        const uint32_t gl = group_of(row0 + place<true, BITS>(q, lane >> 2)) - group_of(row0);
                        uint32_t sp[8];
#pragma unroll
                        for (uint32_t b = 0; b < 8; b++)
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(sp[b]) : "r"(scales_at + ws * kScales + gl * (P::kAlong * 2u) + turn * 128u + b * 16u + (lane & 3u) * 4u));
                        uint32_t m[kChunks][2][4];
#pragma unroll
                        for (uint32_t c = 0; c < kChunks; c++)
#pragma unroll
                            for (uint32_t hh = 0; hh < 2; hh++) {
                                const uint32_t n = turn * 64u + hh * 32u + lane, sw = BITS == 8 ? n & 7u : BITS == 4 ? (n >> 1) & 3u : (n >> 2) & 1u;
                                ldmatrix_trans(rows_at + n * P::kBytes + (((chunk + c) ^ sw) << 4), m[c][hh]);
                            }
                        // sixteen lanes of tensor memory at a time: code j of the registers to lanes 0 .. 7, code j + 1 to lanes 8 .. 15
#pragma unroll
                        for (int half = 0; half < 2; half++)
#pragma unroll
                            for (int b = 0; b < 8; b++)
#pragma unroll
                                for (int j = 0; j < 2; j++) {
                                    uint32_t v = m[BITS == 8 ? half : 0][b >> 2][b & 3];
                                    if (BITS == 2) v >>= (q & 1u) * 8u;
                                    h[half * 16 + 2 * b + j] = hmul2(row_pair<BITS>(v, (BITS == 8 ? 0 : 2 * half) + j), sp[b]);
                                }
                    }
                    // every code has left shared memory when all of these are there, and only then may the copy engine have the stage
                    use16(h);
                    use16(h + 16);
                }
                __syncwarp();
                bar_arrive_if(bar(bWEmpty + ws), lane == 0 && !wait.lost);
                if (work) {
                    const uint32_t to = lane_base + ar.at * 32u;
                    wait(bar(bEmpty + ar.at), ar.lap ^ 1u);
                    fence_after();
                    __syncwarp();
                    if constexpr (!GRAD) {
                        tmem_st32(to, h);
                    } else {
                        tmem_st_16x128b(to, h);
                        tmem_st_16x128b(to + (16u << 16), h + 16);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    fence_before();
                    __syncwarp();
                    arrive_cluster_if(full0 + 8u * ar.at, lane == 0 && !wait.lost);
                    ar.at += kSets;
                    if (ar.at >= a.ns) { ar.at -= a.ns; ar.lap ^= 1u; }
                    turn += kSets;
                }
                turn -= have;
            }
        }
    } else if (warp == kWProducts) {
        // ---- products of both CTAs' rows, by the first one
        if (rank == 0) {
            const uint32_t idesc = (1u << 4) | ((a.T >> 3) << 17) | ((2u * kRows >> 4) << 24);
            const uint64_t desc0 = sw128_desc(base + a.at_x);
            Ring ar, dr;
            bool ready = false;
            for (uint64_t at = head, left = run1 - run0; left; dr.next(a.nd)) {
                const Part s = part_at(at);
                go_on(at, left, s);
                const uint32_t d = tmem + dr.at * a.T;
                wait(bar(bOutEmpty + dr.at), dr.lap ^ 1u);
                fence_after();
                for (uint32_t i = 0; i < s.blocks; i++) {
                    if (!ready) wait(bar(bFull + ar.at), ar.lap);
                    fence_after();
                    Ring nr = ar;
                    nr.next(a.ns);
                    const bool there = bar_test(bar(bFull + nr.at), nr.lap);         // asked for while this block's products are being issued
                    // (past the last column of a forward product the codes are the copy's zeros, times a scale, and the activations zeros)
                    if (!wait.lost) mma_block(d, tmem + a_base + ar.at * 32u, desc0 + ((ar.at * xstage) >> 4), idesc, i, bar(bEmpty + ar.at));
                    ready = for_the_warp(there);
                    ar = nr;
                }
                if (!wait.lost) commit_pair(bar(bOutFull + dr.at));       // else the way out's waits run out too, in both CTAs
            }
        }
    } else if (warp == kWCodes) {
        // ---- weight copies: a resident weight depends on nothing that came before in the stream
        const bool leader = elect();
        Ring wr;
        uint32_t used = 0;
        for (uint64_t at = head, left = run1 - run0; left;) {
            const Part s = part_at(at);
            go_on(at, left, s);
            for (uint32_t p = s.p0; p < s.p1; p++, wr.next(a.nw)) {
                wait(bar(bWEmpty + wr.at), wr.lap ^ 1u);
                if (leader && !wait.lost) {
                    used++;
                    const uint32_t to = base + wr.at * P::kStage, full = bar(bWFull + wr.at);
                    bar_expect(full, P::kStage);
                    if constexpr (GRAD) {
                        const uint32_t which = p >= a.per_weight, x = first_row(s.tile) / kWide * P::kBytes, y = (p - (which ? a.per_weight : 0u)) * P::kAlong;
                        if (which) tma_2d(to, &umap, x, y, full);
                        else tma_2d(to, &gmap, x, y, full);
                    } else {
                        tma_2d(to, &gmap, p * P::kBytes, first_row(s.tile), full);
                        tma_2d(to + P::kStage / 2u, &umap, p * P::kBytes, first_row(s.tile), full);
                    }
                }
                __syncwarp();
            }
        }
        if (leader) *word(bUsedW) = used;
    } else if (warp == kWTokens) {
        // ---- activation copies: this CTA's half of a block's tokens; the first CTA's barrier counts both halves' bytes
        const bool leader = elect();
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (leader) word(bMark)[1] = 1u;
        const uint32_t full0 = in_cta(bar(bFull), 0u);
        Ring xr;
        for (uint64_t at = head, left = run1 - run0; left;) {
            const Part s = part_at(at);
            go_on(at, left, s);
            const uint32_t token = first_token(s.tile) + rank * (a.T / 2u);
            for (uint32_t i = 0; i < s.blocks; i++, xr.next(a.ns)) {
                wait(bar(bEmpty + xr.at), xr.lap ^ 1u);
                if (leader && !wait.lost) {
                    if (rank == 0) bar_expect(bar(bFull + xr.at), 2u * xstage);
                    uint32_t along = (s.p0 * P::kBlocks + i) * 64u, y = token;
                    if (GRAD && along >= a.per_weight * P::kAlong) { along -= a.per_weight * P::kAlong; y += a.M; }
                    tma_2d_pair(base + a.at_x + xr.at * xstage, &xmap, along, y, full0 + 8u * xr.at);
                }
                __syncwarp();
            }
        }
    } else if (warp == kWScales) {
        // ---- scales of a piece, [group][row], a piece ahead of the stage they wait for.  Gradient: zero past the last weight row, so that what lies behind it (there the activations are zeros) cannot be an infinity.
        constexpr uint32_t kGroups = GRAD ? 4u : 8u;
        constexpr uint32_t kEach = (GRAD ? P::kAlong : kRows) / 32u;              // rows a lane
        struct Fetched { uint16_t v[kEach][kGroups]; uint32_t ng; };
        struct { uint64_t at, left; uint32_t p, p1, row0; } c = {head, run1 - run0, 0u, 0u, 0u};       // what is to be fetched next
        auto fetch = [&](Fetched &f) {
            f.ng = 0u;
            if (c.p == c.p1) {
                if (!c.left) return;
                const Part s = part_at(c.at);
                go_on(c.at, c.left, s);
                c.p = s.p0; c.p1 = s.p1;
                c.row0 = first_row(s.tile);
            }
            const uint32_t p = c.p++;
            if constexpr (GRAD) {
                const uint32_t which = p >= a.per_weight, n0 = (p - (which ? a.per_weight : 0u)) * P::kAlong, g_first = group_of(min(c.row0, a.K - 1u));
                const uint16_t *from = (which ? a.scales[1] : a.scales[0]) + g_first;
                const uint32_t ng = group_of(min(c.row0 + 127u, a.K - 1u)) - g_first + 1u;
#pragma unroll
                for (uint32_t j = 0; j < kEach; j++) {
                    const uint32_t n = n0 + j * 32u + lane;
#pragma unroll
                    for (uint32_t g = 0; g < kGroups; g++) f.v[j][g] = g < ng && n < a.N ? __ldg(from + (size_t)n * a.groups + g) : (uint16_t)0;
                }
                f.ng = kGroups;
            } else {
                const uint32_t g0 = group_of(p * P::kAlong);
                f.ng = group_of(min((p + 1u) * P::kAlong, a.K) - 1u) - g0 + 1u;
#pragma unroll
                for (uint32_t j = 0; j < kEach; j++) {
                    const uint16_t *from = a.scales[j >> 1] + (size_t)min(c.row0 + lane + 32u * (j & 1u), a.N - 1u) * a.groups + g0;
#pragma unroll
                    for (uint32_t g = 0; g < kGroups; g++) if (g < f.ng) f.v[j][g] = __ldg(from + g);
                }
            }
        };
        Fetched f;
        fetch(f);
        for (Ring wr; f.ng; wr.next(a.nw)) {
            wait(bar(bWEmpty + wr.at), wr.lap ^ 1u);
#pragma unroll
            for (uint32_t j = 0; j < kEach; j++)
#pragma unroll
                for (uint32_t g = 0; g < kGroups; g++)
                    if (g < f.ng) asm volatile("st.shared.u16 [%0], %1;" ::"r"(scales_at + wr.at * kScales + g * (kEach * 64u) + j * 64u + lane * 2u), "h"(f.v[j][g]) : "memory");
            __syncwarp();
            bar_arrive_if(bar(bWFull + wr.at), lane == 0 && !wait.lost);
            fetch(f);
        }
    } else {
        // ---- the way out.  A lane keeps its row: of 32 tokens at a time, a warp of the gate's rows hands the later sixteen to the warp that has the same
        // features' up rows, and gets the earlier sixteen's, so that both make h of sixteen tokens, all in flight together.
        const uint32_t q = warp & 3u, tid = threadIdx.x - kWOut * 32u, row = place<GRAD, BITS>(q, lane), empty0 = in_cta(bar(bOutEmpty), 0u);
        const bool gate = q < 2u;                                // (forward)
        const uint32_t exchange = base + a.at_out, maxima = exchange + 8u * 2048u;
        asm volatile("griddepcontrol.wait;" ::: "memory");       // outputs, scratch and counters are the kernels' before this one until here
        // sixteen tokens' values of this lane's column, `stride` apart, the first `count` of them
        auto put = [&](void *to, size_t at, uint32_t stride, uint32_t count, const float (&v)[16]) {
            uint16_t *p = reinterpret_cast<uint16_t *>(to) + at, o[16];
            if (a.dtype == EOQ_B200_F16) {
#pragma unroll
                for (uint32_t j = 0; j < 16; j++) o[j] = __half_as_ushort(__float2half_rn(v[j]));
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 16; j++) o[j] = __bfloat16_as_ushort(__float2bfloat16_rn(v[j]));
            }
            if (count >= 16u) {
#pragma unroll
                for (uint32_t j = 0; j < 16; j++, p += stride) *p = o[j];
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 16; j++, p += stride) if (j < count) *p = o[j];
            }
        };
        uint32_t turn = 0;                                       // buffers of the exchange alternate
        float spoilt = 0.0f;                                     // NaN once a sum of this tile is not finite
        auto look_at = [&](const float (&v)[16]) {
            uint64_t s = pack2(v[0], v[1]);
#pragma unroll
            for (int j = 2; j < 16; j += 2) s = add2(s, pack2(v[j], v[j + 1]));
            spoilt = fmaf(low2(s) + high2(s), 0.0f, spoilt);
        };
        // a tile, its rows' sums of sixteen tokens from `take`; `behind` is called when the last have been taken
        auto finish = [&](uint32_t tile, auto &&take, auto &&behind) {
            const uint32_t row0 = first_row(tile), tok0 = first_token(tile), tokens = min(a.T, a.M - tok0);
            if constexpr (GRAD) {
                const uint32_t k = row0 + row;
                for (uint32_t t0 = 0; t0 < a.T; t0 += 16u) {
                    float v[16];
                    take(t0, v);
                    if (t0 + 16u >= a.T) behind();
                    if (t0 >= tokens || k >= a.K) continue;
                    look_at(v);
                    if (a.factor) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++) v[j] *= __ldg(a.factor + min(tok0 + t0 + j, a.M - 1u));
                    }
                    put(a.y, (size_t)(tok0 + t0) * a.K + k, a.K, tokens - t0, v);
                }
            } else {
                const uint32_t n = row0 + (q & 1u) * 32u + lane;
                const bool there = n < a.N;
                const float bg = there ? bias_at(a.bias[0], n, a.bias_dtype) : 0.0f, bu = there ? bias_at(a.bias[1], n, a.bias_dtype) : 0.0f;
                for (uint32_t t0 = 0; t0 < a.T; t0 += 32u, turn ^= 1u) {
                    float g[16], u[16];
                    const bool two = t0 + 16u < a.T;             // else the later sixteen do not exist
                    const uint32_t mine = exchange + (turn * 4u + q) * 2048u + lane * 4u, other = exchange + (turn * 4u + (q ^ 2u)) * 2048u + lane * 4u;
                    take(gate ? t0 + 16u : t0, g);               // what is handed over, first
                    if (!gate || two) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++) asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + j * 128u), "f"(g[j]) : "memory");
                    }
                    take(gate ? t0 : t0 + 16u, g);
                    if (t0 + 32u >= a.T) behind();
                    asm volatile("bar.sync %0, 64;" ::"r"(1u + (q & 1u)) : "memory");
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(u[j]) : "r"(other + j * 128u));
                    const uint32_t t = gate ? t0 : t0 + 16u;
                    const bool work = gate || two;
                    if (!gate) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++) { const float v = g[j]; g[j] = u[j]; u[j] = v; }
                    }
                    if (a.factor) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++) {
                            const float f = __ldg(a.factor + min(tok0 + t + j, a.M - 1u));
                            g[j] *= f;
                            u[j] *= f;
                        }
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++) { g[j] += bg; u[j] += bu; }
                    if (work && there && t < tokens) {
                        const size_t at = (size_t)(tok0 + t) * a.N + n;
                        float h[16];
                        if (a.act == kActSilu) {
#pragma unroll
                            for (uint32_t j = 0; j < 16; j++) h[j] = activation(g[j], kActSilu) * u[j];
                        } else {
#pragma unroll
                            for (uint32_t j = 0; j < 16; j++) h[j] = activation(g[j], a.act) * u[j];
                        }
                        look_at(h);                              // (not finite where g or u is not)
                        put(a.y, at, a.N, tokens - t, h);
                        if (a.keep.form == kKeepFull) {
                            put(a.keep.v[0], at, a.N, tokens - t, g);
                            put(a.keep.v[1], at, a.N, tokens - t, u);
                        }
                    }
                    if (a.keep.form == kKeep8bit) {
                        // the tile's 64 features of a token are one block of the 8-bit form: this warp's 32, and its neighbour's
                        const uint32_t to = maxima + (turn * 4u + q) * 128u, from = maxima + (turn * 4u + (q ^ 1u)) * 128u;
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++) {
                            const uint32_t mg = __reduce_max_sync(0xffffffffu, there ? __float_as_uint(g[j]) & 0x7fffffffu : 0u);
                            const uint32_t mu = __reduce_max_sync(0xffffffffu, there ? __float_as_uint(u[j]) & 0x7fffffffu : 0u);
                            if (lane == 0) asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + j * 8u), "r"(mg), "r"(mu) : "memory");
                        }
                        asm volatile("bar.sync %0, 64;" ::"r"(3u + (q >> 1)) : "memory");
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++) {
                            uint32_t mg, mu, eg, eu;
                            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(mg), "=r"(mu) : "r"(to + j * 8u) : "memory");
                            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(eg), "=r"(eu) : "r"(from + j * 8u) : "memory");
                            if (!work || t + j >= tokens) continue;
                            const Storer sg(max(mg, eg)), su(max(mu, eu));
                            const size_t m = tok0 + t + j, at = m * a.N + n, block = m * ((a.N + kStoreBlock - 1) / kStoreBlock) + row0 / 64u;
                            if (there) {
                                reinterpret_cast<int8_t *>(a.keep.v[0])[at] = (int8_t)sg.code(g[j]);
                                reinterpret_cast<int8_t *>(a.keep.v[1])[at] = (int8_t)su.code(u[j]);
                            }
                            if ((q & 1u) == 0 && lane == 0 && there) { a.keep.scale[0][block] = sg.scale; a.keep.scale[1][block] = su.scale; }
                        }
                    }
                }
            }
        };
        auto any_of_all = [&](bool yes) {                        // of the four warps
            uint32_t r;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 5, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((uint32_t)yes) : "memory");
            return r != 0;
        };
        // a tile with sums that are not finite, and weights that may be why
        auto made_good = [&](uint32_t tile) {
            const bool yes = any_of_all(spoilt != 0.0f && !wait.lost);
            spoilt = 0.0f;
            const uint32_t first = first_row(tile), which = GRAD ? 0u : q >> 1, n = GRAD ? min(first + row, a.K - 1u) : min(first + (q & 1u) * 32u + lane, a.N - 1u);
            if (!yes) return;
            const bool mine = GRAD ? beyond_fp16<BITS>(a, 0u, a.per_tile / a.per_weight, tid, a.N, 128u, min(first, a.K - 1u) / a.group, min(first + 127u, a.K - 1u) / a.group + 1u)
                                   : beyond_fp16<BITS>(a, which, which + 1u, n, n + 1u, 1u, 0u, a.groups);
            if (!any_of_all(mine)) return;
            finish(tile, [&](uint32_t t, float (&v)[16]) {
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = 0.0f;
                if (t < a.T) sums_in_fp32<GRAD, BITS>(a, which, n, first_token(tile) + t, v);
            }, [] {});
            spoilt = 0.0f;
        };
        auto partial_of = [&](uint32_t p, uint32_t begins) { return a.partial + ((size_t)(p * 2u + begins) * 2u + rank) * a.T * kRows + q * 32u + lane; };
        Ring dr;
        for (uint64_t at = head, left = run1 - run0; left; dr.next(a.nd)) {
            const Part s = part_at(at);
            go_on(at, left, s);
            wait(bar(bOutFull + dr.at), dr.lap);
            __syncwarp();
            fence_after();
            const uint32_t from = tmem + ((q * 32u) << 16) + dr.at * a.T;
            auto take = [&](uint32_t t, float (&v)[16]) {
                uint32_t r[16] = {};
                if (t < a.T) { tmem_ld16(from + t, r); tmem_ld_wait(r); }
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = wait.lost ? __uint_as_float(0x7fffffffu) : __uint_as_float(r[j]);
            };
            auto release = [&]() {                               // the next tile may have the accumulator
                fence_before();
                __syncwarp();
                arrive_cluster_if(empty0 + 8u * dr.at, lane == 0 && !wait.lost);
            };
            if (s.p1 - s.p0 == a.per_tile) {
                finish(s.tile, take, release);
                made_good(s.tile);
                continue;
            }
            // the tile's other parts are other pairs': the last to arrive adds them up, in the order of the pairs, its own (the same bits)
            // from the accumulator where the others' are there already
            const uint64_t first = (uint64_t)s.tile * a.per_tile, total = (uint64_t)a.tiles * a.per_tile;
            const uint32_t p_first = (uint32_t)(((first + 1) * pairs - 1) / total), p_last = (uint32_t)(((first + a.per_tile) * pairs - 1) / total);
            uint32_t *count = a.count + s.tile * 2u + rank;
            auto ask = [&](uint32_t add) {                       // parts that have arrived before this one
                asm volatile("bar.sync 5, 128;" ::: "memory");
                if (tid == 0) *word(bTicket) = add ? atomicAdd(count, 1u) : *reinterpret_cast<volatile uint32_t *>(count);
                asm volatile("bar.sync 5, 128;" ::: "memory");
                return *word(bTicket) == p_last - p_first;
            };
            const bool here = pairs <= a.tiles && ask(0u);       // (parts that all run at the same time end so, too)
            if (!here) {
                float *mine = partial_of(pair, s.p0 == 0u);
                for (uint32_t t0 = 0; t0 < a.T; t0 += 16u) {
                    float v[16];
                    take(t0, v);
                    if (t0 + 16u >= a.T) release();
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++) __stcg(mine + (size_t)(t0 + j) * kRows, v[j]);
                }
                __threadfence();
                if (!ask(1u)) continue;
            }
            __threadfence();
            finish(s.tile, [&](uint32_t t, float (&v)[16]) {
                float o[16];
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = 0.0f;
                if (t >= a.T) return;
                for (uint32_t p = p_first; p <= p_last; p++) {
                    if (here && p == pair) {
                        take(t, o);
                    } else {
                        const float *part = partial_of(p, run_start(p) <= first) + (size_t)t * kRows;
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = __ldcg(part + j * kRows);
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] += o[j];
                }
            }, [&]() { if (here) release(); });
            made_good(s.tile);
        }
    }
    __syncwarp();
    __syncthreads();
    cg::cluster_group cluster = cg::this_cluster();
    if (wait.stopped()) {
        // nothing may be under way any more when tensor and shared memory are given back.  (Activations: their barrier also counts
        // arrivals that may not come, so what is left of them gets the time of a lost copy.)
        if (warp == kWProducts && rank == 0) { commit_pair(bar(bDrain)); drain(bar(bDrain), 1u, 1u); }
        if (warp == kWCodes) drain(bar(bWFull), *word(bUsedW), a.nw);
        if (warp == kWTokens) { const long long t0 = clock64(); while (clock64() - t0 < 20000000ll) {} }
    }
    __syncthreads();
    cluster.sync();                            // the other CTA's arrivals and products are behind
    if (warp == kWProducts) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem) : "memory");
    }
}

std::atomic<long long> g_limit{4000000000ll};      // about two seconds

struct Layout { uint32_t nw, ns, nd, at_x, at_out, at_bar; size_t smem; };

// Two accumulators where they leave as many stages of operands as there are producer sets: these wait for a stage's last use by its parity, which is
// right while the use before that is behind, and the set's own last block is `kSets` back.
Layout lay_out(uint32_t T, uint32_t stage_w)
{
    const uint32_t fixed = 1024 + 8 * bEnd + 8, room = 226u * 1024u - fixed - kOut, xstage = T * 64u;
    Layout l = {};
    l.nd = 2u * T + kSets * 32u <= kTmem ? 2u : 1u;
    l.ns = std::min(8u, (kTmem - l.nd * T) / 32u);
    l.nw = std::min(8u, (room - l.ns * xstage) / (stage_w + kScales));
    l.at_x = l.nw * stage_w;
    l.at_out = l.at_x + l.ns * xstage;
    l.at_bar = l.at_out + kOut;
    l.smem = l.at_bar + 8 * bEnd + 8 + (size_t)l.nw * kScales + 1024;
    return l;
}

struct Plan { uint32_t T, tok_tiles, tiles, per_tile, per_weight, pairs, unit; };       // runs are whole numbers of `unit` pieces: 1, or a tile's

// Tokens of a tile, and pairs of CTAs.  In clocks, as measured: a block of 64 takes its products (two a token) or what the products' warp and the
// producers take at least (some 430; gate and up of 8 bits, 600), whichever is longer; with one accumulator a tile's way out (70 a token) comes on top, else only the last one's.
// Sums of shared tiles go through scratch: where pairs outnumber tiles 60 a token and part (11008 x 4096 gradient, us, tiles of 48, 112, 208 and 256
// tokens in one part: 38.9, 41.7, 48.4, 58.4; in two: 26.1, 33.1, 47.5, 56.8; in four: 23.6, 35.4, 54.8, 65.5), and as much again where a run holds parts of
// two tiles (16 tiles by 74 pairs: 26.8, 43.6, 71.3, 85.8); else 100 a token at the end, which runs of whole tiles spare (4096 x 2816 8-bit gated block,
// 1024 rows, 128 tiles: 74 pairs 73.8, 64 pairs of two tiles 54.0).  More tiles of tokens unpack the codes more often, beside all this: they are taken
// where they seem to save 15 per cent.
template <bool GRAD, int BITS>
Plan plan_for(uint32_t N, uint32_t K, uint32_t M, int nw)
{
    using P = Piece<GRAD, BITS>;
    Plan best = {};
    best.per_weight = GRAD ? (N + P::kAlong - 1) / P::kAlong : 0u;
    best.per_tile = GRAD ? best.per_weight * nw : (K + P::kAlong - 1) / P::kAlong;
    const uint32_t room = (uint32_t)std::max(1, device_sm_count() / 2), across = (GRAD ? K + 255u : N + 127u) / (GRAD ? 256u : 128u);
    double least = 1e30, fewer = 1e30;           // of the plans so far, and of those with fewer tokens' tiles than this one's
    uint32_t last = 0;
    for (uint32_t n = (M + 255u) / 256u; n < (M + 255u) / 256u * 2u + 3u; n++) {
        Plan p = best;
        p.T = ((M + n - 1) / n + 15u) / 16u * 16u;
        if (p.T == last) continue;
        last = p.T;
        fewer = least;
        p.tok_tiles = (M + p.T - 1) / p.T;
        p.tiles = across * p.tok_tiles;
        const double block = std::max(!GRAD && BITS == 8 ? 600.0 : 430.0, 2.0 * p.T), out = 70.0 * p.T, each = p.T > 160u ? out : 0.0;
        auto consider = [&](uint32_t pairs, uint32_t unit, double cost) {
            if (cost >= least || cost >= 0.85 * fewer) return;
            least = cost;
            best = p;
            best.pairs = pairs;
            best.unit = unit;
        };
        if (p.tiles >= room) {
            const uint32_t rounds = (p.tiles + room - 1) / room;
            consider((p.tiles + rounds - 1) / rounds, p.per_tile, rounds * (p.per_tile * P::kBlocks * block + each) - each + out);
            if (p.tiles % room) consider(room, 1u, (double)p.tiles / room * (p.per_tile * P::kBlocks * block + each) + out + 100.0 * p.T);
            continue;
        }
        for (uint32_t pairs = p.tiles; pairs <= room && pairs <= (uint64_t)p.tiles * p.per_tile; pairs++) {
            const double pieces = std::ceil((double)p.tiles * p.per_tile / pairs), parts = std::ceil((double)pairs / p.tiles);
            consider(pairs, pairs > p.tiles ? 1u : p.per_tile, pieces * P::kBlocks * block + out + (pairs > p.tiles ? 60.0 * p.T * (1.0 + parts + (pairs % p.tiles != 0)) : 0.0));
        }
    }
    return best;
}

template <bool GRAD>
Plan plan_of(uint32_t N, uint32_t K, uint32_t bits, uint32_t M, int nw)
{
    return bits == 4 ? plan_for<GRAD, 4>(N, K, M, nw) : bits == 2 ? plan_for<GRAD, 2>(N, K, M, nw) : plan_for<GRAD, 8>(N, K, M, nw);
}

size_t count_bytes(const Plan &p) { return ((size_t)p.tiles * 8 + 255) & ~(size_t)255; }
size_t scratch_bytes(const Plan &p) { return count_bytes(p) + (size_t)p.pairs * 4 * p.T * kRows * 4; }

template <bool GRAD, int BITS>
int run(ProductArgs a, const PackedPair &w, int nw, const void *x, uint32_t pitch, void *scratch, cudaStream_t st)
{
    using P = Piece<GRAD, BITS>;
    auto kern = gated_product_kernel<GRAD, BITS>;
    const Plan p = plan_for<GRAD, BITS>(w.N, w.K, a.M, nw);
    const Layout l = lay_out(p.T, P::kStage);
    const uint32_t at_once = resident_ctas(reinterpret_cast<const void *>(kern), kThreads, l.smem, 2) / 2u;
    if (!at_once) return (int)cudaErrorNotSupported;
    a.T = p.T; a.tok_tiles = p.tok_tiles; a.tiles = p.tiles; a.per_tile = p.per_tile; a.per_weight = p.per_weight; a.unit = p.unit;
    a.nw = l.nw; a.ns = l.ns; a.nd = l.nd; a.at_x = l.at_x; a.at_out = l.at_out; a.at_bar = l.at_bar;
    a.count = static_cast<uint32_t *>(scratch);
    a.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + count_bytes(p));
    a.x = static_cast<const uint16_t *>(x);
    a.pitch = pitch;
    CUtensorMap maps[2], xmap;
    constexpr CUtensorMapSwizzle sw = P::kBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : P::kBytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    for (int i = 0; i < 2; i++)
        if (!map_2d(maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes[i], w.row_bytes, w.N, w.row_bytes, P::kBytes, GRAD ? P::kAlong : kRows / 2, sw)) return (int)cudaErrorNotSupported;
    if (!map_2d(xmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, x, GRAD ? w.N : w.K, (uint64_t)a.M * (GRAD ? nw : 1), (uint64_t)pitch * 2, 64, p.T / 2u, CU_TENSOR_MAP_SWIZZLE_128B))
        return (int)cudaErrorNotSupported;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2u * std::min(p.pairs, at_once));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = l.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launches();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, maps[0], maps[1], xmap);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

ProductArgs common(const PackedPair &w, const float *factor, uint32_t M, void *y, int dtype)
{
    ProductArgs a = {};
    for (int i = 0; i < 2; i++) { a.scales[i] = w.scales[i]; a.codes[i] = w.codes[i]; }
    a.row_bytes = w.row_bytes;
    a.factor = factor; a.y = y; a.N = w.N; a.K = w.K; a.M = M; a.group = w.group; a.groups = w.K / w.group; a.dtype = dtype;
    a.inverse = (uint32_t)(((1ull << 32) + w.group / 16u - 1) / (w.group / 16u));
    a.limit = g_limit.load(std::memory_order_relaxed);
    return a;
}

}  // namespace

bool product_takes(const PackedPair &w, int nw)
{
    for (int i = 0; i < nw; i++)
        if (!qmm_takes(w.K, w.bits, w.group, w.codes[i], w.codes[i])) return false;
    return w.K < 1u << 20;                     // (group_of: K / 16 times group / 16 is below 2^32)
}

Scratch gated_product_scratch(const PackedPair &w, uint32_t M)
{
    const Plan p = plan_of<false>(w.N, w.K, w.bits, M, 1);
    return Scratch{scratch_bytes(p), p.tiles * 2u};
}
Scratch input_grad_product_scratch(const PackedPair &w, int nw, uint32_t M)
{
    const Plan p = plan_of<true>(w.N, w.K, w.bits, M, nw);
    return Scratch{scratch_bytes(p), p.tiles * 2u};
}

int launch_gated_product(const GatedCall &c, const uint16_t *x, const float *factor, void *scratch, void *stream)
{
    ProductArgs a = common(c.w, factor, c.M, c.h, c.dtype);
    a.bias[0] = c.bias[0]; a.bias[1] = c.bias[1];
    a.keep = c.keep;
    a.act = c.act;
    a.bias_dtype = c.bias_dtype;
    cudaStream_t st = (cudaStream_t)stream;
    if (c.w.bits == 4) return run<false, 4>(a, c.w, 2, x, c.w.K, scratch, st);
    if (c.w.bits == 2) return run<false, 2>(a, c.w, 2, x, c.w.K, scratch, st);
    return run<false, 8>(a, c.w, 2, x, c.w.K, scratch, st);
}

int launch_input_grad_product(const PackedPair &w, int nw, const uint16_t *dy, uint32_t pitch, const float *factor, uint32_t M, void *dx, int dtype, void *scratch, void *stream)
{
    const ProductArgs a = common(w, factor, M, dx, dtype);
    cudaStream_t st = (cudaStream_t)stream;
    if (w.bits == 4) return run<true, 4>(a, w, nw, dy, pitch, scratch, st);
    if (w.bits == 2) return run<true, 2>(a, w, nw, dy, pitch, scratch, st);
    return run<true, 8>(a, w, nw, dy, pitch, scratch, st);
}

void set_gated_wait_us(int v) { g_limit.store(std::min(std::max(v, 0), 60000000) * 2000ll); }

long long gated_wait_limit() { return g_limit.load(std::memory_order_relaxed); }

uint32_t *gated_status_word()
{
    static std::atomic<uint32_t *> known[16];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
    uint32_t *p = dev < 16 ? known[dev].load() : nullptr;
    if (!p) {
        if (cudaGetSymbolAddress(reinterpret_cast<void **>(&p), g_gated_status) != cudaSuccess) return nullptr;
        if (dev < 16) known[dev].store(p);
    }
    return p;
}

uint32_t gated_status()
{
    uint32_t v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_gated_status, 4) != cudaSuccess) return ~0u;
    if (v && cudaMemcpyToSymbol(g_gated_status, &zero, 4) != cudaSuccess) return ~0u;
    return v;
}

}  // namespace eoq
