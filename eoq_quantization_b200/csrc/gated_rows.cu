// The gated block for a few rows of 16-bit activations, one pass over both weights' codes: up to eight rows here, up to 32 in the
// second kernel below.
//
// Warp-level products, D[16 x 8] += A[16 x 16] B[16 x 8] (mma.sync m16n8k16), the codes exact and the scales applied to the sums in
// fp32, with gate rows and up rows of the same features in one instruction: lane (g, t) takes gate row g as A's row g and up row g as
// A's row g + 8, so that the sums of both, for the same feature and rows of x, end in the same lane.  The contraction index is a
// dummy: a lane feeds its codes in the order in which they leave their words cheapest (packed_mma.h), and the activations, brought
// to shared memory in that order once per CTA, follow.
//
// A CTA takes a run of neighbouring eights of features ("tiles"), and its warps equal runs of the tiles' chunks, 128 bytes of all
// sixteen rows, whichever tile these belong to; a warp leaves its sums of a tile in shared memory where it goes on to the next one,
// and what the warps left is added up in their order.  Each warp has a ring of chunks of its own, which TMA fills some chunks ahead:
// what has to be under way to keep HBM busy (50 KB an SM) would not fit the registers.
//   Measured (4 bits, groups of 128, fp16, back to back, codes from HBM; in brackets what both weights' bytes take at 6470 GB/s): 11008 x 4096
// one row 13.1 us (7.2), eight 15.0; 28672 x 8192 one row 51.0 (37.4); 704 x 512 3.0; 11008 x 4096 of 8 bits 19.1 (14.2).  What bounds it at
// length is the issue slots (70 % of active cycles) and the integer pipe (51 %) of the unpacking, with HBM at 53 %; short calls are their start.
//   Waits are bounded: a warp whose copy does not come marks the CTA, whose results become NaN, and sets the status word.
#include "gated.h"
#include "packed_mma.h"
#include "tensor_core.h"

#include <algorithm>
#include <type_traits>

#include "activations.cuh"

namespace eoq {
namespace {

// Scales of `ntiles` tiles from tile0 on to shared memory by whole rows, [gate, up][row][pitch]: a load of a few of each row would touch as many
// lines as one of their codes.  Eight rows a warp and step, all requested before the first is stored.
template <bool WORDS>
__device__ __forceinline__ void fetch_scales(const uint16_t *gate, const uint16_t *up, uint32_t *to, uint32_t tile0, uint32_t ntiles, uint32_t N, uint32_t groups,
                                             uint32_t pitch, uint32_t warp, uint32_t nwarps, uint32_t lane)
{
    using T = std::conditional_t<WORDS, uint32_t, uint16_t>;       // two groups at a time, or one
    const uint32_t rows = ntiles * 16u, half = ntiles * 8u, count = WORDS ? groups / 2u : groups;
    for (uint32_t j = lane; j < count; j += 32u)
        for (uint32_t r0 = warp; r0 < rows; r0 += 8u * nwarps) {
            T v[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                const uint32_t row = min(r0 + i * nwarps, rows - 1u), n = min(tile0 * 8u + (row >= half ? row - half : row), N - 1u);
                v[i] = __ldg(reinterpret_cast<const T *>((row >= half ? up : gate) + (size_t)n * groups) + j);
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) if (r0 + i * nwarps < rows) reinterpret_cast<T *>(to + (r0 + i * nwarps) * pitch)[j] = v[i];
        }
}

// The addresses of a chunk's loads come from here, behind the wait for it: the loads themselves may move among the products.
__device__ __forceinline__ void pin(uint32_t &w, uint32_t &x, uint32_t &s) { asm volatile("" : "+r"(w), "+r"(x), "+r"(s)::"memory"); }

struct RowsArgs {
    const uint16_t *scales[2];
    const void *bias[2];
    const void *x;
    void *h;
    void *kept[2];               // [batch][N] of x's type, fp32 (kept32), or null
    uint32_t N, K, group, batch, per, more;      // tiles a CTA takes, and how many CTAs take one more
    uint32_t most, pitch, slots; // tiles at a time, words that a row's scales take in shared memory, chunks of a warp's ring
    int act, kept32, bias_dtype;
    long long limit;             // clock ticks a wait may take
    uint32_t *status;            // set when one runs out
};

constexpr int most_threads(int bt) { return bt == 1 ? 1024 : 768; }        // 64 or 80 registers a thread
constexpr int kParts = 3;        // tiles that a warp's run touches at most, for up to two tiles a warp

// A unit (half of one, where that has 128 bytes) in bytes and columns: a lane takes a quarter of it.
template <int BITS, int U> struct Part { static constexpr int kBytes = U * BITS / 8 < 64 ? U * BITS / 8 : 64, kCols = kBytes * 8 / BITS; };

// x in the order of the codes: sixteen-byte pieces [span][i][row][t], piece i of lane (row, t) the columns of its registers 4 i .. 4 i + 3.
template <int BITS, int U>
__device__ __forceinline__ uint4 piece_load(const uint16_t *x, uint32_t span, uint32_t i, uint32_t t)
{
    if constexpr (BITS == 2) {       // columns 16 j + (r & 7) and + 8 of a lane's, j = i / 2
        const uint32_t j = i >> 1, c = span * 128u + (U == 128 ? t * 32u + j * 16u : j * 64u + t * 16u) + (i & 1u) * 4u;
        const uint2 a = __ldg(reinterpret_cast<const uint2 *>(x + c)), b = __ldg(reinterpret_cast<const uint2 *>(x + c + 8u));
        return make_uint4(a.x, a.y, b.x, b.y);
    } else {
        return __ldg(reinterpret_cast<const uint4 *>(x + span * 128u + (U == 128 ? t * 32u + i * 8u : U == 64 ? (i >> 1) * 64u + t * 16u + (i & 1u) * 8u : i * 32u + t * 8u)));
    }
}
template <int BITS>
__device__ __forceinline__ uint4 piece_order(const uint4 &v)
{
    if constexpr (BITS == 8) return v;
    else return make_uint4(__byte_perm(v.x, v.z, 0x5410u), __byte_perm(v.x, v.z, 0x7632u), __byte_perm(v.y, v.w, 0x5410u), __byte_perm(v.y, v.w, 0x7632u));
}

// U: columns of a unit whose scale is applied on its own.
// EXACT: units are groups, and a chunk's scales lie together; else a group is several units.
// BT: rows of x that shared memory has room for.
//   Lane (g, t) takes the tile's row whose number is g's three bits reversed: with the copies' 128-byte swizzle the rows that a load's
// phase covers then lie in different banks, for loads of 16, 8 and 4 bytes.
//   What it takes 128 columns (2048 codes a warp): at four bits 72 instructions for the codes, 8 products, 6 loads of codes and activations.
template <int BITS, bool BF16, int U, bool EXACT, int BT>
__global__ void __launch_bounds__(most_threads(BT), 1) gated_rows_kernel(const RowsArgs a, const __grid_constant__ CUtensorMap gmap, const __grid_constant__ CUtensorMap umap)
{
    static_assert(BITS != 2 || U >= 64, "a unit of 32 two-bit codes is no whole word of a lane");
    using P = Part<BITS, U>;
    constexpr int CH = 8 / BITS;                                   // spans of 128 columns a chunk has
    constexpr int kUnits = 128 / U, kParts128 = 128 / P::kBytes, kWords = P::kBytes / 16;      // units of a span, parts of a chunk, words of a lane's share of a part
    constexpr int kScales = (CH * kUnits + 1) / 2;                 // words of a chunk's scales (EXACT)
    constexpr uint32_t kHalf = 1024u, kSlot = 2048u;               // a chunk's codes of one weight, of both
    extern __shared__ uint8_t raw[];
    const uint32_t lane = threadIdx.x & 31u, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), nwarps = blockDim.x >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t sgroups = a.K / a.group, chunks = a.K / (128u * CH), gunits = a.group / U, myrow = (g & 1u) << 2 | (g & 2u) | g >> 2;
    constexpr uint32_t kPieces = 16u * BT * CH;                    // of a chunk of x
    // shared memory: rings, activations, scales [gate, up][row of the tiles][pitch], sums, barriers and the mark
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    uint4 *xs = reinterpret_cast<uint4 *>(smem + (size_t)nwarps * a.slots * kSlot);
    uint32_t *scales = reinterpret_cast<uint32_t *>(xs + (size_t)chunks * kPieces);
    float (*red)[kParts][16][BT] = reinterpret_cast<float (*)[kParts][16][BT]>(scales + (size_t)a.most * 16u * a.pitch);
    const uint32_t ring = saddr(smem) + warp * a.slots * kSlot, bars = saddr(red + nwarps) + warp * a.slots * 8u, mark = saddr(red + nwarps) + nwarps * a.slots * 8u;
    uint32_t tile0 = blockIdx.x * a.per + min(blockIdx.x, a.more), ntiles;
    const uint32_t last = tile0 + a.per + (blockIdx.x < a.more);

    // a warp's run of chunks of the tiles at hand; copies are requested `slots` chunks ahead
    uint32_t next, end, to_load = 0, load_tile, load_chunk;
    bool gave_up = false;
    auto begin = [&]() {
        ntiles = min(last - tile0, a.most);
        const uint32_t n = ntiles * chunks;
        next = to_load = n * warp / nwarps;
        end = n * (warp + 1) / nwarps;
        load_tile = next / chunks;
        load_chunk = next - load_tile * chunks;
    };
    auto load = [&](uint32_t slot) {
        if (to_load >= end || gave_up) return;
        to_load++;
        if (lane == 0) {
            const uint32_t bar = bars + slot * 8u, to = ring + slot * kSlot, row = (tile0 + load_tile) * 8u, at = load_chunk * 128u;
            bar_expect(bar, kSlot);
            tma_2d(to, &gmap, at, row, bar);
            tma_2d(to + kHalf, &umap, at, row, bar);
        }
        if (++load_chunk == chunks) { load_chunk = 0; load_tile++; }
    };
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (for_the_warp(bar_test(bar, parity))) return;
        const long long t0 = clock64();
        bool late = a.limit == 0;                  // no patience at all: what is not there has run out
        while (!late && !bar_try(bar, parity)) late = clock64() - t0 > a.limit;
        gave_up = __any_sync(0xffffffffu, late);
        if (gave_up && lane == 0) {
            asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(mark), "r"(1u) : "memory");
            *reinterpret_cast<volatile uint32_t *>(a.status) = 1u;
        }
    };
    auto fetch = [&]() { fetch_scales<EXACT && (CH * kUnits > 1)>(a.scales[0], a.scales[1], scales, tile0, ntiles, a.N, sgroups, a.pitch, warp, nwarps, lane); };

    // codes and scales do not depend on the kernel before this one in the stream, the activations may
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane == 0) for (uint32_t i = 0; i < a.slots; i++) bar_init(bars + i * 8u, 1);
    if (threadIdx.x == 0) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(mark), "r"(0u) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    begin();
    for (uint32_t i = 0; i < a.slots; i++) load(i);
    fetch();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t e = threadIdx.x; e < chunks * kPieces; e += blockDim.x) {
        const uint32_t tt = e & 3u, b = (e >> 2) % BT, i = (e >> 2) / BT & 3u, s = e / (16u * BT);
        if (b < a.batch) xs[e] = piece_order<BITS>(piece_load<BITS, P::kCols>(reinterpret_cast<const uint16_t *>(a.x) + (size_t)b * a.K, s, i, tt));
    }
    __syncthreads();

    // (columns of the products behind the last row of x are left: what lanes of such rows read is any other row)
    const uint32_t x0 = (uint32_t)__cvta_generic_to_shared(xs) + (min(g, a.batch - 1u) * 4u + t) * 16u;
    const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(scales) + myrow * a.pitch * 4u;
    const uint32_t w0 = ring + myrow * 128u + ((((t * (P::kBytes / 4)) >> 4) ^ myrow) << 4) + ((t * (P::kBytes / 4)) & 15u);
    float tot[4];
    // w, x, s: shared addresses of the lane's share of the chunk's codes, of the activations, and of the gate row's scales
    auto multiply = [&](uint32_t w, uint32_t x, uint32_t s, uint32_t chunk) {
        pin(w, x, s);
        uint32_t code[2][8];
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int p = 0; p < kParts128; p++) {
                const uint32_t at = (w ^ (p * P::kBytes)) + r * kHalf;
                uint32_t *d = &code[r][p * kWords];
                if constexpr (kWords == 1) asm("ld.shared.b32 %0, [%1];" : "=r"(d[0]) : "r"(at));
                else if constexpr (kWords == 2) asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "r"(at));
                else asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(at));
            }
        uint32_t sc[2][kScales] = {};
        if constexpr (EXACT) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const uint32_t at = s + r * ntiles * 32u * a.pitch;
                if constexpr (CH * kUnits == 1) asm("ld.shared.u16 %0, [%1];" : "=r"(sc[r][0]) : "r"(at));
                else if constexpr (kScales == 1) asm("ld.shared.b32 %0, [%1];" : "=r"(sc[r][0]) : "r"(at));
                else if constexpr (kScales == 2) asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(sc[r][0]), "=r"(sc[r][1]) : "r"(at));
                else asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(sc[r][0]), "=r"(sc[r][1]), "=r"(sc[r][2]), "=r"(sc[r][3]) : "r"(at));
            }
        }
        auto scale = [&](int r, int u) {
            uint32_t v;
            if (EXACT) v = sc[r][u / 2] >> (16 * (u & 1));
            else asm("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(s + r * ntiles * 32u * a.pitch + (chunk * (uint32_t)(CH * kUnits) + u) / gunits * 2u));
            return __half2float(__ushort_as_half((uint16_t)v));
        };
        // four registers of codes a row and span at a time, and their piece of the activations: two products.  The accumulators of the
        // chunk's spans (of one span: two) alternate, so that consecutive products do not wait for one another.
        float c[CH == 1 ? 2 : CH][4];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int sp = 0; sp < CH; sp++) {
                uint4 q;
                asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(x + (sp * 4 + i) * (BT * 64)));
                uint32_t h[2][4];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    if constexpr (BITS == 4) {
                        unpack_word<BITS, BF16>(code[r][sp * 4 + i], h[r]);
                    } else if constexpr (BITS == 2) {
                        uint32_t e[8];
                        unpack_word<BITS, BF16>(code[r][sp * 2 + i / 2], e);
#pragma unroll
                        for (int j = 0; j < 4; j++) h[r][j] = e[4 * (i & 1) + j];
                    } else {
                        uint32_t e[2];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            unpack_word<BITS, BF16>(code[r][2 * i + j], e);
                            h[r][2 * j] = e[0]; h[r][2 * j + 1] = e[1];
                        }
                    }
                }
                constexpr int kOfUnit = 4 / kUnits;                    // pieces
                float (&one)[4] = c[CH == 1 ? 0 : sp], (&two)[4] = c[CH == 1 ? 1 : sp];
                if (i % kOfUnit == 0) {
                    mma_m16n8k16_first<BF16>(one, h[0][0], h[1][0], h[0][1], h[1][1], q.x, q.y);
                    if (CH > 1) mma_m16n8k16<BF16>(two, h[0][2], h[1][2], h[0][3], h[1][3], q.z, q.w);
                    else mma_m16n8k16_first<BF16>(two, h[0][2], h[1][2], h[0][3], h[1][3], q.z, q.w);
                } else {
                    mma_m16n8k16<BF16>(one, h[0][0], h[1][0], h[0][1], h[1][1], q.x, q.y);
                    mma_m16n8k16<BF16>(two, h[0][2], h[1][2], h[0][3], h[1][3], q.z, q.w);
                }
                if (i % kOfUnit == kOfUnit - 1) {
                    const int u = sp * kUnits + i / kOfUnit;
#pragma unroll
                    for (int j = 0; j < 4; j++) tot[j] = fmaf(scale(j >> 1, u), CH > 1 ? one[j] : one[j] + two[j], tot[j]);
                }
            }
    };
    Ring at_slot, lost;                            // (laps go on over the rounds of tiles)
    uint32_t owing = 0;
    for (;;) {
        const uint32_t first_tile = next / chunks;
        uint32_t chunk = next - first_tile * chunks, part = 0, x = x0 + chunk * (kPieces * 16u);
        constexpr uint32_t kStep = EXACT ? CH * kUnits * 2u : 0u;
        uint32_t sc = s0 + first_tile * 32u * a.pitch + chunk * kStep;
        tot[0] = tot[1] = tot[2] = tot[3] = 0.0f;
        auto leave = [&]() {
            if (2u * t < BT) {
                float (*to)[BT] = red[warp][part];
                to[g][2 * t] = tot[0]; to[g + 8][2 * t] = tot[2];
                if (BT > 1) { to[g][2 * t + (BT > 1)] = tot[1]; to[g + 8][2 * t + (BT > 1)] = tot[3]; }
            }
            part++;
            tot[0] = tot[1] = tot[2] = tot[3] = 0.0f;
        };
        for (; next < end; next++) {
            if (!gave_up) {
                wait(bars + at_slot.at * 8u, at_slot.lap);
                if (gave_up) { lost = at_slot; owing = to_load - next; }
            }
            multiply(w0 + at_slot.at * kSlot, x, sc, chunk);
            // every lane's codes have gone into products: the slot is free
            __syncwarp();
            load(at_slot.at);
            at_slot.next(a.slots);
            x += kPieces * 16u;
            sc += kStep;
            if (++chunk == chunks) {
                leave();
                chunk = 0;
                x = x0;
                sc += 32u * a.pitch - chunks * kStep;
            }
        }
        if (chunk) leave();
        if (owing) {                               // no copy may be under way when the CTA ends
            const long long t0 = clock64();
            for (; owing; owing--, lost.next(a.slots)) while (!bar_try(bars + lost.at * 8u, lost.lap) && clock64() - t0 < 20000000ll) {}
        }
        __syncthreads();
        uint32_t stopped;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(stopped) : "r"(mark) : "memory");
        // every (tile, row of x, feature): the parts of the warps whose runs touch the tile, in their order
        const uint32_t n = ntiles * chunks;
        for (uint32_t i = threadIdx.x; i < ntiles * 8u * BT; i += blockDim.x) {
            const uint32_t f = i & 7u, b = (i >> 3) % BT, tile = i / (8u * BT), feature = (tile0 + tile) * 8u + ((f & 1u) << 2 | (f & 2u) | f >> 2);
            if (feature >= a.N || b >= a.batch) continue;
            const uint32_t first = tile * chunks, behind = first + chunks;
            // the warp that has chunk s: the last w with n w / nwarps <= s
            uint32_t w = ((first + 1) * nwarps - 1) / n;
            float gs = 0.0f, us = 0.0f;
            for (uint32_t from = n * w / nwarps; w < nwarps && from < behind; w++) {
                const uint32_t to = n * (w + 1) / nwarps;
                if (to > from) {
                    const uint32_t part_of = tile - from / chunks;
                    gs += red[w][part_of][f][b];
                    us += red[w][part_of][8 + f][b];
                }
                from = to;
            }
            gs += bias_at(a.bias[0], feature, a.bias_dtype);
            us += bias_at(a.bias[1], feature, a.bias_dtype);
            if (stopped) gs = us = __uint_as_float(0x7fffffffu);
            const size_t at = (size_t)b * a.N + feature;
            auto put = [&](void *to, float value) {
                if (BF16) reinterpret_cast<__nv_bfloat16 *>(to)[at] = __float2bfloat16_rn(value);
                else reinterpret_cast<__half *>(to)[at] = __float2half_rn(value);
            };
            put(a.h, activation(gs, a.act) * us);
            if (!a.kept[0]) continue;
            if (a.kept32) {
                reinterpret_cast<float *>(a.kept[0])[at] = gs;
                reinterpret_cast<float *>(a.kept[1])[at] = us;
            } else {
                put(a.kept[0], gs);
                put(a.kept[1], us);
            }
        }
        tile0 += ntiles;
        if (tile0 >= last) break;
        __syncthreads();
        gave_up = stopped != 0;
        begin();
        // (the slots in the order in which the ring comes by them)
        for (uint32_t i = 0, slot = at_slot.at; i < a.slots; i++, slot = slot + 1 == a.slots ? 0 : slot + 1) load(slot);
        fetch();
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Nine to 32 rows (24 of large weights): the same products with NT eights of rows, each lane's codes unpacked once for all of them.  The activations do not fit
// shared memory beside the rings, so four warps bring them there a slice of columns at a time, into two buffers in turn, and a warp keeps
// its tile, its sums in registers, through all slices; where a CTA has fewer tiles than warps, SPLIT warps take a tile's chunks in turn, and
// what they have is added up in their order at the end.
//   What bounds it: the warp-level tensor pipe (8 clocks a product and scheduler, 8 NT products of 128 columns), then the unpacking, and
// with few warps an SM their waits for shared memory (28672 x 8192, 24 rows: 13 of 20 warps work, for a tile takes whole warps and a CTA has
// 25 tiles in two rounds of 13; tensor pipe 38 % of active cycles, slots 46 %).  11008 features are ten tiles a CTA, two warps each.
//   Measured as above: 11008 x 4096 16 rows 18.2 us, 24 rows 22.9 (7.3), 28672 x 8192 24 rows 108 to 116.
// ---------------------------------------------------------------------------
constexpr uint32_t kManyWarps = 20, kStagers = 4;

struct ManyArgs {
    const uint16_t *scales[2];
    const void *bias[2];
    const void *x;
    void *h;
    void *kept[2];
    uint32_t N, K, group, batch, per, more;      // tiles a CTA takes, and how many CTAs take one more
    uint32_t most, split, slice, pitch;          // tiles at a time, warps of a tile, chunks of a slice, words of a row's scales
    int act, kept32, bias_dtype;
    long long limit;
    uint32_t *status;
};

template <int BITS, bool BF16, int U, bool EXACT, int NT>
__global__ void __launch_bounds__((kManyWarps + kStagers) * 32, 1)
gated_many_rows_kernel(const ManyArgs a, const __grid_constant__ CUtensorMap gmap, const __grid_constant__ CUtensorMap umap)
{
    static_assert(BITS != 2 || U >= 64, "a unit of 32 two-bit codes is no whole word of a lane");
    using P = Part<BITS, U>;
    constexpr int CH = 8 / BITS;                                   // spans of 128 columns a chunk has
    constexpr int kUnits = 128 / U, kParts128 = 128 / P::kBytes, kWords = P::kBytes / 16;
    constexpr int kScales = (CH * kUnits + 1) / 2;                 // words of a chunk's scales (EXACT)
    constexpr uint32_t kHalf = 1024u, kSlot = 2048u, kSlots = 2u, kPieces = 16u * 8u * NT * CH;        // pieces of x of a chunk
    extern __shared__ uint8_t raw[];
    const uint32_t lane = threadIdx.x & 31u, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), nwarps = a.most * a.split, g = lane >> 2, t = lane & 3u;
    const uint32_t sgroups = a.K / a.group, chunks = a.K / (128u * CH), gunits = a.group / U, myrow = (g & 1u) << 2 | (g & 2u) | g >> 2;
    const uint32_t slices = (chunks + a.slice - 1) / a.slice;
    // shared memory: rings, two slices of x, scales [gate, up][row of the tiles][pitch], barriers and the mark
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    uint4 *xs = reinterpret_cast<uint4 *>(smem + nwarps * kSlots * kSlot);
    uint32_t *scales = reinterpret_cast<uint32_t *>(xs + 2u * a.slice * kPieces);
    const uint32_t bars = saddr(scales + (size_t)a.most * 16u * a.pitch), full = bars, empty = bars + 16u, mark = bars + 32u, mine = bars + 40u + warp * kSlots * 8u;
    uint32_t tile0 = blockIdx.x * a.per + min(blockIdx.x, a.more);
    const uint32_t last = tile0 + a.per + (blockIdx.x < a.more);

    // A warp that has given up, by itself or because another one of the CTA has, requests nothing and tells no barrier: a slice that it
    // has not seen would be handed over, or written under those who still read it.
    bool gave_up = false;
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (gave_up || for_the_warp(bar_test(bar, parity))) return;
        const long long t0 = clock64();
        bool late = a.limit == 0;
        while (!late && !bar_try(bar, parity)) {
            uint32_t stop;
            asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(stop) : "r"(mark) : "memory");
            late = stop || clock64() - t0 > a.limit;
        }
        if (__any_sync(0xffffffffu, late)) {
            gave_up = true;
            if (lane == 0) {
                asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(mark), "r"(1u) : "memory");
                *reinterpret_cast<volatile uint32_t *>(a.status) = 1u;
            }
        }
    };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; i++) { bar_init(full + 8u * i, kStagers); bar_init(empty + 8u * i, nwarps); }
        for (uint32_t i = 0; i < nwarps * kSlots; i++) bar_init(bars + 40u + 8u * i, 1);
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(mark), "r"(0u) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    if (warp >= nwarps) {
        // ---- activations, in the order of the codes
        asm volatile("griddepcontrol.wait;" ::: "memory");
        Ring r;
        for (uint32_t tiles_left = last - tile0; tiles_left; tiles_left -= min(tiles_left, a.most))
            for (uint32_t s = 0; s < slices; s++, r.next(2u)) {
                wait(empty + 8u * r.at, r.lap ^ 1u);
                if (gave_up) break;
                const uint32_t c0 = s * a.slice, have = min(a.slice, chunks - c0);
                uint4 *to = xs + r.at * a.slice * kPieces;
                // 128 columns of two rows a warp and step: whole lines to read, and no two of a store's phase in one bank; eight steps under way
                const uint32_t units = have * CH * 4u * NT, b = lane >> 2 & 1u, i = lane >> 3;
                for (uint32_t u0 = warp - nwarps; u0 < units; u0 += 8u * kStagers) {
                    uint4 v[8];
#pragma unroll
                    for (uint32_t j = 0; j < 8; j++) {
                        const uint32_t u = min(u0 + j * kStagers, units - 1u), sp = u / (4u * NT), row = min((u - sp * 4u * NT) * 2u + b, a.batch - 1u);
                        v[j] = piece_load<BITS, P::kCols>(reinterpret_cast<const uint16_t *>(a.x) + (size_t)row * a.K, c0 * CH + sp, i, t);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 8; j++) {
                        const uint32_t u = u0 + j * kStagers, sp = u / (4u * NT), row = (u - sp * 4u * NT) * 2u + b;
                        if (u < units && row < a.batch) to[((sp * 4u + i) * (8u * NT) + row) * 4u + t] = piece_order<BITS>(v[j]);
                    }
                }
                __syncwarp();
                if (lane == 0) bar_arrive(full + 8u * r.at);
            }
    } else {
        const uint32_t my_tile = warp / a.split, part = warp - my_tile * a.split, ring = saddr(smem) + warp * kSlots * kSlot;
        const uint32_t w0 = ring + myrow * 128u + ((((t * (P::kBytes / 4)) >> 4) ^ myrow) << 4) + ((t * (P::kBytes / 4)) & 15u);
        const uint32_t x0 = saddr(xs) + (g * 4u + t) * 16u;
        Ring xr, wr, lost;
        uint32_t owing = 0;
        for (; tile0 < last; tile0 += a.most) {
            const uint32_t ntiles = min(last - tile0, a.most);
            const bool work = my_tile < ntiles;
            uint32_t requested = part;                         // the chunk that is to be requested next
            auto request = [&](uint32_t slot) {
                if (!work || requested >= chunks || gave_up) return;
                if (lane == 0) {
                    const uint32_t to = ring + slot * kSlot, row = (tile0 + my_tile) * 8u;
                    bar_expect(mine + slot * 8u, kSlot);
                    tma_2d(to, &gmap, requested * 128u, row, mine + slot * 8u);
                    tma_2d(to + kHalf, &umap, requested * 128u, row, mine + slot * 8u);
                }
                requested += a.split;
            };
            for (uint32_t i = 0, slot = wr.at; i < kSlots; i++, slot ^= 1u) request(slot);
            fetch_scales<EXACT && (CH * kUnits > 1)>(a.scales[0], a.scales[1], scales, tile0, ntiles, a.N, sgroups, a.pitch, warp, nwarps, lane);
            asm volatile("bar.sync 1, %0;" ::"r"(nwarps * 32u) : "memory");
            asm volatile("griddepcontrol.wait;" ::: "memory");         // (the time of the kernels before this one is not a slice's)
            const uint32_t s0 = saddr(scales) + (my_tile * 8u + myrow) * a.pitch * 4u, up = ntiles * 32u * a.pitch;

            float tot[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) tot[n][j] = 0.0f;
            uint32_t chunk = part;
            // copies of this warp are under way, whichever wait runs out
            auto wait_for = [&](uint32_t bar, uint32_t parity) {
                if (gave_up) return;
                wait(bar, parity);
                if (gave_up) { lost = wr; owing = (requested - chunk) / a.split; }
            };
            for (uint32_t s = 0; s < slices; s++, xr.next(2u)) {
                wait_for(full + 8u * xr.at, xr.lap);
                const uint32_t end = work ? min(chunks, (s + 1) * a.slice) : 0u;
                for (; chunk < end; chunk += a.split, wr.next(kSlots)) {
                    wait_for(mine + wr.at * 8u, wr.lap);
                    uint32_t w = w0 + wr.at * kSlot, x = x0 + (xr.at * a.slice + chunk - s * a.slice) * (kPieces * 16u), at_scale = s0 + (EXACT ? chunk * (CH * kUnits * 2u) : 0u);
                    pin(w, x, at_scale);
                    uint32_t sc[2][kScales] = {};
                    if constexpr (EXACT) {
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const uint32_t at = at_scale + r * up;
                            if constexpr (CH * kUnits == 1) asm("ld.shared.u16 %0, [%1];" : "=r"(sc[r][0]) : "r"(at));
                            else if constexpr (kScales == 1) asm("ld.shared.b32 %0, [%1];" : "=r"(sc[r][0]) : "r"(at));
                            else if constexpr (kScales == 2) asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(sc[r][0]), "=r"(sc[r][1]) : "r"(at));
                            else asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(sc[r][0]), "=r"(sc[r][1]), "=r"(sc[r][2]), "=r"(sc[r][3]) : "r"(at));
                        }
                    }
                    auto scale = [&](int r, int u) {
                        uint32_t v;
                        if (EXACT) v = sc[r][u / 2] >> (16 * (u & 1));
                        else asm("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(at_scale + r * up + (chunk * (uint32_t)(CH * kUnits) + u) / gunits * 2u));
                        return __half2float(__ushort_as_half((uint16_t)v));
                    };
#pragma unroll
                    for (int sp = 0; sp < CH; sp++) {
                        constexpr int kSpanParts = kParts128 / CH;             // parts of a span
                        uint32_t code[2][BITS];
#pragma unroll
                        for (int r = 0; r < 2; r++)
#pragma unroll
                            for (int p = 0; p < kSpanParts; p++) {
                                const uint32_t at = (w ^ ((sp * kSpanParts + p) * P::kBytes)) + r * kHalf;
                                uint32_t *d = &code[r][p * kWords];
                                if constexpr (kWords == 1) asm("ld.shared.b32 %0, [%1];" : "=r"(d[0]) : "r"(at));
                                else if constexpr (kWords == 2) asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "r"(at));
                                else asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(at));
                            }
                        float c[NT][4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            uint32_t h[2][4];
#pragma unroll
                            for (int r = 0; r < 2; r++) {
                                if constexpr (BITS == 4) {
                                    unpack_word<BITS, BF16>(code[r][i], h[r]);
                                } else if constexpr (BITS == 2) {
                                    uint32_t e[8];
                                    unpack_word<BITS, BF16>(code[r][i / 2], e);
#pragma unroll
                                    for (int j = 0; j < 4; j++) h[r][j] = e[4 * (i & 1) + j];
                                } else {
                                    uint32_t e[2];
#pragma unroll
                                    for (int j = 0; j < 2; j++) {
                                        unpack_word<BITS, BF16>(code[r][2 * i + j], e);
                                        h[r][2 * j] = e[0]; h[r][2 * j + 1] = e[1];
                                    }
                                }
                            }
                            uint4 q[NT];
#pragma unroll
                            for (int n = 0; n < NT; n++)
                                asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q[n].x), "=r"(q[n].y), "=r"(q[n].z), "=r"(q[n].w) : "r"(x + (sp * 4 + i) * (NT * 512) + n * 512));
                            constexpr int kOfUnit = 4 / kUnits;                    // pieces
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                if (i % kOfUnit == 0) mma_m16n8k16_first<BF16>(c[n], h[0][0], h[1][0], h[0][1], h[1][1], q[n].x, q[n].y);
                                else mma_m16n8k16<BF16>(c[n], h[0][0], h[1][0], h[0][1], h[1][1], q[n].x, q[n].y);
                            }
#pragma unroll
                            for (int n = 0; n < NT; n++) mma_m16n8k16<BF16>(c[n], h[0][2], h[1][2], h[0][3], h[1][3], q[n].z, q[n].w);
                            if (i % kOfUnit == kOfUnit - 1) {
                                const int u = sp * kUnits + i / kOfUnit;
                                const float fa = scale(0, u), fb = scale(1, u);
#pragma unroll
                                for (int n = 0; n < NT; n++) {
                                    tot[n][0] = fmaf(fa, c[n][0], tot[n][0]); tot[n][1] = fmaf(fa, c[n][1], tot[n][1]);
                                    tot[n][2] = fmaf(fb, c[n][2], tot[n][2]); tot[n][3] = fmaf(fb, c[n][3], tot[n][3]);
                                }
                            }
                        }
                    }
                    // every lane's codes have gone into products: the slot is free
                    __syncwarp();
                    request(wr.at);
                }
                __syncwarp();
                if (lane == 0 && !gave_up) bar_arrive(empty + 8u * xr.at);
            }
            if (owing) {                               // no copy may be under way when its place is used otherwise
                const long long t0 = clock64();
                for (; owing; owing--, lost.next(kSlots)) while (!bar_try(mine + lost.at * 8u, lost.lap) && clock64() - t0 < 20000000ll) {}
            }
            // the warp's sums, [row][row of x], where its ring was
            float *red = reinterpret_cast<float *>(smem + warp * kSlots * kSlot);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint32_t b = n * 8u + 2u * t;
                red[g * (8 * NT) + b] = tot[n][0]; red[g * (8 * NT) + b + 1] = tot[n][1];
                red[(g + 8) * (8 * NT) + b] = tot[n][2]; red[(g + 8) * (8 * NT) + b + 1] = tot[n][3];
            }
            asm volatile("bar.sync 1, %0;" ::"r"(nwarps * 32u) : "memory");
            uint32_t stopped;
            asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(stopped) : "r"(mark) : "memory");
            for (uint32_t i = threadIdx.x; i < ntiles * 64u * NT; i += nwarps * 32u) {
                const uint32_t f = i & 7u, b = (i >> 3) % (8u * NT), tile = i / (64u * NT), feature = (tile0 + tile) * 8u + ((f & 1u) << 2 | (f & 2u) | f >> 2);
                if (feature >= a.N || b >= a.batch) continue;
                float gs = 0.0f, us = 0.0f;
                for (uint32_t w = tile * a.split; w < (tile + 1) * a.split; w++) {
                    const float *from = reinterpret_cast<const float *>(smem + w * kSlots * kSlot);
                    gs += from[f * (8 * NT) + b];
                    us += from[(8 + f) * (8 * NT) + b];
                }
                gs += bias_at(a.bias[0], feature, a.bias_dtype);
                us += bias_at(a.bias[1], feature, a.bias_dtype);
                if (stopped) gs = us = __uint_as_float(0x7fffffffu);
                const size_t at = (size_t)b * a.N + feature;
                auto put = [&](void *to, float value) {
                    if (BF16) reinterpret_cast<__nv_bfloat16 *>(to)[at] = __float2bfloat16_rn(value);
                    else reinterpret_cast<__half *>(to)[at] = __float2half_rn(value);
                };
                put(a.h, activation(gs, a.act) * us);
                if (!a.kept[0]) continue;
                if (a.kept32) {
                    reinterpret_cast<float *>(a.kept[0])[at] = gs;
                    reinterpret_cast<float *>(a.kept[1])[at] = us;
                } else {
                    put(a.kept[0], gs);
                    put(a.kept[1], us);
                }
            }
            // the rings are the copies' again when all have read
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 1, %0;" ::"r"(nwarps * 32u) : "memory");
            gave_up = gave_up || stopped;
        }
    }
}

uint32_t rounded(uint32_t batch) { return batch <= 1 ? 1u : batch <= 4 ? 4u : 8u; }

// How a call is laid out: CTAs to an SM, warps, chunks of a warp's ring, tiles whose scales are in shared memory at a time (up to two a
// warp, see kParts, and 64 KB of scales).  A row's scales are an odd number of their loads' sizes apart, so that the rows of a tile lie in
// different banks.
struct Room { uint32_t warps, slots, most, pitch; size_t smem; };
Room room_for(const PackedPair &w, uint32_t bt, uint32_t warps, uint32_t slots, uint32_t tiles)
{
    // groups of a chunk (1024 bits of a row), whose scales one load of as many halves of a word fetches where that is a whole number
    const uint32_t groups = w.K / w.group, chunk = 1024u / (w.bits == 2 || w.bits == 4 ? w.bits : 8u) / w.group, load = std::max(1u, chunk / 2u);
    Room r;
    r.warps = warps;
    r.slots = slots;
    r.pitch = ((groups + 1) / 2 + load - 1) / load * load;
    if (r.pitch / load % 2 == 0) r.pitch += load;
    r.most = std::max(1u, std::min({2u * warps, tiles, 65536u / (64u * r.pitch)}));
    r.smem = 1024 + (size_t)warps * slots * (2048 + 8) + (size_t)w.K * bt * 2 + (size_t)r.most * 64 * r.pitch + (size_t)warps * kParts * 16 * bt * 4 + 16;
    return r;
}

typedef void (*Kernel)(RowsArgs, CUtensorMap, CUtensorMap);
typedef void (*ManyKernel)(ManyArgs, CUtensorMap, CUtensorMap);

template <int BITS, bool BF16, int U, bool EXACT>
Kernel by_batch(uint32_t bt)
{
    return bt == 1 ? (Kernel)gated_rows_kernel<BITS, BF16, U, EXACT, 1> : bt == 4 ? (Kernel)gated_rows_kernel<BITS, BF16, U, EXACT, 4> : (Kernel)gated_rows_kernel<BITS, BF16, U, EXACT, 8>;
}

// Groups that are several units go one scale at a time.
template <int BITS, bool BF16>
Kernel by_group(uint32_t group, uint32_t bt)
{
    constexpr int kLeast = BITS == 2 ? 64 : 32;
    if (group == 128u) return by_batch<BITS, BF16, 128, true>(bt);
    if (group == 64u) return by_batch<BITS, BF16, 64, true>(bt);
    if (group == 32u && kLeast == 32) return by_batch<BITS, BF16, kLeast, true>(bt);
    if (group % 128u == 0) return by_batch<BITS, BF16, 128, false>(bt);
    return by_batch<BITS, BF16, kLeast, false>(bt);
}

}  // namespace

// Nine to 32 rows: tiles at a time, warps of a tile, and as many chunks of activations a slice as two slices have room for.
struct ManyRoom { uint32_t nt, grid, most, split, slice, pitch; size_t smem; };
static ManyRoom many_room(const PackedPair &w, uint32_t batch)
{
    const uint32_t bits = w.bits == 2 || w.bits == 4 ? w.bits : 8u, tiles = (w.N + 7u) / 8u, chunks = w.row_bytes / 128u;
    ManyRoom r = {};
    r.nt = (batch + 7u) / 8u;
    r.grid = std::min(tiles, (uint32_t)std::max(1, device_sm_count()));
    const uint32_t per = (tiles + r.grid - 1) / r.grid, rounds = (per + kManyWarps - 1) / kManyWarps;
    r.most = (per + rounds - 1) / rounds;
    r.split = std::max(1u, std::min(kManyWarps / r.most, chunks));
    r.pitch = room_for(w, 8, 16, 2, 1).pitch;
    const uint32_t piece = 1024u / bits * 16u * r.nt;                  // bytes of a chunk of x
    const size_t fixed = 1024 + (size_t)r.most * r.split * (2 * 2048 + 16) + (size_t)r.most * 64 * r.pitch + 48;
    const size_t room = 226u * 1024u;
    if (fixed + 2 * piece > room) return ManyRoom{};
    r.slice = (uint32_t)std::min<size_t>((room - fixed) / (2 * piece), (chunks + 1) / 2);
    r.slice = std::max(1u, r.slice);
    if (r.slice > r.split) r.slice = r.slice / r.split * r.split;      // (every warp of a tile as many chunks of a slice)
    r.smem = fixed + 2 * (size_t)r.slice * piece;
    return r;
}

// Rows of whole 128-byte lines, whole units a group, scales that can be loaded two at a time, activations that fit beside two chunks a warp.
// 32 rows, or 24 of large weights, for which the products of pairs of SMs are quicker from there on (us, here at 32 rows and there at 33: 2816 x 1024
// 7.9 and 10.9, 11008 x 4096 30.2 and 33.6, 14336 x 4096 40.8 and 37.2, 28672 x 8192 141 and 111; here at 24 rows 32.5 and 113 for the last two.
// The large ones run 13 warps here; a size between with all 20 has not been measured).
bool gated_rows_takes(const PackedPair &w, uint32_t batch)
{
    const uint32_t most = (uint64_t)w.N * w.K > 50ull << 20 ? 24u : 32u;
    const uintptr_t scales = reinterpret_cast<uintptr_t>(w.scales[0]) | reinterpret_cast<uintptr_t>(w.scales[1]);
    return batch <= most && (scales & 3u) == 0 && product_takes(w, 2) && w.row_bytes % 128u == 0 && (w.bits != 2 || w.group % 64u == 0) &&
           (batch > 8 ? many_room(w, batch).smem > 0 : room_for(w, rounded(batch), 16, 2, 1u << 20).smem <= 226u * 1024u);
}

template <int BITS, bool BF16, int U, bool EXACT>
static ManyKernel many_of(uint32_t nt)
{
    return nt == 2 ? (ManyKernel)gated_many_rows_kernel<BITS, BF16, U, EXACT, 2> : nt == 3 ? (ManyKernel)gated_many_rows_kernel<BITS, BF16, U, EXACT, 3>
                                                                                          : (ManyKernel)gated_many_rows_kernel<BITS, BF16, U, EXACT, 4>;
}
template <int BITS, bool BF16>
static ManyKernel many_by_group(uint32_t group, uint32_t nt)
{
    constexpr int kLeast = BITS == 2 ? 64 : 32;
    if (group == 128u) return many_of<BITS, BF16, 128, true>(nt);
    if (group == 64u) return many_of<BITS, BF16, 64, true>(nt);
    if (group == 32u && kLeast == 32) return many_of<BITS, BF16, kLeast, true>(nt);
    if (group % 128u == 0) return many_of<BITS, BF16, 128, false>(nt);
    return many_of<BITS, BF16, kLeast, false>(nt);
}

static int launch_many_rows(const GatedCall &c, void *stream)
{
    const ManyRoom room = many_room(c.w, c.M);
    ManyArgs a = {};
    for (int i = 0; i < 2; i++) { a.scales[i] = c.w.scales[i]; a.bias[i] = c.bias[i]; a.kept[i] = c.keep.v[i]; }
    a.x = c.x; a.h = c.h; a.N = c.w.N; a.K = c.w.K; a.group = c.w.group; a.batch = c.M; a.act = c.act; a.kept32 = c.keep.form == kKeepF32; a.bias_dtype = c.bias_dtype;
    a.limit = gated_wait_limit();
    a.status = gated_status_word();
    if (!a.status) return (int)cudaErrorInvalidDevice;
    const uint32_t tiles = (a.N + 7u) / 8u;
    a.per = tiles / room.grid;
    a.more = tiles % room.grid;
    a.most = room.most; a.split = room.split; a.slice = room.slice; a.pitch = room.pitch;
    const bool bf = c.dtype == EOQ_B200_BF16;
    const ManyKernel kern = c.w.bits == 4   ? (bf ? many_by_group<4, true>(a.group, room.nt) : many_by_group<4, false>(a.group, room.nt))
                            : c.w.bits == 2 ? (bf ? many_by_group<2, true>(a.group, room.nt) : many_by_group<2, false>(a.group, room.nt))
                                            : (bf ? many_by_group<8, true>(a.group, room.nt) : many_by_group<8, false>(a.group, room.nt));
    CUtensorMap maps[2];
    for (int i = 0; i < 2; i++)
        if (!map_2d(maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, c.w.codes[i], c.w.row_bytes, c.w.N, c.w.row_bytes, 128, 8, CU_TENSOR_MAP_SWIZZLE_128B)) return (int)cudaErrorNotSupported;
    const uint32_t threads = (room.most * room.split + kStagers) * 32u;
    if (resident_ctas(reinterpret_cast<const void *>(kern), threads, room.smem, 1) == 0) return (int)cudaErrorNotSupported;      // (raises the kernel's limit of shared memory)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(room.grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = room.smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launches();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, maps[0], maps[1]);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_gated_rows(const GatedCall &c, void *stream)
{
    if (c.M > 8) return launch_many_rows(c, stream);
    RowsArgs a = {};
    for (int i = 0; i < 2; i++) { a.scales[i] = c.w.scales[i]; a.bias[i] = c.bias[i]; a.kept[i] = c.keep.v[i]; }
    a.x = c.x; a.h = c.h; a.N = c.w.N; a.K = c.w.K; a.group = c.w.group; a.batch = c.M; a.act = c.act; a.kept32 = c.keep.form == kKeepF32; a.bias_dtype = c.bias_dtype;
    a.limit = gated_wait_limit();
    a.status = gated_status_word();
    if (!a.status) return (int)cudaErrorInvalidDevice;
    const uint32_t bt = rounded(c.M);
    const bool bf = c.dtype == EOQ_B200_BF16;
    const Kernel kern = c.w.bits == 4   ? (bf ? by_group<4, true>(a.group, bt) : by_group<4, false>(a.group, bt))
                        : c.w.bits == 2 ? (bf ? by_group<2, true>(a.group, bt) : by_group<2, false>(a.group, bt))
                                        : (bf ? by_group<8, true>(a.group, bt) : by_group<8, false>(a.group, bt));
    const uint32_t sms = (uint32_t)device_sm_count(), tiles = (a.N + 7u) / 8u;
    // One row: 32 warps an SM, in four CTAs where a call is short, so that the next one's start comes under the end of this one's (11008 x
    // 4096, four bits 13.4 us with 4 x 8 warps, 13.6 with 2 x 16, 15.8 with 1 x 24; 28672 x 8192 62.0, 51.5, 54.3); more rows: 24, whose
    // activations leave no room for more.  Rings of three chunks are no quicker than of two.
    const bool brief = (uint64_t)tiles * (c.w.row_bytes / 128u) < 400ull * sms;
    uint32_t per_sm = bt == 1 && brief ? 4u : 2u, warps = bt > 1 ? 12u : brief ? 8u : 16u, slots = 2u;
    uint32_t grid = std::min(tiles, sms * per_sm);
    Room room = room_for(c.w, bt, warps, slots, (tiles + grid - 1) / grid);
    while (room.smem > 226u * 1024u / per_sm) {
        if (per_sm > 1) { per_sm /= 2; warps = std::min(24u, warps * 2); }
        else if (warps > 16) warps -= 4;
        else return (int)cudaErrorNotSupported;
        grid = std::min(tiles, sms * per_sm);
        room = room_for(c.w, bt, warps, slots, (tiles + grid - 1) / grid);
    }
    a.per = tiles / grid;
    a.more = tiles % grid;
    a.most = room.most;
    a.pitch = room.pitch;
    a.slots = room.slots;
    CUtensorMap maps[2];
    for (int i = 0; i < 2; i++)
        if (!map_2d(maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, c.w.codes[i], c.w.row_bytes, c.w.N, c.w.row_bytes, 128, 8, CU_TENSOR_MAP_SWIZZLE_128B)) return (int)cudaErrorNotSupported;
    if (resident_ctas(reinterpret_cast<const void *>(kern), warps * 32u, room.smem, 1) == 0) return (int)cudaErrorNotSupported;      // (raises the kernel's limit of shared memory)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(warps * 32u);
    cfg.dynamicSmemBytes = room.smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launches();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, maps[0], maps[1]);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace eoq
