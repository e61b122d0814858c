// The gated block on the fifth-generation tensor cores, straight from packed codes:
//   forward   h[m][n] = act(g + bg) (u + bu),  g = sum over k of x[m][k] wg[n][k], u likewise
//   gradient  dx[m][k] = sum over n of dg[m][n] wg[n][k] + du[m][n] wu[n][k]   (or of one weight)
//
// Both are products of a weight tile of 128 rows, which is the A operand and lives in tensor memory, with up to 256 tokens,
// which are the B operand, brought by TMA (128-byte swizzle).  Packed codes come by TMA too; producer warps turn them into
// code x scale, rounded to fp16 once, and store them to tensor memory, so that a dequantised weight touches neither global nor
// shared memory.  Activations are fp16, with one power of two per row where they were something else.
//
//   forward: a CTA's 128 rows are 64 features of the gate and the same 64 of the up projection, so that h is made where both
// sums are, on the way out.  A thread owns a row and turns 64 of its codes at a time into A's 32 columns.
//   gradient: a CTA's 128 rows are 128 columns of the weights, and the products run over the weights' rows, gate's first.  The
// codes lie the wrong way for that: a matrix load from shared memory transposes them, 16 bits (two, four or eight codes of a
// weight row) at a time, and leaves in each register the codes of two neighbouring weight rows at the same columns, half and
// half: what masking and a packed multiply-add make of it is a pair along the products' axis.  Its lanes are then sets of
// columns, not neighbouring ones; tensor memory takes them in that order, and the way out puts them back (`place`).
//
// Few tiles: the products' axis is split over the CTAs of a cluster, which add their sums up through distributed shared memory,
// in a fixed order.  Waits are bounded, as in the product kernel for one weight (qmm.cu): one that runs out marks the CTA,
// whose results become NaN, and sets a status word.
#include "gated.h"
#include "tensor_core.h"

#include <algorithm>
#include <atomic>
#include <cooperative_groups.h>

#include "activations.cuh"

namespace cg = cooperative_groups;

namespace eoq {

__device__ uint32_t g_gated_status = 0;

namespace {

constexpr uint32_t kRows = 128;            // of a weight tile
constexpr int kSets = 4;                   // producer sets of four warps, one per quadrant of tensor memory
constexpr uint32_t kThreads = (4 * kSets + 4) * 32, kTmem = 512;

struct ProductArgs {
    const uint16_t *scales[2];   // [N][groups] fp16
    const float *bias[2];        // forward: [N] or null
    const float *factor;         // [M] or null
    void *y;                     // [M][N] or, gradient, [M][K]
    Kept keep;                   // forward
    uint32_t N, K, M, T, group, groups, units, per_weight, split;
    uint32_t nw, ns;             // stages of packed weights and of operands
    uint32_t at_x, at_bar;       // shared-memory offsets
    int dtype, act;
    long long limit;             // clock ticks a wait may take
};

// Two words of shared memory at `mark`: the CTA has given up; the kernels before this one have ended (their time does not count).
struct Patience {
    uint32_t mark;
    long long limit;
    __device__ __forceinline__ bool stopped() const
    {
        uint32_t v;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(mark) : "memory");
        return v != 0;
    }
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) const
    {
        if (!bar_try(bar, parity)) slow(bar, parity, mark, limit);
    }
    // the same, and whether the CTA has not given up: a copy is requested then only
    __device__ __forceinline__ bool go(uint32_t bar, uint32_t parity) const
    {
        (*this)(bar, parity);
        return !stopped();
    }
    static __device__ __noinline__ void slow(uint32_t bar, uint32_t parity, uint32_t mark, long long limit)
    {
        long long t0 = clock64();
        while (!bar_try(bar, parity)) {
            const long long now = clock64();
            uint32_t stop, alone;
            asm volatile("ld.volatile.shared.v2.u32 {%0, %1}, [%2];" : "=r"(stop), "=r"(alone) : "r"(mark) : "memory");
            if (!alone && limit) t0 = now;
            // once a launch has given up, the others of a grid of many rounds wait an eighth as long
            if (!stop && now - t0 <= limit && !(now - t0 > limit / 8 && *reinterpret_cast<volatile uint32_t *>(&g_gated_status))) continue;
            asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(mark), "r"(1u) : "memory");
            *reinterpret_cast<volatile uint32_t *>(&g_gated_status) = 1u;
            return;
        }
    }
};

// What one weight copy brings, in blocks of 64 along the products' axis.
template <bool GRAD, int BITS>
struct Piece {
    static constexpr uint32_t kBytes = GRAD ? 16u * BITS : BITS == 2 ? 64u : 128u;      // of one row
    static constexpr uint32_t kAlong = GRAD ? 128u : kBytes * 8u / BITS;                 // along the products' axis
    static constexpr uint32_t kBlocks = kAlong / 64u;
    static constexpr uint32_t kStage = kRows * kBytes;
};

// barriers, eight bytes each
enum { bWFull = 0, bWEmpty = 8, bFull = 16, bEmpty = 24, bDone = 32, bSFull = 40, bSEmpty = 44, bTmem = 48, bDrain = 49, bMark = 50, bUsedW = 51, bUsedX = 52 };
constexpr uint32_t kScaleRing = 4, kScaleEntry = 8u * kRows * 2u;      // forward: 8 groups x 128 rows an entry; gradient: up to 4 groups x 128

__device__ __forceinline__ void ldmatrix_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// sixteen lanes x 32 columns: register 2 b to lane (thread / 4), column 4 b + thread % 4, register 2 b + 1 to lane 8 + thread / 4
__device__ __forceinline__ void tmem_st_16x128b(uint32_t addr, const uint32_t (&r)[16])
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

template <bool GRAD, int BITS>
__global__ void __launch_bounds__(kThreads, 1)
gated_product_kernel(const ProductArgs a, const __grid_constant__ CUtensorMap gmap, const __grid_constant__ CUtensorMap umap, const __grid_constant__ CUtensorMap xmap)
{
    using P = Piece<GRAD, BITS>;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023u) & ~(uintptr_t)1023u);
    const uint32_t base = saddr(smem), bars = base + a.at_bar;
    auto bar = [&](uint32_t i) { return bars + 8u * i; };
    auto word = [&](uint32_t i) { return reinterpret_cast<volatile uint32_t *>(smem + a.at_bar + 8u * i); };
    const Patience wait{bar(bMark), a.limit};
    const uint32_t scale_ring = bars + 512u;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u;
    const uint32_t rank = blockIdx.x % a.split, tile = blockIdx.x / a.split, tok0 = blockIdx.y * a.T;
    const uint32_t row0 = tile * (GRAD ? 128u : 64u);                // first column, or feature
    const uint32_t u0 = (uint32_t)((uint64_t)a.units * rank / a.split), u1 = (uint32_t)((uint64_t)a.units * (rank + 1) / a.split);
    // forward: the last piece's blocks past the last column are left out; gradient: rows past the last one are zeros
    const uint32_t kb0 = u0 * P::kBlocks, nkb = (GRAD ? u1 * P::kBlocks : min(u1 * P::kBlocks, (a.K + 63u) / 64u)) - kb0;
    const uint32_t xstage = a.T * 128u, a_base = a.T;
    const uint32_t grp0 = kb0 * 64u / a.group, ngroups = GRAD ? 0u : (min((kb0 + nkb) * 64u, a.K) - 1u) / a.group - grp0 + 1u;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 8; i++) {
            bar_init(bar(bWFull + i), 1); bar_init(bar(bWEmpty + i), 4 * P::kBlocks);
            bar_init(bar(bFull + i), 5); bar_init(bar(bEmpty + i), 1);          // four producer warps and the activation copy
        }
        for (uint32_t i = 0; i < kScaleRing; i++) { bar_init(bar(bSFull + i), 1); bar_init(bar(bSEmpty + i), 4 * (GRAD ? P::kBlocks : kSets)); }
        bar_init(bar(bDone), 1);
        bar_init(bar(bDrain), 1);
        word(bMark)[0] = word(bMark)[1] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 4 * kSets) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar(bTmem)), "n"(kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    constexpr uint32_t tmem = 0;               // all 512 columns are this CTA's

    if (warp < 4 * kSets) {
        // ---- producers: codes, a block of 64 along the products' axis at a time, to the A operand in tensor memory
        const uint32_t set = warp >> 2, q = warp & 3u, r = q * 32u + lane;
        const uint32_t lane_base = tmem + ((q * 32u) << 16) + a_base;
        Ring wr, ar, sr;
        uint32_t unit = 0, entry = 0, gi = 0, pos = 0;
        bool here = false;
        if (!GRAD) { const uint32_t c = (kb0 + set) * 64u; gi = c / a.group; pos = c - gi * a.group; gi -= grp0; }
        // forward: scales of this row in the order of the groups, out of the ring
        auto scale_of = [&](uint32_t g) {
            while ((g >> 3) > entry) {
                __syncwarp();
                if (lane == 0) bar_arrive(bar(bSEmpty + sr.at));
                sr.next(kScaleRing);
                entry++;
                here = false;
            }
            if (!here) { wait(bar(bSFull + sr.at), sr.lap); here = true; }
            uint16_t v;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(scale_ring + sr.at * kScaleEntry + (g & 7u) * (kRows * 2u) + r * 2u));
            return v;
        };
        for (uint32_t j = 0; j < set; j++) ar.next(a.ns);
        for (uint32_t i = set; i < nkb; i += kSets) {
            const uint32_t qb = i % P::kBlocks, st = ar.at;
            for (; unit < i / P::kBlocks; unit++) { wr.next(a.nw); if (GRAD) sr.next(kScaleRing); }
            const uint32_t ws = wr.at;
            wait(bar(bWFull + ws), wr.lap);
            if constexpr (!GRAD) {
                constexpr int kWords = BITS == 4 ? 8 : BITS == 2 ? 4 : 16;
                const uint32_t row_at = base + ws * P::kStage + r * P::kBytes, sw = BITS == 2 ? (r >> 1) & 3u : r & 7u;
                uint32_t w[kWords], h[32];
#pragma unroll
                for (uint32_t c = 0; c < kWords / 4; c++)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[4 * c]), "=r"(w[4 * c + 1]), "=r"(w[4 * c + 2]), "=r"(w[4 * c + 3])
                                 : "r"(row_at + (((qb * (kWords / 4) + c) ^ sw) << 4)));
                const uint16_t s0 = scale_of(gi);
                const bool other = pos + 32u >= a.group && (kb0 + i) * 64u + 32u < a.K;
                const uint16_t s1 = other ? scale_of(gi + 1u) : s0;
                for (pos += 64u * kSets; pos >= a.group; pos -= a.group) gi++;
#pragma unroll
                for (int c = 0; c < kWords; c++) codes_scaled<BITS, false>(w[c], h + c * (32 / kWords), c < kWords / 2 ? s0 : s1);
                wait(bar(bEmpty + st), ar.lap ^ 1u);
                fence_after();
                __syncwarp();
                tmem_st32(lane_base + st * 32u, h);
            } else {
                constexpr int kChunks = BITS == 8 ? 2 : 1;            // 16-byte pieces of a weight row that a quadrant's 32 columns take
                const uint32_t rows_at = base + ws * P::kStage, chunk = BITS == 4 ? q : BITS == 8 ? 2u * q : q >> 1;
                // scales of neighbouring weight rows at this lane's columns' group
                const uint32_t col = place<true, BITS>(q, lane >> 2), gl = (row0 + col) / a.group - row0 / a.group;
                wait(bar(bSFull + sr.at), sr.lap);
                uint32_t sp[8];
#pragma unroll
                for (uint32_t b = 0; b < 8; b++)
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(sp[b]) : "r"(scale_ring + sr.at * kScaleEntry + gl * (kRows * 2u) + qb * 128u + b * 16u + (lane & 3u) * 4u));
                uint32_t m[kChunks][2][4];
#pragma unroll
                for (uint32_t c = 0; c < kChunks; c++)
#pragma unroll
                    for (uint32_t hh = 0; hh < 2; hh++) {
                        const uint32_t n = qb * 64u + hh * 32u + lane, sw = BITS == 8 ? n & 7u : BITS == 4 ? (n >> 1) & 3u : (n >> 2) & 1u;
                        ldmatrix_trans(rows_at + n * P::kBytes + (((chunk + c) ^ sw) << 4), m[c][hh]);
                    }
                // sixteen lanes of tensor memory at a time: code j of the registers to lanes 0 .. 7, code j + 1 to lanes 8 .. 15
                uint32_t h[2][16];
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int b = 0; b < 8; b++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            uint32_t v = m[BITS == 8 ? half : 0][b >> 2][b & 3];
                            if (BITS == 2) v >>= (q & 1u) * 8u;
                            h[half][2 * b + j] = hmul2(row_pair<BITS>(v, (BITS == 8 ? 0 : 2 * half) + j), sp[b]);
                        }
                wait(bar(bEmpty + st), ar.lap ^ 1u);
                fence_after();
                __syncwarp();
                tmem_st_16x128b(lane_base + st * 32u, h[0]);
                tmem_st_16x128b(lane_base + (16u << 16) + st * 32u, h[1]);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            fence_before();
            __syncwarp();
            // every lane's codes are converted and stored: only now may the copy engine have the stage.  A CTA that has given up
            // tells nobody (an arrival beyond a barrier's count while a copy is under way would break it)
            if (lane == 0 && !wait.stopped()) {
                bar_arrive(bar(bFull + st));
                bar_arrive(bar(bWEmpty + ws));
                if (GRAD) bar_arrive(bar(bSEmpty + sr.at));
            }
#pragma unroll
            for (int j = 0; j < kSets; j++) ar.next(a.ns);
        }
    } else if (warp == 4 * kSets) {
        // ---- products
        const uint32_t idesc = (1u << 4) | ((a.T >> 3) << 17) | ((kRows >> 4) << 24);
        const uint64_t desc0 = sw128_desc(base + a.at_x);
        uint32_t acc = 0;
        Ring ar;
        for (uint32_t i = 0; i < nkb; i++) {
            wait(bar(bFull + ar.at), ar.lap);
            fence_after();
            const uint32_t at = tmem + a_base + ar.at * 32u;
            const uint64_t desc = desc0 + ((ar.at * xstage) >> 4);
            // (past the last column of a forward product the codes are zeros of the copy, times a scale, and the activations zeros)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) { mma_ts(tmem, at + j * 8u, desc + j * 2u, idesc, acc); acc = 1; }
            mma_commit(bar(bEmpty + ar.at));
            ar.next(a.ns);
        }
        mma_commit(bar(bDone));
    } else if (warp == 4 * kSets + 1) {
        // ---- weight copies: a resident weight depends on nothing that came before in the stream
        const bool leader = elect();
        Ring wr;
        uint32_t used = 0;
        for (uint32_t u = u0; u < u1; u++) {
            const bool go = wait.go(bar(bWEmpty + wr.at), wr.lap ^ 1u);
            if (leader && go) {
                used++;
                const uint32_t to = base + wr.at * P::kStage, full = bar(bWFull + wr.at);
                bar_expect(full, P::kStage);
                if constexpr (GRAD) {
                    const uint32_t which = u >= a.per_weight;
                    tma_2d(to, which ? &umap : &gmap, tile * P::kBytes, (u - (which ? a.per_weight : 0u)) * P::kAlong, full);
                } else {
                    tma_2d(to, &gmap, u * P::kBytes, row0, full);
                    tma_2d(to + P::kStage / 2u, &umap, u * P::kBytes, row0, full);
                }
            }
            __syncwarp();
            wr.next(a.nw);
        }
        if (leader) *word(bUsedW) = used;
    } else if (warp == 4 * kSets + 2) {
        // ---- activation copies
        const bool leader = elect();
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (leader) word(bMark)[1] = 1u;
        Ring xr;
        uint32_t used = 0;
        for (uint32_t i = 0; i < nkb; i++) {
            const bool go = wait.go(bar(bEmpty + xr.at), xr.lap ^ 1u);
            if (leader && go) {
                used++;
                bar_expect(bar(bFull + xr.at), xstage);
                uint32_t along = (kb0 + i) * 64u, rows = tok0;
                if (GRAD && along >= a.per_weight * P::kAlong) { along -= a.per_weight * P::kAlong; rows += a.M; }
                tma_2d(base + a.at_x + xr.at * xstage, &xmap, along, rows, bar(bFull + xr.at));
            }
            __syncwarp();
            xr.next(a.ns);
        }
        if (leader) *word(bUsedX) = used;
    } else if constexpr (!GRAD) {
        // ---- scales: eight groups of 128 rows at a time, transposed on the way ([group][row])
        Ring sr;
        for (uint32_t g0 = 0; g0 < ngroups; g0 += 8u) {
            uint16_t v[4][8];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint16_t *srow = a.scales[j >> 1] + (size_t)min(row0 + lane + 32u * (j & 1u), a.N - 1u) * a.groups;
#pragma unroll
                for (uint32_t g = 0; g < 8; g++) v[j][g] = __ldg(srow + min(grp0 + g0 + g, a.groups - 1u));
            }
            wait(bar(bSEmpty + sr.at), sr.lap ^ 1u);
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
#pragma unroll
                for (uint32_t g = 0; g < 8; g++)
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(scale_ring + sr.at * kScaleEntry + g * (kRows * 2u) + j * 64u + lane * 2u), "h"(v[j][g]) : "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(bar(bSFull + sr.at));
            sr.next(kScaleRing);
        }
    } else {
        // ---- scales of a piece's 128 weight rows at the tile's columns, up to four groups ([group][row]); zero past the last row, so
        // that what lies behind it (there the activations are zeros) cannot be an infinity
        const uint32_t g_first = row0 / a.group, ng = (min(row0 + 127u, a.K - 1u)) / a.group - g_first + 1u;
        Ring sr;
        for (uint32_t u = u0; u < u1; u++) {
            const uint32_t which = u >= a.per_weight, n0 = (u - (which ? a.per_weight : 0u)) * P::kAlong;
            uint16_t v[4][4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t n = n0 + j * 32u + lane;
#pragma unroll
                for (uint32_t g = 0; g < 4; g++) v[j][g] = g < ng && n < a.N ? __ldg(a.scales[which] + (size_t)n * a.groups + g_first + g) : (uint16_t)0;
            }
            wait(bar(bSEmpty + sr.at), sr.lap ^ 1u);
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
#pragma unroll
                for (uint32_t g = 0; g < 4; g++)
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(scale_ring + sr.at * kScaleEntry + g * (kRows * 2u) + j * 64u + lane * 2u), "h"(v[j][g]) : "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(bar(bSFull + sr.at));
            sr.next(kScaleRing);
        }
    }
    __syncwarp();
    if (warp < 4 * kSets) {
        // sums to shared memory, [token][row]: sixteen tokens at a time.  (All products are behind: the stages are free.)
        wait(bar(bDone), 0u);
        __syncwarp();
        fence_after();
        const uint32_t q = warp & 3u, to = place<GRAD, BITS>(q, lane);
        for (uint32_t c = (warp >> 2) * 16u; c < a.T; c += kSets * 16u) {
            uint32_t v[16];
            tmem_ld16(tmem + ((q * 32u) << 16) + c, v);
            tmem_ld_wait(v);
#pragma unroll
            for (int j = 0; j < 16; j++) reinterpret_cast<float *>(smem)[(size_t)(c + j) * kRows + to] = __uint_as_float(v[j]);
        }
        fence_before();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    if (wait.stopped()) {                          // the same for all threads: whoever sets the mark does so before the barrier above
        // nothing may be under way any more when tensor and shared memory are given back
        if (warp == 4 * kSets) { mma_commit(bar(bDrain)); drain(bar(bDrain), 1u, 1u); }
        if (warp == 4 * kSets + 1) drain(bar(bWFull), *word(bUsedW), a.nw);
        if (warp == 4 * kSets + 2) drain(bar(bFull), *word(bUsedX), a.ns);
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < a.T * kRows; e += kThreads) reinterpret_cast<uint32_t *>(smem)[e] = 0x7fffffffu;
        __syncthreads();
    }
    if (warp == 4 * kSets) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem) : "memory");
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (a.split > 1) cluster.sync();
    const float *mine = reinterpret_cast<const float *>(smem);
    // four values of a token, all the cluster's CTAs' added up; requested before the first is added
    auto sum4 = [&](uint32_t at) {
        if (a.split == 1) return *reinterpret_cast<const float4 *>(mine + at);
        float4 o[8], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) o[k] = k < a.split ? *reinterpret_cast<const float4 *>(cluster.map_shared_rank(mine, k) + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) { v.x += o[k].x; v.y += o[k].y; v.z += o[k].z; v.w += o[k].w; }
        return v;
    };
    auto store4 = [&](void *to, size_t at, uint32_t left, bool vec, const float (&o)[4]) {
        if (a.dtype == EOQ_B200_F32) {
            float *y = reinterpret_cast<float *>(to) + at;
            if (vec) *reinterpret_cast<float4 *>(y) = make_float4(o[0], o[1], o[2], o[3]);
            else for (uint32_t j = 0; j < 4; j++) if (j < left) y[j] = o[j];
            return;
        }
        uint32_t p[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (a.dtype == EOQ_B200_F16) { const __half2 h = __floats2half2_rn(o[2 * j], o[2 * j + 1]); p[j] = *reinterpret_cast<const uint32_t *>(&h); }
            else p[j] = pack_bf16(o[2 * j], o[2 * j + 1]);
        }
        uint16_t *y = reinterpret_cast<uint16_t *>(to) + at;
        if (vec) *reinterpret_cast<uint2 *>(y) = make_uint2(p[0], p[1]);
        else for (uint32_t j = 0; j < 4; j++) if (j < left) y[j] = (uint16_t)(p[j >> 1] >> (16 * (j & 1)));
    };
    constexpr uint32_t kQuads = GRAD ? 32u : 16u;              // of a token's results in this tile
    const uint32_t width = GRAD ? a.K : a.N;
    const bool vec = (width & 3u) == 0;
    // (whole warps go on together: the 8-bit form's lanes exchange values)
    for (uint32_t e = rank * kThreads + threadIdx.x; (e & ~31u) < a.T * kQuads; e += kThreads * a.split) {
        const uint32_t t = e / kQuads, c = (e % kQuads) * 4u, m = tok0 + t, n = row0 + c;
        const bool here = t < a.T && m < a.M && n < width;
        if constexpr (GRAD) {
            if (!here) continue;
            const float4 v = sum4(t * kRows + c);
            const float f = a.factor ? __ldg(a.factor + m) : 1.0f;
            const float o[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
            store4(a.y, (size_t)m * width + n, width - n, vec, o);
        } else {
            float g[4] = {}, u[4] = {}, h[4];
            if (here) {
                const float4 vg = sum4(t * kRows + c), vu = sum4(t * kRows + 64u + c);
                const float f = a.factor ? __ldg(a.factor + m) : 1.0f;
                g[0] = vg.x * f; g[1] = vg.y * f; g[2] = vg.z * f; g[3] = vg.w * f;
                u[0] = vu.x * f; u[1] = vu.y * f; u[2] = vu.z * f; u[3] = vu.w * f;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    if (n + j >= a.N) { g[j] = u[j] = 0.0f; continue; }       // (would count in an 8-bit block's largest)
                    if (a.bias[0]) g[j] += __ldg(a.bias[0] + n + j);
                    if (a.bias[1]) u[j] += __ldg(a.bias[1] + n + j);
                }
                const size_t at = (size_t)m * a.N + n;
#pragma unroll
                for (int j = 0; j < 4; j++) h[j] = activation(g[j], a.act) * u[j];
                store4(a.y, at, a.N - n, vec, h);
                if (a.keep.form == kKeepFull) {
                    store4(a.keep.v[0], at, a.N - n, vec, g);
                    store4(a.keep.v[1], at, a.N - n, vec, u);
                }
            }
            if (a.keep.form == kKeep8bit) {
                // the tile's 64 features of a token are one block of the 8-bit form, four a lane
                uint32_t mg = 0u, mu = 0u;
#pragma unroll
                for (int j = 0; j < 4; j++) { mg = max(mg, __float_as_uint(g[j]) & 0x7fffffffu); mu = max(mu, __float_as_uint(u[j]) & 0x7fffffffu); }
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) { mg = max(mg, __shfl_xor_sync(0xffffffffu, mg, d)); mu = max(mu, __shfl_xor_sync(0xffffffffu, mu, d)); }
                const Storer sg(mg), su(mu);
                if (here) {
                    const size_t at = (size_t)m * a.N + n, block = (size_t)m * ((a.N + kStoreBlock - 1) / kStoreBlock) + tile;
                    if (c == 0) { a.keep.scale[0][block] = sg.scale; a.keep.scale[1][block] = su.scale; }
                    uint32_t pg = 0u, pu = 0u;
#pragma unroll
                    for (int j = 0; j < 4; j++) { pg |= (uint32_t)(uint8_t)sg.code(g[j]) << (8 * j); pu |= (uint32_t)(uint8_t)su.code(u[j]) << (8 * j); }
                    uint8_t *kg = reinterpret_cast<uint8_t *>(a.keep.v[0]) + at, *ku = reinterpret_cast<uint8_t *>(a.keep.v[1]) + at;
                    if (vec) { *reinterpret_cast<uint32_t *>(kg) = pg; *reinterpret_cast<uint32_t *>(ku) = pu; }
                    else for (uint32_t j = 0; j < 4; j++) if (n + j < a.N) { kg[j] = (uint8_t)(pg >> (8 * j)); ku[j] = (uint8_t)(pu >> (8 * j)); }
                }
            }
        }
    }
    if (a.split > 1) cluster.sync();               // nobody leaves while its sums are being read
}

std::atomic<long long> g_limit{4000000000ll};      // about two seconds

struct Layout { uint32_t nw, ns, at_x, at_bar; size_t smem; };

// A producer set has to come by every operand stage on every lap (its parity waits look one lap back): stages in multiples of the
// sets, weight stages in multiples of the copies that a set steps over.
Layout lay_out(uint32_t T, uint32_t stage_w, uint32_t blocks)
{
    const uint32_t fixed = 512 + 1024 + kScaleRing * kScaleEntry, room = 226u * 1024u - fixed, xstage = T * 128u, step = std::max(1u, kSets / blocks);
    Layout l = {};
    l.ns = T <= 128u ? 8u : 4u;
    if (room < l.ns * xstage + 4u * stage_w) l.ns = 4u;
    l.nw = std::min(8u, (room - l.ns * xstage) / stage_w) / step * step;
    l.at_x = l.nw * stage_w;
    l.at_bar = std::max(l.at_x + l.ns * xstage, T * kRows * 4u);
    l.smem = l.at_bar + fixed;
    return l;
}

struct Cut { uint32_t T, tok_tiles, split; };

// Token tile and split with the least rounds of resident CTAs x what a CTA takes: blocks of 64, each the longer of its products
// (two cycles a token) and its producers' work, and some four thousand cycles to start, fill and store (half as many more to meet in a
// cluster).
template <class Room>
Cut cut(uint32_t tiles, uint32_t M, uint32_t units, uint32_t blocks, Room &&room)
{
    Cut best = {};
    double least = 1e30;
    const uint32_t fewest = (M + 255u) / 256u;
    for (uint32_t n = fewest; n < fewest + 4; n++) {
        const uint32_t T = ((M + n - 1) / n + 15u) / 16u * 16u;
        if (n > fewest && (T >= best.T || (M + T - 1) / T < n)) continue;
        const double block = std::max(400.0, 2.0 * T + 150.0);
        for (uint32_t split = 1; split <= 8 && split <= units; split++) {
            const uint32_t at_once = room(T, split);
            if (!at_once) continue;
            const double cost = (double)(((uint64_t)tiles * n * split + at_once - 1) / at_once) *
                                ((double)((units + split - 1) / split) * blocks * block + 4000.0 * (split > 1 ? 1.5 : 1.0));
            if (cost < least * (n > best.tok_tiles && best.T ? 0.95 : 0.999)) { least = cost; best = Cut{T, n, split}; }
        }
    }
    return best;
}

template <bool GRAD, int BITS>
int run(ProductArgs a, const PackedPair &w, int nw, const void *x, uint32_t pitch, cudaStream_t st)
{
    using P = Piece<GRAD, BITS>;
    auto kern = gated_product_kernel<GRAD, BITS>;
    const uint32_t tiles = GRAD ? (a.K + 127u) / 128u : (a.N + 63u) / 64u;
    a.per_weight = GRAD ? (a.N + P::kAlong - 1) / P::kAlong : 0u;
    a.units = GRAD ? a.per_weight * nw : (a.K + P::kAlong - 1) / P::kAlong;
    // the cuts of the last shapes (a model has a handful)
    struct Known { uint32_t tiles, M, units; int dev; Cut c; };
    static std::mutex mu;
    static Known known[32];
    static uint32_t used = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return (int)cudaErrorInvalidDevice;
    Cut c = {};
    {
        std::lock_guard<std::mutex> lock(mu);
        for (uint32_t i = 0; i < std::min(used, 32u); i++)
            if (known[i].tiles == tiles && known[i].M == a.M && known[i].units == a.units && known[i].dev == dev) c = known[i].c;
    }
    if (!c.T) {
        c = cut(tiles, a.M, a.units, P::kBlocks, [&](uint32_t T, uint32_t split) {
            return resident_ctas(reinterpret_cast<const void *>(kern), kThreads, lay_out(T, P::kStage, P::kBlocks).smem, split);
        });
        if (!c.T) return (int)cudaErrorNotSupported;
        std::lock_guard<std::mutex> lock(mu);
        known[used % 32] = Known{tiles, a.M, a.units, dev, c};
        used = used + 1 >= 64 ? 32 : used + 1;
    }
    const Layout l = lay_out(c.T, P::kStage, P::kBlocks);
    a.T = c.T; a.split = c.split; a.nw = l.nw; a.ns = l.ns; a.at_x = l.at_x; a.at_bar = l.at_bar;
    CUtensorMap maps[2], xmap;
    constexpr CUtensorMapSwizzle sw = P::kBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : P::kBytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    for (int i = 0; i < 2; i++)
        if (!map_2d(maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes[i], w.row_bytes, w.N, w.row_bytes, P::kBytes, GRAD ? kRows : kRows / 2, sw)) return (int)cudaErrorNotSupported;
    if (!map_2d(xmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, x, GRAD ? w.N : w.K, (uint64_t)a.M * (GRAD ? nw : 1), (uint64_t)pitch * 2, 64, c.T, CU_TENSOR_MAP_SWIZZLE_128B))
        return (int)cudaErrorNotSupported;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * c.split, c.tok_tiles);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = l.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launches();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = c.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, maps[0], maps[1], xmap);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

ProductArgs common(const PackedPair &w, const float *factor, uint32_t M, void *y, int dtype)
{
    ProductArgs a = {};
    a.scales[0] = w.scales[0]; a.scales[1] = w.scales[1];
    a.factor = factor; a.y = y; a.N = w.N; a.K = w.K; a.M = M; a.group = w.group; a.groups = w.K / w.group; a.dtype = dtype;
    a.limit = g_limit.load(std::memory_order_relaxed);
    return a;
}

}  // namespace

bool product_takes(const PackedPair &w, int nw)
{
    for (int i = 0; i < nw; i++)
        if (!qmm_takes(w.K, w.bits, w.group, w.codes[i], w.codes[i])) return false;
    return true;
}

int launch_gated_product(const GatedCall &c, const uint16_t *x, const float *factor, void *stream)
{
    ProductArgs a = common(c.w, factor, c.M, c.h, c.dtype);
    a.bias[0] = c.bias[0]; a.bias[1] = c.bias[1];
    a.keep = c.keep;
    a.act = c.act;
    cudaStream_t st = (cudaStream_t)stream;
    if (c.w.bits == 4) return run<false, 4>(a, c.w, 2, x, c.w.K, st);
    if (c.w.bits == 2) return run<false, 2>(a, c.w, 2, x, c.w.K, st);
    return run<false, 8>(a, c.w, 2, x, c.w.K, st);
}

int launch_input_grad_product(const PackedPair &w, int nw, const uint16_t *dy, uint32_t pitch, const float *factor, uint32_t M, void *dx, int dtype, void *stream)
{
    const ProductArgs a = common(w, factor, M, dx, dtype);
    cudaStream_t st = (cudaStream_t)stream;
    if (w.bits == 4) return run<true, 4>(a, w, nw, dy, pitch, st);
    if (w.bits == 2) return run<true, 2>(a, w, nw, dy, pitch, st);
    return run<true, 8>(a, w, nw, dy, pitch, st);
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
