// The gated block for a few rows (up to eight of 16-bit activations): one pass over both weights' codes.
//
// Warp-level products, D[16 x 8] += A[16 x 16] B[16 x 8] (mma.sync m16n8k16), the codes exact and the scales applied to the sums in
// fp32, with gate rows and up rows of the same features in one instruction: lane (g, t) takes gate row g as A's row g and up row g as
// A's row g + 8, so that the sums of both, for the same feature and rows of x, end in the same lane.  The contraction index is a
// dummy: a lane feeds its codes in the order in which they leave their words cheapest (packed_mma.h), and the activations, brought
// to shared memory in that order once per CTA, follow.
//
// A CTA takes a run of neighbouring eights of features ("tiles"), and its warps equal runs of the tiles' 128-column spans, whichever
// tile these belong to; a warp leaves its sums of a tile in shared memory where it goes on to the next one, and what the warps left is
// added up in their order.
#include "gated.h"
#include "packed_mma.h"

#include <algorithm>
#include <atomic>
#include <cuda_fp16.h>
#include <mutex>
#include <vector>

#include "activations.cuh"

namespace eoq {
namespace {

struct RowsArgs {
    const uint8_t *codes[2];
    const uint16_t *scales[2];
    const float *bias[2];
    const void *x;
    void *h;
    void *kept[2];               // [batch][N] of x's type, fp32 (kept32), or null
    uint32_t N, K, group, row_bytes, batch, tiles;
    int act, kept32;
};

constexpr uint32_t kMostThreads = 768;
constexpr int kParts = 3;        // tiles that a warp's run touches at most, for up to two tiles a warp

// x in the order of the codes: sixteen-byte pieces [span][i][row][t], piece i of lane (row, t) the columns of its registers 4 i .. 4 i + 3.
template <int BITS, int U>
__device__ __forceinline__ uint4 piece_of(const uint16_t *x, uint32_t span, uint32_t i, uint32_t t)
{
    if constexpr (BITS == 2) {       // columns 16 j + (r & 7) and + 8 of a lane's, j = i / 2
        const uint32_t j = i >> 1, c = span * 128u + (U == 128 ? t * 32u + j * 16u : j * 64u + t * 16u) + (i & 1u) * 4u;
        const uint2 a = __ldg(reinterpret_cast<const uint2 *>(x + c)), b = __ldg(reinterpret_cast<const uint2 *>(x + c + 8u));
        return make_uint4(__byte_perm(a.x, b.x, 0x5410u), __byte_perm(a.x, b.x, 0x7632u), __byte_perm(a.y, b.y, 0x5410u), __byte_perm(a.y, b.y, 0x7632u));
    } else {
        const uint32_t c = span * 128u + (U == 128 ? t * 32u + i * 8u : U == 64 ? (i >> 1) * 64u + t * 16u + (i & 1u) * 8u : i * 32u + t * 8u);
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(x + c));
        if constexpr (BITS == 8) return v;
        return make_uint4(__byte_perm(v.x, v.z, 0x5410u), __byte_perm(v.x, v.z, 0x7632u), __byte_perm(v.y, v.w, 0x5410u), __byte_perm(v.y, v.w, 0x7632u));
    }
}

// U: columns of a unit whose scale is applied on its own, the largest of 128, 64 and 32 that divides a group.  Of a span's units a lane
// takes an equal part each, 32 columns in all.  BT: rows of x, of which `batch` are there.
template <int BITS, bool BF16, int U, int BT>
__global__ void __launch_bounds__(kMostThreads, 1) gated_rows_kernel(const RowsArgs a)
{
    static_assert(BITS != 2 || U >= 64, "a unit of 32 two-bit codes is no whole word of a lane");
    constexpr int kUnits = 128 / U, kWords = BITS / kUnits;        // of a lane's part of a unit
    constexpr int kSets = BITS == 8 || U < 128 ? 2 : 3;            // register sets of codes and scales, all but one on their way (more spill)
    extern __shared__ uint4 xs[];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t sgroups = a.K / a.group, nspans = a.K >> 7, gunits = a.group / U;
    float (*red)[kParts][16][BT] = reinterpret_cast<float (*)[kParts][16][BT]>(xs + (size_t)nspans * 16u * BT);
    const uint32_t last = (uint32_t)((uint64_t)a.tiles * (blockIdx.x + 1) / gridDim.x);
    uint32_t tile0 = (uint32_t)((uint64_t)a.tiles * blockIdx.x / gridDim.x), ntiles = min(last - tile0, 2u * nwarps);

    // a warp's run of spans of the tiles at hand, and what one load of it brings: both rows' codes and scales
    uint32_t next, end, load_tile, load_span;
    const uint8_t *pw[2];
    const uint16_t *ps[2];
    auto at_tile = [&]() {
        const uint32_t row = min((tile0 + load_tile) * 8u + g, a.N - 1u);
#pragma unroll
        for (int r = 0; r < 2; r++) {
            pw[r] = a.codes[r] + (size_t)row * a.row_bytes + t * (4u * BITS / kUnits);
            ps[r] = a.scales[r] + (size_t)row * sgroups;
        }
    };
    auto begin = [&]() {
        const uint32_t n = ntiles * nspans;
        next = (uint32_t)((uint64_t)n * warp / nwarps);
        end = (uint32_t)((uint64_t)n * (warp + 1) / nwarps);
        load_tile = next / nspans;
        load_span = next - load_tile * nspans;
        at_tile();
    };
    struct Loaded { uint32_t w[2][BITS]; uint16_t sc[2][kUnits]; };
    uint32_t to_load = 0;
    auto load = [&](Loaded &l) {
        if (to_load >= end) return;
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int u = 0; u < kUnits; u++) {
                const uint8_t *p = pw[r] + load_span * (16u * BITS) + u * (U * BITS / 8);
                if constexpr (kWords == 1) {
                    l.w[r][u] = __ldg(reinterpret_cast<const uint32_t *>(p));
                } else if constexpr (kWords == 2) {
                    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
                    l.w[r][2 * u] = v.x; l.w[r][2 * u + 1] = v.y;
                } else {
#pragma unroll
                    for (int h = 0; h < kWords / 4; h++) {
                        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + h);
                        uint32_t *d = &l.w[r][u * kWords + 4 * h];
                        d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
                    }
                }
                const uint32_t at = load_span * kUnits + u;
                l.sc[r][u] = __ldg(ps[r] + (gunits == 1u ? at : at / gunits));
            }
        to_load++;
        if (++load_span == nspans) { load_span = 0; load_tile++; at_tile(); }
    };

    // codes and scales do not depend on the kernel before this one in the stream, the activations may
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    begin();
    to_load = next;
    Loaded buf[kSets];
#pragma unroll
    for (int d = 0; d < kSets - 1; d++) load(buf[d]);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t e = threadIdx.x; e < nspans * 16u * BT; e += blockDim.x) {
        const uint32_t tt = e & 3u, b = (e >> 2) % BT, i = (e >> 2) / BT & 3u, s = e / (16u * BT);
        xs[e] = b < a.batch ? piece_of<BITS, U>(reinterpret_cast<const uint16_t *>(a.x) + (size_t)b * a.K, s, i, tt) : make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();

    float tot[4];
    auto multiply = [&](const Loaded &l, uint32_t span) {
        const uint4 *xp = xs + (size_t)span * 16u * BT + g * 4u + t;
        // four registers of codes a row at a time, and their piece of the activations: two products, whose accumulators alternate, so
        // that consecutive ones do not wait for one another
        float c[4], d[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (BT == 8 || g < BT) q = xp[i * 4 * BT];
            uint32_t h0[4], h1[4];
            if constexpr (BITS == 4) {
                unpack_word<BITS, BF16>(l.w[0][i], h0);
                unpack_word<BITS, BF16>(l.w[1][i], h1);
            } else if constexpr (BITS == 2) {
                uint32_t e0[8], e1[8];
                unpack_word<BITS, BF16>(l.w[0][i / 2], e0);
                unpack_word<BITS, BF16>(l.w[1][i / 2], e1);
#pragma unroll
                for (int j = 0; j < 4; j++) { h0[j] = e0[4 * (i & 1) + j]; h1[j] = e1[4 * (i & 1) + j]; }
            } else {
                uint32_t e[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    unpack_word<BITS, BF16>(l.w[0][2 * i + j], e);
                    h0[2 * j] = e[0]; h0[2 * j + 1] = e[1];
                    unpack_word<BITS, BF16>(l.w[1][2 * i + j], e);
                    h1[2 * j] = e[0]; h1[2 * j + 1] = e[1];
                }
            }
            constexpr int kPieces = 4 / kUnits;                    // of a unit
            if (i % kPieces == 0) {
                mma_m16n8k16_first<BF16>(c, h0[0], h1[0], h0[1], h1[1], q.x, q.y);
                mma_m16n8k16_first<BF16>(d, h0[2], h1[2], h0[3], h1[3], q.z, q.w);
            } else {
                mma_m16n8k16<BF16>(c, h0[0], h1[0], h0[1], h1[1], q.x, q.y);
                mma_m16n8k16<BF16>(d, h0[2], h1[2], h0[3], h1[3], q.z, q.w);
            }
            if (i % kPieces == kPieces - 1) {
                const float fa = __half2float(__ushort_as_half(l.sc[0][i / kPieces])), fb = __half2float(__ushort_as_half(l.sc[1][i / kPieces]));
                tot[0] = fmaf(fa, c[0] + d[0], tot[0]); tot[1] = fmaf(fa, c[1] + d[1], tot[1]);
                tot[2] = fmaf(fb, c[2] + d[2], tot[2]); tot[3] = fmaf(fb, c[3] + d[3], tot[3]);
            }
        }
    };
    for (;;) {
        uint32_t span = next % nspans, part = 0;
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
        while (next < end) {
#pragma unroll
            for (int d = 0; d < kSets; d++) {                       // register sets in rotation: every index is static
                if (next >= end) break;
                load(buf[(d + kSets - 1) % kSets]);
                multiply(buf[d], span);
                next++;
                if (++span == nspans) { leave(); span = 0; }
            }
        }
        if (span) leave();
        __syncthreads();
        // every (tile, row of x, feature): the parts of the warps whose runs touch the tile, in their order
        const uint32_t n = ntiles * nspans;
        for (uint32_t i = threadIdx.x; i < ntiles * 8u * BT; i += blockDim.x) {
            const uint32_t f = i & 7u, b = (i >> 3) % BT, tile = i / (8u * BT), feature = (tile0 + tile) * 8u + f;
            if (feature >= a.N || b >= a.batch) continue;
            const uint32_t first = tile * nspans, behind = first + nspans;
            // the warp that has span s: the last w with n w / nwarps <= s
            uint32_t w = (uint32_t)(((uint64_t)(first + 1) * nwarps - 1) / n);
            float gs = 0.0f, us = 0.0f;
            for (uint32_t from = (uint32_t)((uint64_t)n * w / nwarps); w < nwarps && from < behind; w++) {
                const uint32_t to = (uint32_t)((uint64_t)n * (w + 1) / nwarps);
                if (to > from) {
                    const uint32_t part_of = tile - from / nspans;
                    gs += red[w][part_of][f][b];
                    us += red[w][part_of][8 + f][b];
                }
                from = to;
            }
            if (a.bias[0]) gs += __ldg(a.bias[0] + feature);
            if (a.bias[1]) us += __ldg(a.bias[1] + feature);
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
        ntiles = min(last - tile0, 2u * nwarps);
        __syncthreads();
        begin();
        to_load = next;
#pragma unroll
        for (int d = 0; d < kSets - 1; d++) load(buf[d]);
    }
}

std::atomic<int> g_warps{0}, g_ctas{0};        // 0: by shape

uint32_t rounded(uint32_t batch) { return batch <= 1 ? 1u : batch <= 2 ? 2u : batch <= 4 ? 4u : 8u; }
size_t rows_smem(uint32_t K, uint32_t bt, uint32_t warps) { return (size_t)K * bt * 2 + (size_t)warps * kParts * 16 * bt * 4; }

template <int BITS, bool BF16, int U>
void (*by_batch(uint32_t bt))(RowsArgs)
{
    return bt == 1 ? gated_rows_kernel<BITS, BF16, U, 1> : bt == 2 ? gated_rows_kernel<BITS, BF16, U, 2> : bt == 4 ? gated_rows_kernel<BITS, BF16, U, 4>
                                                                                                                   : gated_rows_kernel<BITS, BF16, U, 8>;
}

}  // namespace

void set_gated_rows(int warps, int ctas) { g_warps.store(warps); g_ctas.store(ctas); }

// Whole spans a row, whole units a group, activations that fit beside the warps' sums.
bool gated_rows_takes(const PackedPair &w, uint32_t batch)
{
    return batch <= 8 && product_takes(w, 2) && w.K % 128u == 0 && (w.bits != 2 || w.group % 64u == 0) && rows_smem(w.K, rounded(batch), kMostThreads / 32) <= 226u * 1024u;
}

int launch_gated_rows(const GatedCall &c, void *stream)
{
    RowsArgs a = {{c.w.codes[0], c.w.codes[1]}, {c.w.scales[0], c.w.scales[1]}, {c.bias[0], c.bias[1]}, c.x, c.h, {c.keep.v[0], c.keep.v[1]},
                  c.w.N, c.w.K, c.w.group, c.w.row_bytes, c.M, (c.w.N + 7u) / 8u, c.act, c.keep.form == kKeepF32};
    const uint32_t bt = rounded(c.M), unit = a.group % 128u == 0 ? 128u : a.group % 64u == 0 ? 64u : 32u;
    void (*kern)(RowsArgs) = nullptr;
#define EOQ_ROWS(B, U) (c.dtype == EOQ_B200_BF16 ? by_batch<B, true, U>(bt) : by_batch<B, false, U>(bt))
    if (c.w.bits == 4) kern = unit == 128u ? EOQ_ROWS(4, 128) : unit == 64u ? EOQ_ROWS(4, 64) : EOQ_ROWS(4, 32);
    else if (c.w.bits == 2) kern = unit == 128u ? EOQ_ROWS(2, 128) : EOQ_ROWS(2, 64);
    else kern = unit == 128u ? EOQ_ROWS(8, 128) : unit == 64u ? EOQ_ROWS(8, 64) : EOQ_ROWS(8, 32);
#undef EOQ_ROWS
    const uint32_t sms = (uint32_t)device_sm_count();
    uint32_t warps = g_warps.load() ? (uint32_t)g_warps.load() : 12u, per_sm = g_ctas.load() ? (uint32_t)g_ctas.load() : 2u;
    const size_t smem = rows_smem(a.K, bt, warps);
    static std::mutex mu;                          // kernels whose shared-memory limit has been raised, per device
    static std::vector<std::pair<const void *, int>> raised;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    {
        std::lock_guard<std::mutex> lock(mu);
        const std::pair<const void *, int> key(reinterpret_cast<const void *>(kern), dev);
        if (std::find(raised.begin(), raised.end(), key) == raised.end()) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            if (e != cudaSuccess) return (int)e;
            raised.push_back(key);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min(a.tiles, sms * per_sm));
    cfg.blockDim = dim3(warps * 32u);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launches();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, a);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

}  // namespace eoq
