// The gated feed-forward block h = act(x Wg^T + bg) * (x Wu^T + bu) and its backward pass on weights that stay packed: the forms
// for any shape and type, and the passes over activations (gradients of the gate, sums over rows, 8-bit storage).
#include "gated.h"

#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "activations.cuh"

namespace eoq {
namespace {

__device__ __forceinline__ float load_as_float(const void *p, size_t i, int dtype)
{
    if (dtype == EOQ_B200_F32) return __ldg(reinterpret_cast<const float *>(p) + i);
    const uint16_t b = __ldg(reinterpret_cast<const uint16_t *>(p) + i);
    return dtype == EOQ_B200_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
}
__device__ __forceinline__ void store_from_float(void *p, size_t i, float v, int dtype)
{
    if (dtype == EOQ_B200_F32) reinterpret_cast<float *>(p)[i] = v;
    else if (dtype == EOQ_B200_F16) reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// Eight values in a row of a type, as they lie in memory: four words, or eight.
template <int DTYPE> struct Raw8 { uint4 v[DTYPE == EOQ_B200_F32 ? 2 : 1]; };

template <int DTYPE>
__device__ __forceinline__ Raw8<DTYPE> load8(const void *p, size_t i)
{
    Raw8<DTYPE> r;
    const uint4 *at = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(p) + i * (DTYPE == EOQ_B200_F32 ? 4 : 2));
    r.v[0] = __ldg(at);
    if constexpr (DTYPE == EOQ_B200_F32) r.v[1] = __ldg(at + 1);
    return r;
}
__device__ __forceinline__ float2 pair_of(uint32_t w, bool half)
{
    if (half) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <int DTYPE>
__device__ __forceinline__ void values_of(const Raw8<DTYPE> &r, float (&f)[8])
{
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
    if constexpr (DTYPE == EOQ_B200_F32) {
        const uint32_t u[4] = {r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
        for (int j = 0; j < 4; j++) { f[j] = __uint_as_float(w[j]); f[4 + j] = __uint_as_float(u[j]); }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) { const float2 p = pair_of(w[j], DTYPE == EOQ_B200_F16); f[2 * j] = p.x; f[2 * j + 1] = p.y; }
    }
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
template <int DTYPE>
__device__ __forceinline__ void store8(void *p, size_t i, const float (&f)[8])
{
    uint4 *at = reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(p) + i * (DTYPE == EOQ_B200_F32 ? 4 : 2));
    if constexpr (DTYPE == EOQ_B200_F32) {
        at[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        at[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    } else if constexpr (DTYPE == EOQ_B200_F16) {
        at[0] = make_uint4(half_pair(f[0], f[1]), half_pair(f[2], f[3]), half_pair(f[4], f[5]), half_pair(f[6], f[7]));
    } else {
        at[0] = make_uint4(bf16_pair(f[0], f[1]), bf16_pair(f[2], f[3]), bf16_pair(f[4], f[5]), bf16_pair(f[6], f[7]));
    }
}

// The largest value of a CTA's threads, in all of them.
__device__ __forceinline__ float largest_of(float v, float *part)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    if ((threadIdx.x & 31u) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (uint32_t w = 0; w < blockDim.x / 32u; w++) v = fmaxf(v, part[w]);
    __syncthreads();
    return v;
}

// Weight (n, k) in fp32: any width and any group of the flattened matrix, rows that end inside a group among them.
__device__ __forceinline__ float weight_at(const PackedPair &w, int which, uint32_t n, uint32_t k, bool whole, uint32_t gk)
{
    const uint8_t *row = w.codes[which] + (size_t)n * w.row_bytes;
    int q;
    if (w.bits == 4) q = (int)((__ldg(row + (k >> 1)) >> (4u * (k & 1u))) & 15u) - 7;
    else if (w.bits == 2) q = (int)((__ldg(row + (k >> 2)) >> (2u * (k & 3u))) & 3u) - 1;
    else q = (int)(int8_t)__ldg(row + k);
    const size_t g = whole ? (size_t)n * (w.K / w.group) + gk : ((size_t)n * w.K + k) / w.group;
    return (float)q * __half2float(__ushort_as_half(__ldg(w.scales[which] + g)));
}

// ---------------------------------------------------------------------------
// h for any shape and type, fp32 throughout: 64 tokens x 32 features a CTA, 32 columns of x and of both weights in shared memory
// at a time.  For what the tensor-core forms do not take.  Bound by instruction issue (a code takes some twenty to be found and
// scaled, whatever the tokens).
// ---------------------------------------------------------------------------
constexpr uint32_t kTokens = 64, kFeatures = 32, kStep = 32;

__global__ void __launch_bounds__(256) gated_general_kernel(const GatedCall c)
{
    __shared__ float xs[kStep][kTokens + 1], ws[2][kStep][kFeatures + 1];
    const PackedPair &w = c.w;
    const uint32_t n0 = blockIdx.x * kFeatures, tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    const bool whole = w.K % w.group == 0;
    const uint32_t tiles = (c.M + kTokens - 1) / kTokens;
    for (uint32_t tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
        const uint32_t m0 = tile * kTokens;
        float acc[2][4][2] = {};
        for (uint32_t k0 = 0; k0 < w.K; k0 += kStep) {
            for (uint32_t i = threadIdx.x; i < kStep * kTokens; i += 256u) {
                const uint32_t k = k0 + i % kStep, m = m0 + i / kStep;
                xs[i % kStep][i / kStep] = k < w.K && m < c.M ? load_as_float(c.x, (size_t)m * w.K + k, c.dtype) : 0.0f;
            }
            for (uint32_t i = threadIdx.x; i < 2u * kStep * kFeatures; i += 256u) {
                const uint32_t which = i / (kStep * kFeatures), j = i % (kStep * kFeatures), k = k0 + j % kStep, n = n0 + j / kStep;
                ws[which][j % kStep][j / kStep] = k < w.K && n < w.N ? weight_at(w, which, n, k, whole, whole ? k / w.group : 0u) : 0.0f;
            }
            __syncthreads();
            const uint32_t steps = min(kStep, w.K - k0);      // (past the last column a NaN of x would meet zeros)
            for (uint32_t k = 0; k < steps; k++) {
                float a[4];
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = xs[k][ty + 16 * i];
#pragma unroll
                for (int which = 0; which < 2; which++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float b = ws[which][k][tx + 16 * j];
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[which][i][j] = fmaf(a[i], b, acc[which][i][j]);
                    }
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (m >= c.M || n >= w.N) continue;
                const float g = acc[0][i][j] + bias_at(c.bias[0], n, c.bias_dtype), u = acc[1][i][j] + bias_at(c.bias[1], n, c.bias_dtype);
                const size_t at = (size_t)m * w.N + n;
                store_from_float(c.h, at, activation(g, c.act) * u, c.dtype);
                if (c.keep.form == kKeepFull || c.keep.form == kKeepF32) {
                    const int type = c.keep.form == kKeepF32 ? EOQ_B200_F32 : c.dtype;
                    store_from_float(c.keep.v[0], at, g, type);
                    store_from_float(c.keep.v[1], at, u, type);
                }
            }
    }
}

// ---------------------------------------------------------------------------
// dx = dy W for any shape and type, fp32 throughout: 64 tokens x 64 columns a CTA, the weights' rows split over gridDim.z, each
// split's sums to its own part of the scratch, which the second kernel adds up in order.
// ---------------------------------------------------------------------------
constexpr uint32_t kGradStep = 16;

struct GradArgs {
    PackedPair w;
    const void *dy[2];
    float *partial;              // [splits][M][K]
    uint32_t M, nw, per;         // rows of a weight (of both, one behind the other) a split takes
    int dy_dtype;
};

__global__ void __launch_bounds__(256) input_grad_general_kernel(const GradArgs a)
{
    __shared__ float ds[kGradStep][kTokens + 1], ws[kGradStep][64 + 1];
    const PackedPair &w = a.w;
    const uint32_t k0 = blockIdx.x * 64u, tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    const bool whole = w.K % w.group == 0;
    const uint32_t tiles = (a.M + kTokens - 1) / kTokens;
    const uint64_t all = (uint64_t)w.N * a.nw, r0 = (uint64_t)blockIdx.z * a.per, r1 = min(all, r0 + a.per);
    for (uint32_t tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
        const uint32_t m0 = tile * kTokens;
        float acc[4][4] = {};
        for (uint64_t r = r0; r < r1; r += kGradStep) {
            for (uint32_t i = threadIdx.x; i < kGradStep * kTokens; i += 256u) {
                const uint64_t at = r + i % kGradStep;
                const uint32_t m = m0 + i / kGradStep, which = at >= w.N, n = (uint32_t)(at - (which ? w.N : 0u));
                ds[i % kGradStep][i / kGradStep] = at < r1 && m < a.M ? load_as_float(a.dy[which], (size_t)m * w.N + n, a.dy_dtype) : 0.0f;
            }
            for (uint32_t i = threadIdx.x; i < kGradStep * 64u; i += 256u) {
                const uint64_t at = r + i / 64u;
                const uint32_t k = k0 + i % 64u, which = at >= w.N, n = (uint32_t)(at - (which ? w.N : 0u));
                ws[i / 64u][i % 64u] = at < r1 && k < w.K ? weight_at(w, which, n, k, whole, whole ? k / w.group : 0u) : 0.0f;
            }
            __syncthreads();
            const uint32_t steps = (uint32_t)min((uint64_t)kGradStep, r1 - r);
            for (uint32_t s = 0; s < steps; s++) {
                float d[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; i++) { d[i] = ds[s][ty + 16 * i]; b[i] = ws[s][tx + 16 * i]; }
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][j] = fmaf(d[i], b[j], acc[i][j]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t m = m0 + ty + 16 * i, k = k0 + tx + 16 * j;
                if (m < a.M && k < w.K) a.partial[((size_t)blockIdx.z * a.M + m) * w.K + k] = acc[i][j];
            }
    }
}

__global__ void __launch_bounds__(256) add_partials_kernel(const float *partial, uint32_t splits, size_t n, void *out, int dtype)
{
    for (size_t i = (size_t)blockIdx.x * 256u + threadIdx.x; i < n; i += (size_t)gridDim.x * 256u) {
        float v = 0.0f;
        for (uint32_t s = 0; s < splits; s++) v += partial[s * n + i];
        store_from_float(out, i, v, dtype);
    }
}

uint32_t grad_splits(const PackedPair &w, uint32_t M)
{
    const uint64_t ctas = (uint64_t)((w.K + 63u) / 64u) * ((M + kTokens - 1) / kTokens);
    return (uint32_t)std::min<uint64_t>(std::max<uint64_t>(1, 592 / std::max<uint64_t>(1, ctas)), std::max(1u, w.N / 64u));
}

// ---------------------------------------------------------------------------
// Gradients of the gate, a row a CTA: what the products' backward takes, in fp32, or as fp16 with one power of two for both
// halves of a row, so that the largest is at 2^14 .. 2^15 and a gradient of any size keeps eleven bits (bf16 would keep eight).
// The row is gone over twice then, first for its largest value.  Bound by the exponentials at two passes.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void set_zeros(const Zeros &z)
{
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < z.n; i += gridDim.x * blockDim.x) z.p[i] = 0u;
}

struct GateGradArgs {
    Kept k;
    const void *dh;
    float *out32[2];
    __half *half;                // [2][M][pitch]
    float *factor;
    uint32_t M, N, pitch;
    int dtype, act;
    Zeros zeros;
};

__device__ __forceinline__ void kept_at(const GateGradArgs &a, uint32_t m, uint32_t n, float &g, float &u)
{
    const size_t at = (size_t)m * a.N + n;
    if (a.k.form == kKeep8bit) {
        const size_t s = (size_t)m * ((a.N + kStoreBlock - 1) / kStoreBlock) + n / kStoreBlock;
        g = (float)__ldg(reinterpret_cast<const int8_t *>(a.k.v[0]) + at) * __ldg(a.k.scale[0] + s);
        u = (float)__ldg(reinterpret_cast<const int8_t *>(a.k.v[1]) + at) * __ldg(a.k.scale[1] + s);
    } else {
        g = load_as_float(a.k.v[0], at, a.dtype);
        u = load_as_float(a.k.v[1], at, a.dtype);
    }
}

__global__ void __launch_bounds__(512) gate_grad_kernel(const GateGradArgs a)
{
    __shared__ float part[16];
    set_zeros(a.zeros);
    for (uint32_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        auto at = [&](uint32_t n, float &dg, float &du) {
            float g, u, act, slope;
            kept_at(a, m, n, g, u);
            activation_and_slope(g, a.act, act, slope);
            const float d = load_as_float(a.dh, (size_t)m * a.N + n, a.dtype);
            dg = d * u * slope;
            du = d * act;
        };
        if (!a.half) {
            for (uint32_t n = threadIdx.x; n < a.N; n += blockDim.x) {
                float dg, du;
                at(n, dg, du);
                a.out32[0][(size_t)m * a.N + n] = dg;
                a.out32[1][(size_t)m * a.N + n] = du;
            }
            continue;
        }
        float most = 0.0f;
        for (uint32_t n = threadIdx.x; n < a.N; n += blockDim.x) {
            float dg, du;
            at(n, dg, du);
            most = fmaxf(most, fmaxf(finite_magnitude(dg), finite_magnitude(du)));
        }
        const int e = half_exponent(largest_of(most, part));
        const float up = power_of_two(e);
        if (threadIdx.x == 0) a.factor[m] = power_of_two(-e);
        for (uint32_t n = threadIdx.x; n < a.pitch; n += blockDim.x) {
            float dg = 0.0f, du = 0.0f;
            if (n < a.N) at(n, dg, du);
            a.half[(size_t)m * a.pitch + n] = __float2half_rn(dg * up);
            a.half[((size_t)a.M + m) * a.pitch + n] = __float2half_rn(du * up);
        }
    }
}

__global__ void __launch_bounds__(256) gate_apply_kernel(const float *__restrict__ g, const float *__restrict__ u, size_t count, int act, void *__restrict__ h, int dtype)
{
    for (size_t i = (size_t)blockIdx.x * 256u + threadIdx.x; i < count; i += (size_t)gridDim.x * 256u)
        store_from_float(h, i, activation(g[i], act) * u[i], dtype);
}

// The same to fp16 where rows are multiples of eight values and aligned: a row's inputs are read once and stay in registers, as they
// came (KEEP8: with their scales), eight values a thread ROUNDS times; the gradients are computed twice.  (A bound of the largest that takes no
// exponential, |dh| max(1.13 |u|, |g|), is any number of bits above it where all gates that dh meets are closed: at silu(-25) it left
// the row's gradients four bits.)
template <int DTYPE, bool KEEP8, int ROUNDS>
__global__ void __launch_bounds__(512) gate_grad_rows_kernel(const GateGradArgs a)
{
    __shared__ float part[16];
    set_zeros(a.zeros);
    struct Kept8 { uint2 v; float s; };
    struct Kept16 { Raw8<DTYPE> v; };
    using K = std::conditional_t<KEEP8, Kept8, Kept16>;
    auto load_kept = [&](int which, size_t m, uint32_t n) {
        K k;
        if constexpr (KEEP8) {
            k.v = __ldg(reinterpret_cast<const uint2 *>(reinterpret_cast<const int8_t *>(a.k.v[which]) + m * a.N + n));
            k.s = __ldg(a.k.scale[which] + m * ((a.N + kStoreBlock - 1) / kStoreBlock) + n / kStoreBlock);
        } else {
            k.v = load8<DTYPE>(a.k.v[which], m * a.N + n);
        }
        return k;
    };
    auto kept_values = [&](const K &k, float (&f)[8]) {
        if constexpr (KEEP8) {
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = (float)(int8_t)((j < 4 ? k.v.x : k.v.y) >> (8 * (j & 3))) * k.s;
        } else {
            values_of<DTYPE>(k.v, f);
        }
    };
    // eight values of both gradients
    auto gradients = [&](const Raw8<DTYPE> &rd, const K &rg, const K &ru, float (&g)[8], float (&u)[8]) {
        float d[8];
        values_of<DTYPE>(rd, d);
        kept_values(rg, g);
        kept_values(ru, u);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float value, slope;
            activation_and_slope(g[j], a.act, value, slope);
            g[j] = d[j] * u[j] * slope;
            u[j] = d[j] * value;
        }
    };
    for (uint32_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        Raw8<DTYPE> rd[ROUNDS];
        K rg[ROUNDS], ru[ROUNDS];
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t n = (r * 512u + threadIdx.x) * 8u;
            if (n >= a.N) continue;
            rd[r] = load8<DTYPE>(a.dh, (size_t)m * a.N + n);
            rg[r] = load_kept(0, m, n);
            ru[r] = load_kept(1, m, n);
        }
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t n = (r * 512u + threadIdx.x) * 8u;
            if (n >= a.N) continue;
            float g[8], u[8];
            gradients(rd[r], rg[r], ru[r], g, u);
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, fmaxf(finite_magnitude(g[j]), finite_magnitude(u[j])));
        }
        const int e = half_exponent(largest_of(most, part));
        const float up = power_of_two(e);
        if (threadIdx.x == 0) a.factor[m] = power_of_two(-e);
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t n = (r * 512u + threadIdx.x) * 8u;
            if (n >= a.N) continue;
            float g[8], u[8];
            gradients(rd[r], rg[r], ru[r], g, u);
#pragma unroll
            for (int j = 0; j < 8; j++) { g[j] *= up; u[j] *= up; }
            store8<EOQ_B200_F16>(a.half, (size_t)m * a.pitch + n, g);
            store8<EOQ_B200_F16>(a.half, ((size_t)a.M + m) * a.pitch + n, u);
        }
    }
}

// Sums over the rows in two steps, so that their order is fixed: 256 rows a CTA and column, then the parts in order.
constexpr uint32_t kSumRows = 256;

struct SumArgs {
    const float *in32[2];
    const __half *half;
    const float *factor;
    float *part;                 // [chunks][2][N]
    void *out[2];
    uint32_t M, N, pitch, chunks;
    int dtype;                   // of out
};

__global__ void __launch_bounds__(256) column_parts_kernel(const SumArgs a)
{
    __shared__ float2 sums[8][32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, n = blockIdx.x * 64u + lane * 2u, which = blockIdx.z;
    for (uint32_t chunk = blockIdx.y; chunk < a.chunks; chunk += gridDim.y) {
        float2 v = make_float2(0.0f, 0.0f);
        const uint32_t last = min(a.M, (chunk + 1) * kSumRows);
        if (n < a.N) {
#pragma unroll 4
            for (uint32_t m = chunk * kSumRows + warp; m < last; m += 8u) {
                if (a.half) {              // (rows are padded to eight)
                    const float f = __ldg(a.factor + m);
                    const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(a.half + ((size_t)which * a.M + m) * a.pitch + n));
                    v.x = fmaf(p.x, f, v.x);
                    v.y = fmaf(p.y, f, v.y);
                } else {
                    v.x += a.in32[which][(size_t)m * a.N + n];
                    if (n + 1 < a.N) v.y += a.in32[which][(size_t)m * a.N + n + 1];
                }
            }
        }
        sums[warp][lane] = v;
        __syncthreads();
        if (warp == 0 && n < a.N) {
            for (int w = 1; w < 8; w++) { v.x += sums[w][lane].x; v.y += sums[w][lane].y; }
            float *to = a.part + ((size_t)chunk * 2 + which) * a.N + n;
            to[0] = v.x;
            if (n + 1 < a.N) to[1] = v.y;
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) column_sums_kernel(const SumArgs a)
{
    const uint32_t n = blockIdx.x * 256u + threadIdx.x, which = blockIdx.y;
    if (n >= a.N || !a.out[which]) return;
    float v = 0.0f;
    for (uint32_t c = 0; c < a.chunks; c++) v += a.part[((size_t)c * 2 + which) * a.N + n];
    store_from_float(a.out[which], n, v, a.dtype);
}

// bf16 or fp16 rows of multiples of eight values, aligned: read once, kept in registers.
template <int DTYPE, int ROUNDS>
__global__ void __launch_bounds__(256) rows_to_half_vector_kernel(const void *__restrict__ x, uint32_t M, uint32_t K, __half *__restrict__ out, float *__restrict__ factor, const Zeros zeros)
{
    __shared__ float part[8];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    set_zeros(zeros);
    for (uint32_t m = blockIdx.x; m < M; m += gridDim.x) {
        Raw8<DTYPE> raw[ROUNDS];
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t k = (r * 256u + threadIdx.x) * 8u;
            if (k < K) raw[r] = load8<DTYPE>(x, (size_t)m * K + k);
        }
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            float f[8];
            if ((r * 256u + threadIdx.x) * 8u >= K) continue;
            values_of<DTYPE>(raw[r], f);
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, finite_magnitude(f[j]));
        }
        const int e = half_exponent(largest_of(most, part));
        const float up = power_of_two(e);
        if (threadIdx.x == 0) factor[m] = power_of_two(-e);
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
            const uint32_t k = (r * 256u + threadIdx.x) * 8u;
            if (k >= K) continue;
            float f[8];
            values_of<DTYPE>(raw[r], f);
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] *= up;
            store8<EOQ_B200_F16>(out, (size_t)m * K + k, f);
        }
    }
}

__global__ void __launch_bounds__(256) rows_to_half_kernel(const void *__restrict__ x, int dtype, uint32_t M, uint32_t K, uint32_t pitch, __half *__restrict__ out,
                                                           float *__restrict__ factor, const Zeros zeros)
{
    __shared__ float part[8];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    set_zeros(zeros);
    for (uint32_t m = blockIdx.x; m < M; m += gridDim.x) {
        float most = 0.0f;
        for (uint32_t k0 = threadIdx.x; k0 < K; k0 += 8u * 256u) {       // eight requested together; past the row's end its last value again
            float v[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) v[j] = load_as_float(x, (size_t)m * K + min(k0 + j * 256u, K - 1u), dtype);
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) most = fmaxf(most, finite_magnitude(v[j]));
        }
        const int e = half_exponent(largest_of(most, part));
        const float up = power_of_two(e);
        if (threadIdx.x == 0) factor[m] = power_of_two(-e);
        for (uint32_t k0 = threadIdx.x; k0 < pitch; k0 += 8u * 256u) {
            float v[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) v[j] = load_as_float(x, (size_t)m * K + min(k0 + j * 256u, K - 1u), dtype);
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const uint32_t k = k0 + j * 256u;
                if (k < pitch) out[(size_t)m * pitch + k] = __float2half_rn(k < K ? v[j] * up : 0.0f);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Activations to 8 bits and back: blocks of 64 values of a row, code = round(127 x / largest magnitude), half to even, and the
// scale largest / 127 in fp32, which half an activation's exponent range would not fit in 16 bits.  A warp takes four blocks, eight
// lanes each, eight values a lane.  A block that holds a NaN or an infinity stands for NaN throughout, so that it shows; one
// whose largest is below 1e-30 for zeros (127 / largest would be infinite at 3.7e-37).  2048 x 11008 bf16: to codes 20.4 us, 3.4 TB/s,
// for which instruction slots stand in the way (fp32 of twice the bytes takes as long an element), and back 12.4 us, 5.5 TB/s: HBM.
// ---------------------------------------------------------------------------
// VEC: rows are multiples of eight values and 16-byte aligned, a lane's eight lie together; else they are eight apart.
template <int DTYPE, bool VEC>
__global__ void __launch_bounds__(256) store_8bit_kernel(const void *__restrict__ x, size_t M, uint32_t N, int8_t *__restrict__ codes, float *__restrict__ scales)
{
    const uint32_t per_row = (N + kStoreBlock - 1) / kStoreBlock, lane8 = threadIdx.x & 7u;
    // a warp's turns: four blocks of one row, `fours` such to a row; on by `warps` of them without dividing again
    const uint32_t fours = (per_row + 3u) / 4u, warps = gridDim.x * 8u, on_m = warps / fours, on_f = warps - on_m * fours;
    const uint32_t t = blockIdx.x * 8u + (threadIdx.x >> 5);
    size_t m = t / fours;
    uint32_t f = t % fours;
    auto first_of = [&](uint32_t f) { return (f * 4u + ((threadIdx.x & 31u) >> 3)) * kStoreBlock; };
    auto fetch = [&](size_t m, uint32_t f) {
        Raw8<DTYPE> raw = {};
        if (VEC && m < M && first_of(f) + lane8 * 8u < N) raw = load8<DTYPE>(x, m * N + first_of(f) + lane8 * 8u);
        return raw;
    };
    Raw8<DTYPE> raw = fetch(m, f);
    while (m < M) {
        // the next turn's values are on their way while this one's are made into codes
        size_t nm = m + on_m;
        uint32_t nf = f + on_f;
        if (nf >= fours) { nf -= fours; nm++; }
        const Raw8<DTYPE> soon = fetch(nm, nf);
        const uint32_t first = first_of(f);
        float v[8] = {};
        if constexpr (VEC) {
            values_of<DTYPE>(raw, v);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) if (first + j * 8u + lane8 < N) v[j] = load_as_float(x, m * N + first + j * 8u + lane8, DTYPE);
        }
        uint32_t most = 0u;
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);      // as whole numbers: infinity and then NaN are the largest
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
        const Storer to(most);
        if (first < N && lane8 == 0) scales[m * per_row + first / kStoreBlock] = to.scale;
        if constexpr (VEC) {
            if (first + lane8 * 8u < N) {
                uint32_t p[2];
#pragma unroll
                for (int j = 0; j < 2; j++)
                    p[j] = __byte_perm(__byte_perm(to.code(v[4 * j]), to.code(v[4 * j + 1]), 0x0040), __byte_perm(to.code(v[4 * j + 2]), to.code(v[4 * j + 3]), 0x0040), 0x5410);
                *reinterpret_cast<uint2 *>(codes + m * N + first + lane8 * 8u) = make_uint2(p[0], p[1]);
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) if (first + j * 8u + lane8 < N) codes[m * N + first + j * 8u + lane8] = (int8_t)to.code(v[j]);
        }
        m = nm; f = nf; raw = soon;
    }
}

// VEC: eight values a thread (a row's eights are whole and lie in one block).
template <int DTYPE, bool VEC>
__global__ void __launch_bounds__(256) load_8bit_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scales, size_t M, uint32_t N, void *__restrict__ y)
{
    const uint32_t per_row = (N + kStoreBlock - 1) / kStoreBlock, width = VEC ? N / 8u : N;
    const size_t count = M * width;
    for (size_t i = (size_t)blockIdx.x * 256u + threadIdx.x; i < count; i += (size_t)gridDim.x * 256u) {
        const size_t m = count <= 0xffffffffu ? (uint32_t)i / width : i / width;
        const uint32_t n = (uint32_t)(i - m * width) * (VEC ? 8u : 1u);
        const float s = __ldg(scales + m * per_row + n / kStoreBlock);
        if constexpr (VEC) {
            const uint2 w = __ldg(reinterpret_cast<const uint2 *>(codes) + i);
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = (float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * s;
            store8<DTYPE>(y, i * 8u, f);
        } else {
            store_from_float(y, i, (float)codes[i] * s, DTYPE);
        }
    }
}

uint32_t ctas_for(size_t work, uint32_t per) { return (uint32_t)std::min<size_t>((work + per - 1) / per, (size_t)device_sm_count() * 16u); }

}  // namespace

static bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int launch_gated_general(const GatedCall &c, void *stream)
{
    const dim3 grid((c.w.N + kFeatures - 1) / kFeatures, std::min((c.M + kTokens - 1) / kTokens, 65535u));
    gated_general_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(c);
    count_launch();
    return (int)cudaGetLastError();
}

size_t input_grad_general_scratch(const PackedPair &w, uint32_t M) { return (size_t)grad_splits(w, M) * M * w.K * 4; }

int launch_input_grad_general(const PackedPair &w, int nw, const void *const dy[2], int dy_dtype, uint32_t M, void *scratch, void *dx, int dtype, void *stream)
{
    cudaStream_t st = (cudaStream_t)stream;
    const uint32_t splits = grad_splits(w, M);
    GradArgs a = {w, {dy[0], nw > 1 ? dy[1] : dy[0]}, (float *)scratch, M, (uint32_t)nw, 0, dy_dtype};
    a.per = (uint32_t)(((uint64_t)w.N * nw + splits - 1) / splits);
    input_grad_general_kernel<<<dim3((w.K + 63u) / 64u, std::min((M + kTokens - 1) / kTokens, 65535u), splits), 256, 0, st>>>(a);
    count_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    add_partials_kernel<<<ctas_for((size_t)M * w.K, 256u), 256, 0, st>>>(a.partial, splits, (size_t)M * w.K, dx, dtype);
    count_launch();
    return (int)cudaGetLastError();
}

__global__ void __launch_bounds__(256) zeros_kernel(const Zeros z)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    set_zeros(z);
}

int launch_zeros(Zeros zeros, void *stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min((zeros.n + 255u) / 256u, 64u));
    cfg.blockDim = dim3(256);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launches();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, zeros_kernel, zeros);
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_gate_apply(const float *g, const float *u, size_t count, int act, void *h, int dtype, void *stream)
{
    gate_apply_kernel<<<ctas_for(count, 256u), 256, 0, (cudaStream_t)stream>>>(g, u, count, act, h, dtype);
    count_launch();
    return (int)cudaGetLastError();
}

int launch_gate_grad(const Kept &k, const void *dh, int dtype, int act, uint32_t M, uint32_t N, float *out32[2], uint16_t *half, uint32_t pitch, float *factor,
                     Zeros zeros, void *stream)
{
    GateGradArgs a = {k, dh, {out32 ? out32[0] : nullptr, out32 ? out32[1] : nullptr}, (__half *)half, factor, M, N, pitch, dtype, act, zeros};
    const bool k8 = k.form == kKeep8bit;
    if (half && dtype != EOQ_B200_F32 && N % 8u == 0 && pitch == N && N <= 7u * 4096u && aligned(dh, 16) && aligned(k.v[0], 16) && aligned(k.v[1], 16) && aligned(half, 16)) {
#define EOQ_GATE(D, R) (k8 ? gate_grad_rows_kernel<D, true, R> : gate_grad_rows_kernel<D, false, R>)
#define EOQ_GATE_ROUNDS(D) (N <= 4096u ? EOQ_GATE(D, 1) : N <= 12288u ? EOQ_GATE(D, 3) : EOQ_GATE(D, 7))
        auto kern = dtype == EOQ_B200_F16 ? EOQ_GATE_ROUNDS(EOQ_B200_F16) : EOQ_GATE_ROUNDS(EOQ_B200_BF16);
#undef EOQ_GATE_ROUNDS
#undef EOQ_GATE
        kern<<<std::min(M, 65535u), N <= 4096u ? (N / 8u + 31u) / 32u * 32u : 512u, 0, (cudaStream_t)stream>>>(a);
    } else {
        gate_grad_kernel<<<std::min(M, 65535u), 512, 0, (cudaStream_t)stream>>>(a);
    }
    count_launch();
    return (int)cudaGetLastError();
}

static uint32_t sum_chunks(uint32_t M) { return (M + kSumRows - 1) / kSumRows; }
size_t column_sums_scratch(uint32_t M, uint32_t N) { return (size_t)sum_chunks(M) * 2 * N * 4; }

int launch_column_sums(const float *const in32[2], const uint16_t *half, uint32_t pitch, const float *factor, uint32_t M, uint32_t N, float *scratch, void *const out[2],
                       int dtype, void *stream)
{
    cudaStream_t st = (cudaStream_t)stream;
    SumArgs a = {{in32 ? in32[0] : nullptr, in32 ? in32[1] : nullptr}, (const __half *)half, factor, scratch, {out[0], out[1]}, M, N, pitch, sum_chunks(M), dtype};
    column_parts_kernel<<<dim3((N + 63u) / 64u, std::min(a.chunks, 65535u), 2), 256, 0, st>>>(a);
    count_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    column_sums_kernel<<<dim3((N + 255u) / 256u, 2), 256, 0, st>>>(a);
    count_launch();
    return (int)cudaGetLastError();
}

int launch_rows_to_half(const void *x, int dtype, uint32_t M, uint32_t K, uint32_t pitch, uint16_t *out, float *factor, Zeros zeros, void *stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min(M, 65535u));
    cfg.blockDim = dim3(256);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = programmatic_launches();
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e;
    if (dtype != EOQ_B200_F32 && K % 8u == 0 && pitch == K && K <= 16384u && aligned(x, 16)) {
#define EOQ_ROWS(D) (K <= 2048u ? rows_to_half_vector_kernel<D, 1> : K <= 4096u ? rows_to_half_vector_kernel<D, 2> : rows_to_half_vector_kernel<D, 8>)
        auto kern = dtype == EOQ_B200_F16 ? EOQ_ROWS(EOQ_B200_F16) : EOQ_ROWS(EOQ_B200_BF16);
#undef EOQ_ROWS
        e = cudaLaunchKernelEx(&cfg, kern, x, M, K, (__half *)out, factor, zeros);
    } else {
        e = cudaLaunchKernelEx(&cfg, rows_to_half_kernel, x, dtype, M, K, pitch, (__half *)out, factor, zeros);
    }
    count_launch();
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

int launch_store_8bit(const void *x, int dtype, size_t M, uint32_t N, int8_t *codes, float *scales, void *stream)
{
    const size_t turns = M * ((N + 4u * kStoreBlock - 1) / (4u * kStoreBlock));
    const bool vec = N % 8u == 0 && aligned(x, 16) && aligned(codes, 8);
    auto kern = dtype == EOQ_B200_F32 ? (vec ? store_8bit_kernel<EOQ_B200_F32, true> : store_8bit_kernel<EOQ_B200_F32, false>)
              : dtype == EOQ_B200_F16 ? (vec ? store_8bit_kernel<EOQ_B200_F16, true> : store_8bit_kernel<EOQ_B200_F16, false>)
                                      : (vec ? store_8bit_kernel<EOQ_B200_BF16, true> : store_8bit_kernel<EOQ_B200_BF16, false>);
    kern<<<ctas_for(turns, 8u), 256, 0, (cudaStream_t)stream>>>(x, M, N, codes, scales);
    count_launch();
    return (int)cudaGetLastError();
}

int launch_load_8bit(const int8_t *codes, const float *scales, size_t M, uint32_t N, void *y, int dtype, void *stream)
{
    const bool vec = N % 8u == 0 && aligned(y, 16) && aligned(codes, 8);
    auto kern = dtype == EOQ_B200_F32 ? (vec ? load_8bit_kernel<EOQ_B200_F32, true> : load_8bit_kernel<EOQ_B200_F32, false>)
              : dtype == EOQ_B200_F16 ? (vec ? load_8bit_kernel<EOQ_B200_F16, true> : load_8bit_kernel<EOQ_B200_F16, false>)
                                      : (vec ? load_8bit_kernel<EOQ_B200_BF16, true> : load_8bit_kernel<EOQ_B200_BF16, false>);
    kern<<<ctas_for(M * (vec ? N / 8u : N), 256u), 256, 0, (cudaStream_t)stream>>>(codes, scales, M, N, y);
    count_launch();
    return (int)cudaGetLastError();
}

}  // namespace eoq
