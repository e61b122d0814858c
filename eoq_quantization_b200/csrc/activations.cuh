// Activations of a gated block and their derivatives in fp32, the power of two that brings a row into fp16's range, and the 8-bit
// storage of a block.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "gated.h"

namespace eoq {

__device__ __forceinline__ float bias_at(const void *p, uint32_t n, int dtype)
{
    if (!p) return 0.0f;
    if (dtype == EOQ_B200_F32) return __ldg(reinterpret_cast<const float *>(p) + n);
    const uint16_t b = __ldg(reinterpret_cast<const uint16_t *>(p) + n);
    return dtype == EOQ_B200_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
}

// value and derivative: silu g s(g), s(g) (1 + g (1 - s(g))); gelu g P(g), P(g) + g p(g) of the normal distribution; gelu_tanh with
// P(g) = (1 + tanh(sqrt(2 / pi) (g + 0.044715 g^3))) / 2
__device__ __forceinline__ void activation_and_slope(float g, int act, float &value, float &slope)
{
    if (act == kActSilu) {
        const float s = __fdividef(1.0f, 1.0f + __expf(-g));      // (0 where the sum is beyond 2^126)
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if (act == kActGelu) {
        const float p = 0.5f * (1.0f + erff(g * 0.70710678f));
        value = g * p;
        slope = p + g * __expf(-0.5f * g * g) * 0.39894228f;
    } else {
        const float t = tanhf(0.79788456f * (g + 0.044715f * g * g * g)), p = 0.5f * (1.0f + t);
        value = g * p;
        slope = p + g * 0.5f * (1.0f - t * t) * 0.79788456f * (1.0f + 0.134145f * fminf(g * g, 1e30f));      // (not zero times infinity)
    }
}

__device__ __forceinline__ float activation(float g, int act)
{
    float value, slope;
    activation_and_slope(g, act, value, slope);
    return value;
}

__device__ __forceinline__ float finite_magnitude(float v) { return fabsf(v) < __int_as_float(0x7f800000) ? fabsf(v) : 0.0f; }

// e with 2^14 <= most 2^e < 2^15, within what a float holds; rows without a finite value other than zero stay as they are
__device__ __forceinline__ int half_exponent(float most) { return most > 0.0f ? min(120, 141 - (int)(__float_as_uint(most) >> 23)) : 0; }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// A block's scale and codes from the bits of its largest magnitude (as a whole number, so that NaN is above infinity).  A code is
// the quotient 127 v / largest to the nearest whole number: the product with the inverse, corrected by what is left of 127 v
// (Markstein's step), so that quotients halfway between two codes, which 16-bit values often have, come out as such and go to
// the even one.
struct Storer {
    float scale, most, inv, up;
    __device__ __forceinline__ explicit Storer(uint32_t bits)
    {
        const float v = __uint_as_float(bits);
        const bool fine = bits < 0x7f800000u, zero = v < 1e-30f;
        // v / 127 by the reciprocal and one such step: the rounded quotient for all 2^23 significands (compared with a division's)
        const float r = 1.0f / 127.0f, q = v * r;
        scale = !fine ? __uint_as_float(0x7fffffffu) : zero ? 0.0f : fmaf(fmaf(-q, 127.0f, v), r, q);
        // in 128ths where 127 v or the products would leave the range; a factor of zero makes every code zero
        up = !fine || zero ? 0.0f : v > 1e36f ? 0.9921875f : 127.0f;
        most = !fine || zero ? 0.0f : v > 1e36f ? v * 0.0078125f : v;
        inv = !fine || zero ? 0.0f : __fdividef(1.0f, most);       // (two units off at most, which the step makes good)
    }
    // in the low byte: beside 1.5 x 2^23 a whole number is all that a sum's rounding leaves (a conversion takes four times an addition's slots)
    __device__ __forceinline__ uint32_t code(float v) const
    {
        const float w = up == 0.0f ? 0.0f : v * up, t = w * inv;
        return __float_as_uint(fmaf(fmaf(-t, most, w), inv, t) + 12582912.0f);
    }
};

}  // namespace eoq
