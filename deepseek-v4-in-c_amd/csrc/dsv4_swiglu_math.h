/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_swiglu_math.h - SwiGLU values in fp32 with a known error, and in fp64:
 *
 *   a = silu(min(g, limit)) * clamp(u, -limit, limit),  silu(g) = g / (1 + e^-g)
 *
 * (limit <= 0: no clamp). The int8 quantizer takes its values from here; a host
 * build (tests/test_swiglu_math.py) holds them to their bound.
 *
 * The fp32 value is within 8 x 2^-24 of the exact one, relatively (exp2 1 ulp, its
 * correction half, 1 + e half, reciprocal 1 ulp, two products half each), as long as
 * every step stays in fp32's normal range. Two kinds of gates leave it: below
 * -87.3 the reciprocal is subnormal or zero, and a subnormal gate's product with
 * it is. There |silu(g)| < 2^-119.4, and so is its error, whatever is computed. A
 * row's codes and scale need its values to 2^-21 of the largest, amax, so fp32
 * serves the row unless 2^-98 of its largest |u| passes amax. No clamp up to 2^32
 * lets that happen in a row whose amax is 2^-60 or more. */
#ifndef DSV4_SWIGLU_MATH_H
#define DSV4_SWIGLU_MATH_H

#include <math.h>

#if defined(__HIPCC__)
#define DSV4_SWIGLU_HD __device__ __forceinline__
#define DSV4_EXP2(x) __builtin_amdgcn_exp2f(x)
#define DSV4_RCP(x) __builtin_amdgcn_rcpf(x)
#define DSV4_MINIMUM(a, b) __builtin_elementwise_minimum(a, b)
#define DSV4_MAXIMUM(a, b) __builtin_elementwise_maximum(a, b)
#else
#define DSV4_SWIGLU_HD static inline
#define DSV4_EXP2(x) exp2f(x)
#define DSV4_RCP(x) (1.0f / (x))
#define DSV4_MINIMUM(a, b) ((a) > (b) ? (b) : (a))
#define DSV4_MAXIMUM(a, b) ((a) < (b) ? (b) : (a))
#endif

namespace dsv4_swiglu {

/* whether a clamp leaves room for up values that make a lost silu count */
DSV4_SWIGLU_HD bool unbounded(float limit) { return !(limit > 0.0f && limit <= 0x1p32f); }

/* whether the fp32 values decide a row: its largest is amax, NaN if any is, and its
 * largest |u| umax (0 with a bounding clamp) */
DSV4_SWIGLU_HD bool fp32_serves(float amax, float umax)
{
    return amax >= 0x1p-60f && amax <= 0x1p120f && umax * 0x1p-98f <= amax;
}

/* NaN stays NaN, through the three-operand minimum and maximum on the device */
DSV4_SWIGLU_HD void clamp(float &g, float &u, float limit)
{
    if (limit > 0.0f) {
        u = DSV4_MAXIMUM(DSV4_MINIMUM(u, limit), -limit);
        g = DSV4_MINIMUM(g, limit);
    }
}

DSV4_SWIGLU_HD double value64(float g, float u, float limit)
{
    clamp(g, u, limit);
    return (double)g / (1.0 + exp(-(double)g)) * (double)u;
}

/* Multiplications and additions round separately (-ffp-contract=off). */
DSV4_SWIGLU_HD float value32(float g, float u, float limit)
{
    clamp(g, u, limit);
    /* exp(-g) = 2^t (1 + ln 2 * r): t the rounded product with log2 e, r what
     * the rounding and log2 e's own last bits left. The correction is a factor
     * next to 1, so that where e passes fp32's range (a gate below -88.7) the sum
     * is infinite and the value 0: a term e * ln 2 * r beside e would be infinite
     * of either sign, and the NaN of their sum would cost the row fp64 values.
     * Infinite and NaN gates give NaN. */
    const float t = -g * 0x1.715476p+0f;
    const float r = fmaf(-g, 0x1.4ae0cp-26f, fmaf(-g, 0x1.715476p+0f, -t));
    const float e = DSV4_EXP2(t);
    return g * DSV4_RCP(fmaf(e, fmaf(r, 0x1.62e43p-1f, 1.0f), 1.0f)) * u;
}

} // namespace dsv4_swiglu

#endif /* DSV4_SWIGLU_MATH_H */
