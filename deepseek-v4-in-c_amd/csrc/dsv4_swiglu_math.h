/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_swiglu_math.h - SwiGLU values in fp32 with a known error, and in fp64:
 *
 *   a = silu(min(g, limit)) * clamp(u, -limit, limit),  silu(g) = g / (1 + e^-g)
 *
 * (limit <= 0: no clamp). The int8 quantizer takes its values from here; a host
 * build (tests/test_swiglu_math.py) holds them to their bound.
 *
 * The fp32 value is within 8 x 2^-24 of the exact one, relatively (exp2 1 ulp and
 * its correction half, 1 + e half, reciprocal 1 ulp, two products), as long as
 * every step stays in fp32's normal range. Two kinds of gates leave it: below
 * -87.3 the reciprocal is subnormal or zero, and a subnormal gate's product with
 * it is. There |silu(g)| < 2^-119, and so is its error, whatever is computed:
 *   |u| <= 2^32    off by less than 2^-87, 2^-27 of the largest value of a row
 *                  whose largest is 2^-60 or more (the only rows that fp32 serves)
 *   |u| > 2^32     the value may matter: it becomes NaN, which sends its row to
 *                  fp64. Only rows without a clamp, or with one beyond 2^32, need
 *                  the check. */
#ifndef DSV4_SWIGLU_MATH_H
#define DSV4_SWIGLU_MATH_H

#include <math.h>

#if defined(__HIPCC__)
#define DSV4_SWIGLU_HD __device__ __forceinline__
#define DSV4_EXP2(x) __builtin_amdgcn_exp2f(x)
#define DSV4_RCP(x) __builtin_amdgcn_rcpf(x)
#else
#define DSV4_SWIGLU_HD static inline
#define DSV4_EXP2(x) exp2f(x)
#define DSV4_RCP(x) (1.0f / (x))
#endif

namespace dsv4_swiglu {

constexpr float U_SURE = 0x1p32f;                  /* |u| up to which no gate's value is lost */
constexpr float SILU_SURE = 0x1p-118f;             /* a |silu| of normal steps throughout     */

/* whether a clamp leaves u's beyond U_SURE */
DSV4_SWIGLU_HD bool unbounded(float limit) { return !(limit > 0.0f && limit <= U_SURE); }

DSV4_SWIGLU_HD void clamp(float &g, float &u, float limit)
{
    if (limit > 0.0f) {
        u = u > limit ? limit : u;
        u = u < -limit ? -limit : u;
        g = g > limit ? limit : g;
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
     * the rounding and log2 e's own last bits left. Infinite and NaN gates give
     * NaN. */
    const float t = -g * 0x1.715476p+0f;
    const float r = fmaf(-g, 0x1.4ae0cp-26f, fmaf(-g, 0x1.715476p+0f, -t));
    const float e = DSV4_EXP2(t);
    return g * DSV4_RCP(1.0f + fmaf(e * 0x1.62e43p-1f, r, e)) * u;
}

/* whether v = value32(g, u, ..) with an unbounded clamp may have lost its value:
 * a |silu| below SILU_SURE, or none, with a u that makes it count */
DSV4_SWIGLU_HD bool lost(float g, float u, float v)
{
    return g != 0.0f && fabsf(u) > U_SURE && !(fabsf(v) >= fabsf(u) * SILU_SURE);
}

} // namespace dsv4_swiglu

#endif /* DSV4_SWIGLU_MATH_H */
