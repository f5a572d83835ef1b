/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_route_groups.hip - the router with softmax, sigmoid or sqrt(softplus)
 * scores, a bias for balance, groups of experts and its gradient:
 *   c = s(x) + bias;  groups by the sum of their one or two largest c; the topk
 *   largest c of the groups kept;  w_k = scale s_k / sum_j s_j  (renorm)
 *   ds_k = scale (dw_k - sum_j dw_j s_j / P) / P,  P = sum_j s_j   (renorm)
 *        = scale dw_k                                             (else)
 *   and onto the logits, with g = ds at the chosen ids + dscores:
 *   sigmoid  dx = s (1 - s) g          softmax  dx = s (g - sum_e s_e g_e)
 *   sqrt(softplus)  dx = sigmoid(x) / (2 s) g   (1 / (2 s) g above 20, as s is
 *   sqrt(x) there)
 * Scores are fp64 rounded once to fp32 (sqrt(softplus) the router's own bits,
 * dsv4_route_math.h); the choice compares fp32 sums, so it depends on no order
 * and, but for a score within 2^-20 of a step of a rounding border, on no exp's
 * last bit.
 *
 * A token is held by L lanes, 16 (four tokens a wave) or 64, lane l the experts 4
 * l + 4 L q + i, i < 4, q < NQ: rows are read in whole lines. A choice is one key
 * an expert, its fp32 bits in an order of unsigned numbers, 0 for an expert that
 * is not there. A pick is the largest key and the least id among equals.
 *
 * Bound: few tokens by the chain of loads, scores, groups and picks (1 token of 256
 * experts in 8 groups, top 6, 4.6 us, 3.9 without groups and top 1); many by the vector
 * unit, 50 instructions a score and 300 for eight picks of four tokens (16,384 tokens,
 * 8 groups, top 8, with scores 16.4 us for 33.5 MB, which HBM alone moves in 7). Backward
 * of 16,384 tokens: four waves a SIMD, all there at once, so loads, 4,700 vector
 * instructions a SIMD and stores follow each other with little overlap (sigmoid 15.2 us
 * for 50 MB, 3.3 TB/s, softmax 16, sqrt(softplus) 23.5 for its logarithms).
 */
#include "dsv4_elem.h"
#include "dsv4_gate_route.h"

namespace dsv4 {

namespace {

template <int N> struct IC { static constexpr int value = N; };

constexpr float NO_EXPERT = -__builtin_inff();     /* the logit of one that is not there */

/* four consecutive elements of a row from e on, at any alignment of one; past
 * the row's end NO_EXPERT */
template <int TYPE>
__device__ __forceinline__ void load4(const void *row, int e, int ne, float (&x)[4])
{
    constexpr int EB = elem_bytes<TYPE>();
    typedef uint32_t W4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint16_t H4 __attribute__((ext_vector_type(4), aligned(2)));
    const uint8_t *p = (const uint8_t *)row + (size_t)e * EB;
    if (e + 4 <= ne) {
        if constexpr (EB == 4) {
            const W4 v = *(const DSV4_GLOBAL W4 *)p;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __uint_as_float(v[i]);
        } else {
            const H4 v = *(const DSV4_GLOBAL H4 *)p;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = widen16<TYPE>(v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = NO_EXPERT;
            if (e + i < ne) {
                if constexpr (EB == 4) x[i] = gptr((const float *)p)[i];
                else x[i] = widen16<TYPE>(gptr((const uint16_t *)p)[i]);
            }
        }
    }
}
template <int TYPE>
__device__ __forceinline__ void store4(void *row, int e, int ne, const float (&x)[4])
{
    constexpr int EB = elem_bytes<TYPE>();
    typedef uint32_t W4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint16_t H4 __attribute__((ext_vector_type(4), aligned(2)));
    uint8_t *p = (uint8_t *)row + (size_t)e * EB;
    if (e + 4 <= ne) {
        if constexpr (EB == 4) {
            W4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = __float_as_uint(x[i]);
            *(DSV4_GLOBAL W4 *)p = v;
        } else {
            H4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (uint16_t)narrow16<TYPE>(x[i]);
            *(DSV4_GLOBAL H4 *)p = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (e + i >= ne) break;
            if constexpr (EB == 4) ((DSV4_GLOBAL float *)p)[i] = x[i];
            else ((DSV4_GLOBAL uint16_t *)p)[i] = (uint16_t)narrow16<TYPE>(x[i]);
        }
    }
}
template <int TYPE>
__device__ __forceinline__ float load1(const void *row, int e)
{
    if constexpr (TYPE == DSV4_HIP_F32) return gptr((const float *)row)[e];
    else return widen16<TYPE>(gptr((const uint16_t *)row)[e]);
}
template <int TYPE>
__device__ __forceinline__ void store1(void *row, int e, float v)
{
    if constexpr (TYPE == DSV4_HIP_F32) ((DSV4_GLOBAL float *)row)[e] = v;
    else ((DSV4_GLOBAL uint16_t *)row)[e] = (uint16_t)narrow16<TYPE>(v);
}

/* Over the L lanes of a token, to all of them, in an order of its own. */
template <int L, class OP>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, OP op)
{
    v = op(v, dpp_u32<DPP_QUAD_1032>(v, v));
    v = op(v, dpp_u32<DPP_QUAD_2301>(v, v));
    v = op(v, dpp_u32<DPP_ROW_HALF_MIRROR>(v, v));
    v = op(v, dpp_u32<DPP_ROW_MIRROR>(v, v));
    if constexpr (L == 64) {
        v = op(v, dpp_u32<DPP_ROW_BCAST15, 0xA>(v, v));
        v = op(v, dpp_u32<DPP_ROW_BCAST31, 0xC>(v, v));
        v = (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
    }
    return v;
}
template <int L>
__device__ __forceinline__ double sum_lanes(double v)
{
#pragma unroll
    for (int d = 1; d < L; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
template <int L>
__device__ __forceinline__ bool any_lane(bool b, int lane)
{
    const uint64_t m = __builtin_amdgcn_ballot_w64(b);
    return L == 64 ? m != 0 : (m >> (lane & 48) & 0xFFFFu) != 0;
}

/* An expert's place as one positive fp64 number, key bits above those of 1023 - id
 * (below 2^62: neither infinite nor NaN): the maximum of two is one instruction
 * and settles ties. Key 0: below every other, no expert. */
__device__ __forceinline__ double place_of(uint32_t key, int id)
{
    return __longlong_as_double((long long)((uint64_t)key << 30 | (uint32_t)(1023 - id)));
}
__device__ __forceinline__ int expert_of(double place)
{
    const uint64_t u = (uint64_t)__double_as_longlong(place);
    return u >> 30 ? 1023 - (int)(u & 1023) : -1;
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
    return __longlong_as_double((long long)((uint64_t)dpp_u32<CTRL, ROWS>(hi, hi) << 32 | dpp_u32<CTRL, ROWS>(lo, lo)));
}
template <int L>
__device__ __forceinline__ double max_lanes(double v)
{
    v = fmax(v, dpp_f64<DPP_QUAD_1032>(v));
    v = fmax(v, dpp_f64<DPP_QUAD_2301>(v));
    v = fmax(v, dpp_f64<DPP_ROW_HALF_MIRROR>(v));
    v = fmax(v, dpp_f64<DPP_ROW_MIRROR>(v));
    if constexpr (L == 64) {
        v = fmax(v, dpp_f64<DPP_ROW_BCAST15, 0xA>(v));
        v = fmax(v, dpp_f64<DPP_ROW_BCAST31, 0xC>(v));
        const uint64_t u = (uint64_t)__double_as_longlong(v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
        v = __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
    }
    return v;
}

/* The l-th largest (l < 8) of the 4 NQ numbers in each of a token's 16 lanes. A lane
 * sorts its own, then sorted lists of eight meet: the eight largest of two are the
 * larger of a[i] and b[7 - i], which rise and then fall, so three rounds of
 * exchanges sort them. 16 numbers a lane: some 300 instructions, eight picks one
 * after the other 500. With 64 lanes and fewer numbers in each the picks are the
 * shorter (us, lists / picks: 1 token of 256 experts in groups, top 8, 4.5 / 4.7, but
 * 4,096 9.9 / 9.4, with softmax and top 6 7.7 / 7.0). */
__device__ __forceinline__ void exchange(double &a, double &b)
{
    const double hi = fmax(a, b);
    b = fmin(a, b);
    a = hi;
}
struct Eight { double v[8]; };
__device__ __forceinline__ void sort_bitonic(Eight &a)
{
#pragma unroll
    for (int d = 4; d; d >>= 1)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (!(i & d)) exchange(a.v[i], a.v[i + d]);
}
__device__ __forceinline__ void sort_any(Eight &a)          /* merges of odd and even places */
{
    constexpr int from[19] = {0, 2, 4, 6, 0, 1, 4, 5, 1, 5, 0, 1, 2, 3, 2, 3, 1, 3, 5};
    constexpr int to[19] = {1, 3, 5, 7, 2, 3, 6, 7, 2, 6, 4, 5, 6, 7, 4, 5, 2, 4, 6};
#pragma unroll
    for (int i = 0; i < 19; i++) exchange(a.v[from[i]], a.v[to[i]]);
}
/* the eight largest of two sorted lists, sorted */
__device__ __forceinline__ void join(Eight &a, const Eight &b)
{
#pragma unroll
    for (int i = 0; i < 8; i++) a.v[i] = fmax(a.v[i], b.v[7 - i]);
    sort_bitonic(a);
}
template <int CTRL>
__device__ __forceinline__ void join_lanes(Eight &a)
{
    Eight b;
#pragma unroll
    for (int i = 0; i < 8; i++) b.v[i] = dpp_f64<CTRL>(a.v[i]);
    join(a, b);
}
template <int NQ>
__device__ __forceinline__ double largest_of_lanes(const double (&v)[4 * NQ], int l)
{
    Eight a;
    if constexpr (NQ == 1) {
#pragma unroll
        for (int i = 0; i < 4; i++) a.v[i] = v[i];
        exchange(a.v[0], a.v[1]);
        exchange(a.v[2], a.v[3]);
        exchange(a.v[0], a.v[2]);
        exchange(a.v[1], a.v[3]);
        exchange(a.v[1], a.v[2]);
#pragma unroll
        for (int i = 0; i < 4; i++) a.v[7 - i] = dpp_f64<DPP_QUAD_1032>(a.v[i]);
        sort_bitonic(a);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) a.v[i] = v[i];
        sort_any(a);
        if constexpr (NQ == 4) {
            Eight b;
#pragma unroll
            for (int i = 0; i < 8; i++) b.v[i] = v[8 + i];
            sort_any(b);
            join(a, b);
        }
        join_lanes<DPP_QUAD_1032>(a);
    }
    join_lanes<DPP_QUAD_2301>(a);
    join_lanes<DPP_ROW_HALF_MIRROR>(a);
    join_lanes<DPP_ROW_MIRROR>(a);
    double o = a.v[0];
#pragma unroll
    for (int i = 1; i < 8; i++) o = l == i ? a.v[i] : o;
    return o;
}

/* order-preserving bits of a number that is not NaN; larger for larger ones. -0
 * does not occur: a score is none, and +0 plus a bias of -0 is +0. */
__device__ __forceinline__ uint32_t order_of(float c)
{
    const uint32_t u = __float_as_uint(c);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

/* e^x in fp64 for |x| <= 700: x = k ln 2 + r with k the nearest integer, read from
 * the low bits of a sum with 1.5 x 2^52, and e^r by the polynomial of degree 10
 * that is nearest to it on |r| <= 0.3466 in the Chebyshev sense (relatively within
 * 2^-52; fitted in 50 digits), k added to the exponent: 15 instructions. */
__device__ __forceinline__ double exp64(double x)
{
    const double magic = 6755399441055744.0, s = fma(x, 1.4426950408889634, magic), k = s - magic;
    const double r = fma(k, -2.3190468138462996e-17, fma(k, -0.6931471805599453, x));
    double p = 2.762637106569635607642e-7;
    p = fma(p, r, 2.764019739169484046713e-6);
    p = fma(p, r, 2.480150431378554016571e-5);
    p = fma(p, r, 1.984117023057028666426e-4);
    p = fma(p, r, 1.388888893251477935536e-3);
    p = fma(p, r, 8.333333385699211726935e-3);
    p = fma(p, r, 4.166666666657306773181e-2);
    p = fma(p, r, 0.1666666666655431458301);
    p = fma(p, r, 0.5000000000000005622546);
    p = fma(p, r, 1.000000000000006749096);
    p = fma(p, r, 1.0);
    return __longlong_as_double(__double_as_longlong(p) + (long long)((uint64_t)__double_as_longlong(s) << 52));
}
/* 1 / v for normal v whose reciprocal is normal: the instruction's 24 bits to 53
 * in one step of third order */
__device__ __forceinline__ double rcp64(double v)
{
    const double y = __builtin_amdgcn_rcp(v), e = fma(-v, y, 1.0);
    return fma(fma(e, e, e), y, y);
}
/* beyond 700 the score is 0 or 1 in fp32, and in fp64 next to it */
__device__ __forceinline__ double sigmoid64(float x)
{
    return rcp64(1.0 + exp64((double)__builtin_amdgcn_fmed3f(-x, -700.0f, 700.0f)));
}
__device__ __forceinline__ double exp_below(float x, float top) { return exp64(fmax((double)x - (double)top, -700.0)); }
/* sqrt(softplus(x)) and its derivative sigmoid(x) / (2 sqrt(softplus(x))) in fp64,
 * relatively within 2^-44; 1 / (2 sqrt(x)) above 20; 0 for an expert that is not
 * there. With 1 + e^x = 2^k (1 + f), 1 + f in [sqrt(1/2), sqrt(2)) (f = e^x itself
 * where k is 0, so that a small one keeps its bits), the logarithm is k ln 2 + 2 t (1 +
 * t^2 / 3 + .. + t^14 / 15), t = f / (2 + f), |t| < 0.172; the square root and the division
 * are one reciprocal root, the instruction's bits and a step of third order. */
struct Root { double s, d; };
__device__ __forceinline__ Root sqrt_softplus64(float x)
{
    const double e = exp64((double)__builtin_amdgcn_fmed3f(x, -700.0f, 20.0f)), u = 1.0 + e;
    const uint64_t bits = (uint64_t)__double_as_longlong(u);
    const int k = ((int)(bits >> 32) - 0x3FE6A09E) >> 20;
    const double m = __longlong_as_double((long long)(bits - ((uint64_t)(uint32_t)k << 52)));
    const double f = k == 0 ? e : m - 1.0, t = f * rcp64(2.0 + f), w = t * t;
    double p = 2.0 / 15;
    p = fma(p, w, 2.0 / 13);
    p = fma(p, w, 2.0 / 11);
    p = fma(p, w, 2.0 / 9);
    p = fma(p, w, 2.0 / 7);
    p = fma(p, w, 2.0 / 5);
    p = fma(p, w, 2.0 / 3);
    p = fma((double)k, 0.6931471805599453, fma(t * w, p, t + t));
    p = x > 20.0f ? fmin((double)x, 1e300) : p;
    double y = __builtin_amdgcn_rsq(p);
    const double h = fma(-p * y, y, 1.0);
    y = fma(y * h, fma(h, 0.375, 0.5), y);
    const double d = (x > 20.0f ? 0.5 : 0.5 * e * rcp64(u)) * y;
    Root o = {p * y, d};
    if (!(x > NO_EXPERT)) o.s = o.d = x < 0.0f ? 0.0 : (double)x;      /* -inf; NaN stays */
    return o;
}

/* softmax over a token's L x 4 NQ logits: e^(x - top), top and 1 / sum; an expert
 * that is not there adds nothing, a token without experts has inv 0 */
struct Norm { float top; double inv; };
template <int L, int NQ>
__device__ __forceinline__ Norm softmax_norm(const float (&x)[NQ][4], double (&p)[NQ][4])
{
    uint32_t top = 0;
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = max32(top, order_of(x[q][i]));
    Norm o;
    o.top = of_order(over_lanes<L>(top, max32));
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            p[q][i] = x[q][i] > NO_EXPERT ? exp_below(x[q][i], o.top) : 0.0;
            sum += p[q][i];
        }
    sum = sum_lanes<L>(sum);
    o.inv = sum > 0.0 ? 1.0 / sum : 0.0;
    return o;
}

/* one score as the forward call gives it */
template <int SCORE>
__device__ __forceinline__ float score32(float x, const Norm &m)
{
    if constexpr (SCORE == DSV4_HIP_SOFTMAX) return x > NO_EXPERT ? (float)(exp_below(x, m.top) * m.inv) : 0.0f;
    else if constexpr (SCORE == DSV4_HIP_SIGMOID) return (float)sigmoid64(x);
    else {
        bool rare = false;
        const float s = dsv4_route::route_orig_most(x, rare);
        return rare ? route_orig(x) : s;
    }
}

/* whether score32 of x, with s its score in fp64, is 0 */
template <int SCORE>
__device__ __forceinline__ bool zero_score(float x, double s)
{
    if constexpr (SCORE == DSV4_HIP_SQRT_SOFTPLUS) return dsv4_route::route_orig_zero(x);
    else return (float)s == 0.0f;
}

} // namespace

template <int TYPE, int SCORE, int L, int NQ>
__global__ __launch_bounds__(256) void k_route_groups(RouteGroupsArgs a)
{
    constexpr int TPW = 64 / L;                    /* tokens of a wave */
    const int lane = threadIdx.x & 63, l = lane % L, ne = a.r.n_experts, topk = a.r.topk;
    const long t0 = ((long)blockIdx.x * 4 + wave_in_group()) * TPW, t = t0 + lane / L;
    if (t0 >= a.n) return;
    const bool there = t < a.n;                    /* tokens past the last: the last again, not stored */
    const size_t tok = (size_t)min(t, (long)a.n - 1);
    const void *row = (const uint8_t *)a.logits + tok * ne * elem_bytes<TYPE>();
    auto id_of = [&](int q, int i) { return 4 * l + 4 * L * q + i; };
    float x[NQ][4];
#pragma unroll
    for (int q = 0; q < NQ; q++) load4<TYPE>(row, id_of(q, 0), ne, x[q]);
    float b[NQ][4];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        if (a.bias) load4<DSV4_HIP_F32>(a.bias, id_of(q, 0), ne, b[q]);
        else
#pragma unroll
            for (int i = 0; i < 4; i++) b[q][i] = 0.0f;
    }
    bool bad = false;
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int i = 0; i < 4; i++) bad |= !(x[q][i] < __builtin_inff());
    const bool refused = any_lane<L>(bad, lane);
    uint32_t key[NQ][4];
    Norm m = {0.0f, 0.0};
    {
        float s[NQ][4];
        if constexpr (SCORE == DSV4_HIP_SOFTMAX) {
            double p[NQ][4];
            m = softmax_norm<L, NQ>(x, p);
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[q][i] = (float)(p[q][i] * m.inv);
        } else if constexpr (SCORE == DSV4_HIP_SIGMOID) {
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[q][i] = score32<SCORE>(x[q][i], m);
        } else {
            /* all without a branch, so that the table's loads overlap (1 token of 256
             * experts 4.6 us, with branches 6.1; 16,384 21, 27); again where that does
             * not serve */
            bool rare = false;
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[q][i] = dsv4_route::route_orig_most(x[q][i], rare);
            if (rare) {
#pragma unroll
                for (int q = 0; q < NQ; q++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[q][i] = route_orig(x[q][i]);
            }
        }
#pragma unroll
        for (int q = 0; q < NQ; q++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float c = __fadd_rn(s[q][i], b[q][i]);
                key[q][i] = x[q][i] > NO_EXPERT && c > NO_EXPERT && !refused ? order_of(c) : 0u;
                if (refused) s[q][i] = __builtin_nanf("");
            }
            if (a.scores && there && id_of(q, 0) < ne) store4<DSV4_HIP_F32>(a.scores + tok * ne, id_of(q, 0), ne, s[q]);
        }
    }
    if (a.r.topk_group < a.r.n_group) {
        /* Keys through LDS, a group's beside each other and groups 4 words further
         * apart, so that lanes with a group each read from different banks. */
        constexpr int E = 4 * L * NQ, G = 64;
        __shared__ __align__(16) uint32_t keys[4][TPW][E + 4 * G];
        uint32_t *const k = keys[wave_in_group()][lane / L];
        const int ng = a.r.n_group, per = ne / ng;
        const uint32_t mul = ((1u << 22) + per - 1) / per;     /* e / per = e mul >> 22 for e < 1024 */
        const bool quads = per % 4 == 0;           /* four neighbours share a group */
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int e = id_of(q, 0);
            if (quads) {
                if (e < ne) *(u32x4 *)(k + e + 4 * (e * mul >> 22)) = u32x4{key[q][0], key[q][1], key[q][2], key[q][3]};
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (e + i < ne) k[e + i + 4 * ((e + i) * mul >> 22)] = key[q][i];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        /* what group grp is worth, in the order of unsigned numbers */
        auto worth_of = [&](int grp) -> uint32_t {
            uint32_t a1 = 0, a2 = 0;
            if (grp < ng) {
                const uint32_t *p = k + grp * (per + 4);
                if (quads)
                    for (int i = 0; i < per; i += 4) {
                        const u32x4 v = *(const u32x4 *)(p + i);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            a2 = max32(a2, min32(a1, v[j]));
                            a1 = max32(a1, v[j]);
                        }
                    }
                else
                    for (int i = 0; i < per; i++) {
                        a2 = max32(a2, min32(a1, p[i]));
                        a1 = max32(a1, p[i]);
                    }
            }
            float w = of_order(a1);
            if (a.r.group_top == 2 && a2) w = __fadd_rn(w, of_order(a2));
            return a1 ? order_of(w == 0.0f ? 0.0f : w) : 0u;
        };
        /* kept: fewer than topk_group groups are worth more, or as much and lower.
         * H groups a lane: l, l + L, .. */
        uint64_t kept = 0;
        auto keep = [&](auto HS) {
            constexpr int H = decltype(HS)::value;
            uint32_t worth[H];
            int before[H];
#pragma unroll
            for (int h = 0; h < H; h++) {
                worth[h] = worth_of(l + L * h);
                before[h] = 0;
            }
#pragma unroll
            for (int h = 0; h < H; h++)
                for (int i = 0; i < L && L * h + i < ng; i++) {
                    const uint32_t w = (uint32_t)__shfl((int)worth[h], i, L);
#pragma unroll
                    for (int o = 0; o < H; o++) before[o] += w > worth[o] || (w == worth[o] && L * h + i < l + L * o);
                }
#pragma unroll
            for (int h = 0; h < H; h++) {
                const uint64_t m64 = __builtin_amdgcn_ballot_w64(l + L * h < ng && before[h] < a.r.topk_group);
                if constexpr (L == 64) kept = m64;
                else kept |= (m64 >> (lane & 48) & 0xFFFFu) << (16 * h);
            }
        };
        if (ng <= L) keep(IC<1>{});
        else keep(IC<G / L>{});
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const uint32_t e = (uint32_t)id_of(q, 0);
            const bool in0 = kept >> min32(e * mul >> 22, 63u) & 1;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool in = quads ? in0 : kept >> min32((e + i) * mul >> 22, 63u) & 1;
                key[q][i] = in ? key[q][i] : 0u;
            }
        }
    }
    double place[4 * NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int i = 0; i < 4; i++) place[4 * q + i] = place_of(key[q][i], id_of(q, i));
    double mine = 0.0;
    if (L == 16 && topk <= 8) {
        mine = largest_of_lanes<NQ>(place, l);
    } else {
#pragma clang loop unroll(disable)
        for (int k = 0; k < topk; k++) {
            double best = place[0];
#pragma unroll
            for (int j = 1; j < 4 * NQ; j++) best = fmax(best, place[j]);
            best = max_lanes<L>(best);
            mine = l == k ? best : mine;
#pragma unroll
            for (int j = 0; j < 4 * NQ; j++) place[j] = place[j] == best ? 0.0 : place[j];
        }
    }
    const int pick = l < topk ? expert_of(mine) : -1;
    /* lane k's pick again, from its logit: the same bits */
    const float got = pick >= 0 ? score32<SCORE>(load1<TYPE>(row, pick), m) : 0.0f;
    const double sum = a.r.renorm ? sum_lanes<16>((double)got) : 1.0;
    if (l < topk && there) {
        const double w = sum != 0.0 ? (double)got * (double)a.r.scale / sum : 0.0;
        a.idx[tok * topk + l] = pick;
        a.w[tok * topk + l] = refused ? __builtin_nanf("") : (float)w;
    }
    if (refused && l == 0 && there) atomicOr(a.status, ST_BAD_EXPERT_ID);
}

/* Gradients that come from dscores (or none), expert by expert; then, when those
 * stores have arrived, the chosen experts', whole, from lane k < topk. Without
 * dscores only softmax without renorm reads the row: elsewhere what is not chosen
 * has gradient 0. */
template <int TYPE, int SCORE, int L, int NQ>
__global__ __launch_bounds__(256) void k_route_groups_bwd(RouteGroupsBwdArgs a)
{
    constexpr int TPW = 64 / L;
    const int lane = threadIdx.x & 63, l = lane % L, ne = a.r.n_experts, topk = a.r.topk;
    const long t0 = ((long)blockIdx.x * 4 + wave_in_group()) * TPW, t = t0 + lane / L;
    if (t0 >= a.n) return;
    const bool there = t < a.n;
    const size_t tok = (size_t)min(t, (long)a.n - 1);
    const void *row = (const uint8_t *)a.logits + tok * ne * elem_bytes<TYPE>();
    void *const out = (uint8_t *)a.dlogits + tok * ne * elem_bytes<TYPE>();
    auto id_of = [&](int q) { return 4 * l + 4 * L * q; };
    const bool dense = a.dscores || SCORE == DSV4_HIP_SOFTMAX;
    /* lane k's expert */
    int id = -1;
    double dw = 0.0;
    if (l < topk) {
        id = a.idx[tok * topk + l];
        if ((unsigned)id >= (unsigned)ne) {
            if (id != -1 && there) atomicOr(a.status, ST_BAD_EXPERT_ID);
            id = -1;
        } else {
            dw = (double)a.dw[tok * topk + l] * (double)a.r.scale;
        }
    }
    const float xk = id >= 0 ? load1<TYPE>(row, id) : 0.0f;
    const double gk = id >= 0 && a.dscores ? (double)gptr(a.dscores)[tok * ne + id] : 0.0;
    float x[NQ][4];
    float g[NQ][4];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        if (dense) load4<TYPE>(row, id_of(q), ne, x[q]);
        if (a.dscores) load4<DSV4_HIP_F32>(a.dscores + tok * ne, id_of(q), ne, g[q]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (!dense) x[q][i] = NO_EXPERT;
            if (!a.dscores || id_of(q) + i >= ne) g[q][i] = 0.0f;
            if (SCORE == DSV4_HIP_SOFTMAX && !(x[q][i] > NO_EXPERT)) g[q][i] = 0.0f;   /* before it enters a sum */
        }
    }
    /* a token that the forward call refuses has ids of -1: without its logits and its
     * scores' gradients it counts as one without experts */
    if (dense) {
        float top = NO_EXPERT;                     /* NaN if one is */
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = __builtin_elementwise_maximum(top, x[q][i]);
        if (any_lane<L>(!(top < __builtin_inff()), lane)) {
            if (l == 0 && there) atomicOr(a.status, ST_BAD_EXPERT_ID);
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[q][i] = NO_EXPERT;
                    g[q][i] = 0.0f;
                }
        }
    }
    Norm m = {0.0f, 0.0};
    double s[NQ][4];
    if constexpr (SCORE == DSV4_HIP_SOFTMAX) m = softmax_norm<L, NQ>(x, s);
    /* a score, and its own derivative (softmax: the score) */
    auto score = [&](float v) -> double {
        if constexpr (SCORE == DSV4_HIP_SOFTMAX) return v > NO_EXPERT ? exp_below(v, m.top) * m.inv : 0.0;
        else if constexpr (SCORE == DSV4_HIP_SIGMOID) return sigmoid64(v);
        else return sqrt_softplus64(v).s;
    };
    auto slope = [&](float v, double sv) -> double {
        if constexpr (SCORE == DSV4_HIP_SOFTMAX) return sv;
        else if constexpr (SCORE == DSV4_HIP_SIGMOID) return sv * (1.0 - sv);
        else return sqrt_softplus64(v).d;
    };
    const double sk = id >= 0 ? score(xk) : 0.0;
    double ds = dw;
    if (a.r.renorm) {
        const double P = sum_lanes<16>(sk), dot = sum_lanes<16>(sk * dw);
        /* the forward call's weights are constant 0 where its fp32 scores are */
        const bool none = !any_lane<L>(id >= 0 && !zero_score<SCORE>(xk, sk), lane);
        ds = none ? 0.0 : (dw - dot / P) / P;
    }
    /* the same expert twice: its gradient holds both */
    double mine = id >= 0 ? gk : 0.0;
#pragma clang loop unroll(disable)
    for (int k = 0; k < topk; k++) {
        const int e = __shfl(id, k, L);
        const double d = __shfl(ds, k, L);
        if (e == id) mine += d;
    }
    double all = 0.0;                              /* softmax: sum_e s_e g_e */
    if constexpr (SCORE == DSV4_HIP_SOFTMAX) {
        if (a.dscores) {
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) all += s[q][i] * m.inv * (double)g[q][i];
        }
        all = sum_lanes<L>(all + (id >= 0 ? sk * ds : 0.0));
    }
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (SCORE == DSV4_HIP_SOFTMAX) {
                o[i] = (float)(s[q][i] * m.inv * ((double)g[q][i] - all));
            } else {
                o[i] = 0.0f;
                if (a.dscores) {
                    const double v = score(x[q][i]);
                    o[i] = x[q][i] > NO_EXPERT ? (float)(slope(x[q][i], v) * (double)g[q][i]) : 0.0f;
                }
            }
        }
        if (there && id_of(q) < ne) store4<TYPE>(out, id_of(q), ne, o);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);            /* vmcnt(0) */
    asm volatile("" ::: "memory");
    if (id >= 0 && there) store1<TYPE>(out, id, (float)(slope(xk, sk) * (mine - all)));
}

namespace {

template <int TYPE, int SCORE, int L, int NQ>
hipError_t launch(const RouteGroupsArgs &a, hipStream_t st)
{
    constexpr int tokens = 4 * (64 / L);
    hipLaunchKernelGGL((k_route_groups<TYPE, SCORE, L, NQ>), dim3((unsigned)((a.n + tokens - 1) / tokens)), dim3(256), 0, st, a);
    return hipGetLastError();
}
template <int TYPE, int SCORE, int L, int NQ>
hipError_t launch(const RouteGroupsBwdArgs &a, hipStream_t st)
{
    constexpr int tokens = 4 * (64 / L);
    hipLaunchKernelGGL((k_route_groups_bwd<TYPE, SCORE, L, NQ>), dim3((unsigned)((a.n + tokens - 1) / tokens)), dim3(256), 0, st,
                       a);
    return hipGetLastError();
}
/* Tokens from which four share a wave: fewer leave lanes of the device idle. us, a
 * wave each / shared, 256 experts: sigmoid, 8 groups, top 8 2,048 tokens 6.8 / 7.2,
 * 3,000 7.8 / 7.3, 16,384 26 / 16.4; softmax, top 6 3,000 6.1 / 6.9, 4,096 7.0 / 6.8,
 * 16,384 19 / 12.3; sqrt(softplus), top 6 4,096 8.9 / 10.4, 8,192 14.0 / 12.6, 16,384 25
 * / 21; backward with scores' gradients 6,000 7.5 / 8.4, 8,192 9.3 / 9.3, 16,384 16.6 /
 * 15.4, softmax 18.6 / 16.4, sqrt(softplus) 26 / 23.5, without 6,000 6.1 / 4.6. Fewer
 * experts go by the same counts. */
int shared_from(const RouteGroupsArgs &a) { return a.r.score == DSV4_HIP_SQRT_SOFTPLUS ? 6144 : 3500; }
int shared_from(const RouteGroupsBwdArgs &a) { return a.dscores ? 8192 : 4096; }
template <int TYPE, int SCORE, class ARGS>
hipError_t launch_size(const ARGS &a, hipStream_t st)
{
    const int ne = a.r.n_experts;
    if (ne <= 256 && a.n >= shared_from(a)) {
        if (ne <= 64) return launch<TYPE, SCORE, 16, 1>(a, st);
        if (ne <= 128) return launch<TYPE, SCORE, 16, 2>(a, st);
        return launch<TYPE, SCORE, 16, 4>(a, st);
    }
    if (ne <= 256) return launch<TYPE, SCORE, 64, 1>(a, st);
    if (ne <= 512) return launch<TYPE, SCORE, 64, 2>(a, st);
    return launch<TYPE, SCORE, 64, 4>(a, st);
}
template <int TYPE, class ARGS>
hipError_t launch_score(const ARGS &a, hipStream_t st)
{
    switch (a.r.score) {
    case DSV4_HIP_SQRT_SOFTPLUS: return launch_size<TYPE, DSV4_HIP_SQRT_SOFTPLUS>(a, st);
    case DSV4_HIP_SOFTMAX: return launch_size<TYPE, DSV4_HIP_SOFTMAX>(a, st);
    case DSV4_HIP_SIGMOID: return launch_size<TYPE, DSV4_HIP_SIGMOID>(a, st);
    default: return hipErrorInvalidValue;
    }
}
template <class ARGS>
hipError_t launch_type(const ARGS &a, int type, hipStream_t st)
{
    if (a.n <= 0 || a.r.n_experts < 1 || a.r.n_experts > GATE_ROUTE_MAX_EXPERTS || a.r.topk < 1 ||
        a.r.topk > GATE_ROUTE_MAX_TOPK)
        return hipErrorInvalidValue;
    switch (type) {
    case DSV4_HIP_F32: return launch_score<DSV4_HIP_F32>(a, st);
    case DSV4_HIP_BF16: return launch_score<DSV4_HIP_BF16>(a, st);
    case DSV4_HIP_F16: return launch_score<DSV4_HIP_F16>(a, st);
    default: return hipErrorInvalidValue;
    }
}

} // namespace

hipError_t route_groups_launch(const RouteGroupsArgs &a, int type, hipStream_t st) { return launch_type(a, type, st); }
hipError_t route_groups_bwd_launch(const RouteGroupsBwdArgs &a, int type, hipStream_t st)
{
    return launch_type(a, type, st);
}

} // namespace dsv4
