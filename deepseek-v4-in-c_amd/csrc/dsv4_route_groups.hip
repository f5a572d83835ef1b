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
 * and on no exp's last bit.
 *
 * A wave takes a token, lane l the NJ experts from l NJ on, so the lowest id of
 * equals is the lowest lane's first. A choice is one key an expert, its fp32
 * bits in an order of unsigned numbers, 0 for an expert that is not there; a pick
 * is a wave maximum and a ballot.
 */
#include "dsv4_elem.h"
#include "dsv4_gate_route.h"

namespace dsv4 {

namespace {

/* the lane's NJ logits of a token's row; past the last expert -inf */
template <int TYPE, int NJ>
__device__ __forceinline__ void load_logits(const void *logits, size_t token, int ne, int e0, float (&x)[NJ])
{
    constexpr int EB = elem_bytes<TYPE>();
    const uint8_t *row = (const uint8_t *)logits + (token * ne + e0) * EB;
    typedef float F32 __attribute__((ext_vector_type(NJ), aligned(4)));
    typedef uint16_t F16 __attribute__((ext_vector_type(NJ), aligned(2)));
    if (e0 + NJ <= ne) {
        if constexpr (EB == 4) {
            const F32 v = *(const DSV4_GLOBAL F32 *)row;
#pragma unroll
            for (int j = 0; j < NJ; j++) x[j] = v[j];
        } else {
            const F16 v = *(const DSV4_GLOBAL F16 *)row;
#pragma unroll
            for (int j = 0; j < NJ; j++) x[j] = widen16<TYPE>(v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            x[j] = -__builtin_inff();
            if (e0 + j < ne) {
                if constexpr (EB == 4) x[j] = ((const DSV4_GLOBAL float *)row)[j];
                else x[j] = widen16<TYPE>(((const DSV4_GLOBAL uint16_t *)row)[j]);
            }
        }
    }
}

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ float wave_max_f32(float v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

/* order-preserving bits of a choice; 0: not there. A choice is never -0: a
 * score is not, and +0 plus a bias of -0 is +0. */
__device__ __forceinline__ uint32_t choice_key(float c)
{
    const uint32_t u = __float_as_uint(c);
    return !(c > -__builtin_inff()) ? 0u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_choice(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

/* softmax's largest logit and sum over a token's experts */
struct Norm { float top; double inv; };
template <int NJ>
__device__ __forceinline__ Norm softmax_norm(const float (&x)[NJ], double (&p)[NJ])
{
    Norm o;
    float top = x[0];
#pragma unroll
    for (int j = 1; j < NJ; j++) top = fmaxf(top, x[j]);
    o.top = wave_max_f32(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        p[j] = x[j] > -__builtin_inff() ? exp((double)x[j] - (double)o.top) : 0.0;
        sum += p[j];
    }
    sum = wave_sum_f64(sum);
    o.inv = sum > 0.0 ? 1.0 / sum : 0.0;
    return o;
}

__device__ __forceinline__ double sigmoid64(float x) { return 1.0 / (1.0 + exp(-(double)x)); }

} // namespace

template <int TYPE, int SCORE, int NJ>
__global__ __launch_bounds__(256) void k_route_groups(RouteGroupsArgs a)
{
    const int lane = threadIdx.x & 63, ne = a.r.n_experts, topk = a.r.topk, e0 = lane * NJ;
    const long t = (long)blockIdx.x * 4 + wave_in_group();
    if (t >= a.n) return;
    float x[NJ], s[NJ];
    load_logits<TYPE, NJ>(a.logits, (size_t)t, ne, e0, x);
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NJ; j++) bad |= !(x[j] < __builtin_inff());
    const bool refused = __builtin_amdgcn_ballot_w64(bad) != 0;
    if constexpr (SCORE == DSV4_HIP_SOFTMAX) {
        double p[NJ];
        const Norm m = softmax_norm<NJ>(x, p);
#pragma unroll
        for (int j = 0; j < NJ; j++) s[j] = (float)(p[j] * m.inv);
    } else {
#pragma unroll
        for (int j = 0; j < NJ; j++) s[j] = SCORE == DSV4_HIP_SIGMOID ? (float)sigmoid64(x[j]) : route_orig(x[j]);
    }
    if (a.scores) {
        float *o = a.scores + (size_t)t * ne + e0;
#pragma unroll
        for (int j = 0; j < NJ; j++)
            if (e0 + j < ne) o[j] = refused ? __builtin_nanf("") : s[j];
    }
    uint32_t key[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const float c = a.bias && e0 + j < ne ? s[j] + a.bias[e0 + j] : s[j];
        key[j] = x[j] > -__builtin_inff() && !refused ? choice_key(c) : 0u;
    }
    if (a.r.topk_group < a.r.n_group) {
        /* the group's two largest by the lanes that hold it, met in LDS */
        __shared__ uint32_t keys[4][64 * NJ];
        uint32_t *k = keys[wave_in_group()];
#pragma unroll
        for (int j = 0; j < NJ; j++) k[e0 + j] = key[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        const int G = a.r.n_group, per = ne / G;
        uint32_t a1 = 0, a2 = 0;
        if (lane < G)
            for (int i = 0; i < per; i++) {
                const uint32_t v = k[lane * per + i];
                a2 = max(a2, min(a1, v));
                a1 = max(a1, v);
            }
        float worth = a1 ? key_choice(a1) : -__builtin_inff();
        if (a.r.group_top == 2 && a2) worth += key_choice(a2);
        /* kept: fewer than topk_group groups are worth more, or as much and lower */
        int before = 0;
        for (int i = 0; i < G; i++) {
            const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(worth), i));
            before += w > worth || (w == worth && i < lane);
        }
        const uint64_t kept = __builtin_amdgcn_ballot_w64(lane < G && before < a.r.topk_group);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int grp = min((e0 + j) / per, 63);
            key[j] = kept >> grp & 1 ? key[j] : 0u;
        }
    }
    int pick = -1;
    float got = 0.0f;
#pragma clang loop unroll(disable)
    for (int k = 0; k < topk; k++) {
        uint32_t mine = key[0];
#pragma unroll
        for (int j = 1; j < NJ; j++) mine = max(mine, key[j]);
        const uint32_t best = wave_max_u32(mine);
        if (!best) break;
        const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine == best));
        int at = 0;
        float sv = s[0];
#pragma unroll
        for (int j = NJ - 1; j >= 0; j--) {
            at = key[j] == best ? j : at;
            sv = key[j] == best ? s[j] : sv;
        }
        const int p = owner * NJ + __builtin_amdgcn_readlane(at, owner);
        const float v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sv), owner));
        if (lane == k) {
            pick = p;
            got = v;
        }
#pragma unroll
        for (int j = 0; j < NJ; j++) key[j] = lane == owner && at == j ? 0u : key[j];
    }
    double sum = 1.0;
    if (a.r.renorm) {
        sum = 0.0;
#pragma clang loop unroll(disable)
        for (int k = 0; k < topk; k++) sum += (double)__int_as_float(__builtin_amdgcn_readlane(__float_as_int(got), k));
    }
    if (lane < topk) {
        const double w = sum != 0.0 ? (double)got * (double)a.r.scale / sum : 0.0;
        a.idx[(size_t)t * topk + lane] = pick;
        a.w[(size_t)t * topk + lane] = refused ? __builtin_nanf("") : (float)w;
    }
    if (refused && lane == 0) atomicOr(a.status, ST_BAD_EXPERT_ID);
}

template <int TYPE, int SCORE, int NJ>
__global__ __launch_bounds__(256) void k_route_groups_bwd(RouteGroupsBwdArgs a)
{
    const int lane = threadIdx.x & 63, ne = a.r.n_experts, topk = a.r.topk, e0 = lane * NJ;
    const long t = (long)blockIdx.x * 4 + wave_in_group();
    if (t >= a.n) return;
    float x[NJ];
    double s[NJ], g[NJ];
    load_logits<TYPE, NJ>(a.logits, (size_t)t, ne, e0, x);
    /* the chosen ones, lane k the k-th */
    int id = -1;
    double dw = 0.0;
    if (lane < topk) {
        id = a.idx[(size_t)t * topk + lane];
        if ((unsigned)id >= (unsigned)ne) {
            if (id != -1) atomicOr(a.status, ST_BAD_EXPERT_ID);
            id = -1;
        } else {
            dw = (double)a.dw[(size_t)t * topk + lane] * (double)a.r.scale;
        }
    }
    Norm m = {0.0f, 0.0};
    if constexpr (SCORE == DSV4_HIP_SOFTMAX) {
        m = softmax_norm<NJ>(x, s);
#pragma unroll
        for (int j = 0; j < NJ; j++) s[j] *= m.inv;
    }
    auto softplus = [](float v) { return v > 20.0f ? (double)v : log1p(exp((double)v)); };
    double mine = 0.0;                             /* the score of id */
    if (id >= 0) {
        float v;
        if constexpr (TYPE == DSV4_HIP_F32) v = ((const float *)a.logits)[(size_t)t * ne + id];
        else v = widen16<TYPE>(((const uint16_t *)a.logits)[(size_t)t * ne + id]);
        if constexpr (SCORE == DSV4_HIP_SOFTMAX) mine = v > -__builtin_inff() ? exp((double)v - (double)m.top) * m.inv : 0.0;
        else if constexpr (SCORE == DSV4_HIP_SIGMOID) mine = sigmoid64(v);
        else mine = sqrt(softplus(v));
    }
    double ds = dw;
    if (a.r.renorm) {
        const double P = wave_sum_f64(mine), dot = wave_sum_f64(mine * dw);
        /* the forward call's weights are constant 0 where its fp32 scores are */
        const bool none = __builtin_amdgcn_ballot_w64((float)mine != 0.0f) == 0;
        ds = none ? 0.0 : (dw - dot / P) / P;
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) g[j] = a.dscores && e0 + j < ne ? (double)a.dscores[(size_t)t * ne + e0 + j] : 0.0;
#pragma clang loop unroll(disable)
    for (int k = 0; k < topk; k++) {
        const int e = __builtin_amdgcn_readlane(id, k);
        const long long b = __double_as_longlong(ds);
        const double d = __longlong_as_double(((long long)__builtin_amdgcn_readlane((int)(b >> 32), k) << 32) |
                                              (uint32_t)__builtin_amdgcn_readlane((int)b, k));
#pragma unroll
        for (int j = 0; j < NJ; j++) g[j] += e0 + j == e ? d : 0.0;
    }
    double all = 0.0;
    if constexpr (SCORE == DSV4_HIP_SOFTMAX) {
#pragma unroll
        for (int j = 0; j < NJ; j++) all += s[j] * g[j];
        all = wave_sum_f64(all);
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        if (e0 + j >= ne) continue;
        double d;
        if constexpr (SCORE == DSV4_HIP_SOFTMAX) {
            d = s[j] * (g[j] - all);
        } else if constexpr (SCORE == DSV4_HIP_SIGMOID) {
            const double v = sigmoid64(x[j]);
            d = v * (1.0 - v) * g[j];
        } else {
            const double v = sqrt(softplus(x[j]));
            d = v == 0.0 ? 0.0 : (x[j] > 20.0f ? 1.0 : sigmoid64(x[j])) / (2.0 * v) * g[j];
        }
        const size_t at = (size_t)t * ne + e0 + j;
        if constexpr (TYPE == DSV4_HIP_F32) ((float *)a.dlogits)[at] = (float)d;
        else ((uint16_t *)a.dlogits)[at] = (uint16_t)narrow16<TYPE>((float)d);
    }
}

namespace {

template <int TYPE, int SCORE, int NJ>
hipError_t launch(const RouteGroupsArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((k_route_groups<TYPE, SCORE, NJ>), dim3((unsigned)((a.n + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError();
}
template <int TYPE, int SCORE, int NJ>
hipError_t launch(const RouteGroupsBwdArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((k_route_groups_bwd<TYPE, SCORE, NJ>), dim3((unsigned)((a.n + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError();
}
template <int TYPE, int SCORE, class ARGS>
hipError_t launch_nj(const ARGS &a, hipStream_t st)
{
    const int nj = (a.r.n_experts + 63) / 64;
    if (nj <= 1) return launch<TYPE, SCORE, 1>(a, st);
    if (nj <= 2) return launch<TYPE, SCORE, 2>(a, st);
    if (nj <= 4) return launch<TYPE, SCORE, 4>(a, st);
    if (nj <= 8) return launch<TYPE, SCORE, 8>(a, st);
    return launch<TYPE, SCORE, RT_MAXJ>(a, st);
}
template <int TYPE, class ARGS>
hipError_t launch_score(const ARGS &a, hipStream_t st)
{
    switch (a.r.score) {
    case DSV4_HIP_SQRT_SOFTPLUS: return launch_nj<TYPE, DSV4_HIP_SQRT_SOFTPLUS>(a, st);
    case DSV4_HIP_SOFTMAX: return launch_nj<TYPE, DSV4_HIP_SOFTMAX>(a, st);
    case DSV4_HIP_SIGMOID: return launch_nj<TYPE, DSV4_HIP_SIGMOID>(a, st);
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
