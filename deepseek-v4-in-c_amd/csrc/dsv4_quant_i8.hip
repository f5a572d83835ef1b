/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_quant_i8.hip - rows to 8-bit integers with one fp32 scale a row, the
 * operands of the int8 products: tokens, weight rows, or the experts' SwiGLU
 * output straight from the gate and up products.
 *
 * With amax = max_j |a_j|:  scale = amax / 127 (fp32, rounded once; 1 for a
 * row of zeros) and code_j = the integer nearest to 127 a_j / amax, ties to
 * even. A row with a value that is not finite has scale NaN and codes 0.
 *
 * EXACT CODES
 *   fp32 gives 127 a_j / amax as a_j * (127 / amax), off by at most 2^-23 of
 *   it (two roundings), so by 2^-16 absolutely: a code is certain unless the
 *   product lies within 2^-15 of a half-integer. Only there (one element in
 *   16,000) fp64 decides, where 127 a_j is exact and the quotient rounds to a
 *   half-integer only if it is one: codes depend on no rounding on the way.
 *   With SwiGLU the values are fp32 ones within 8 x 2^-24 (dsv4_swiglu_math.h), the
 *   product by 127 / amax within 10 x 2^-24 of at most 127: a code is certain
 *   outside 1.24 x 2^-14 (1.375 are taken) of a half-integer. Inside, and for the
 *   row's largest value, the SwiGLU is taken in fp64: codes and scale are those of
 *   fp64 values. Rows whose largest value is below 2^-60, beyond 2^120 or 2^98
 *   times below the largest up value, where fp32 may have lost some, compute
 *   everything in fp64.
 *
 * Bound: HBM for plain rows (8,192 of 4,096 bf16 19.6 us, 5.1 TB/s), the vector
 * unit for SwiGLU (38 instructions an element, 10 of the 13.3 us of 4,206 rows of
 * 2,048 whose bytes take 8.5; 24,576 rows 57, 4.4 TB/s; rows in fp64 190 rather
 * than 13.3), latency for a few rows (one of 4,096 2.6 us, less than the launch
 * costs its caller).
 */
#include "dsv4_elem.h"
#include "dsv4_internal.h"
#include "dsv4_swiglu_math.h"

namespace dsv4 {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int QU = 8;                              /* elements of a lane's unit  */
constexpr float ROUND_MAGIC = 12582912.0f;         /* 1.5 x 2^23: the low byte of v + this is rint(v) */

/* the unit's 8 elements (a, or gate and up) at element offset j */
template <int TYPE>
__device__ __forceinline__ void load8(const void *row, int j, u32x4 (&r)[TYPE == DSV4_HIP_F32 ? 2 : 1])
{
    const uint8_t *p = (const uint8_t *)row + (size_t)j * elem_bytes<TYPE>();
    r[0] = *gptr((const u32x4 *)p);
    if constexpr (TYPE == DSV4_HIP_F32) r[1] = *gptr((const u32x4 *)(p + 16));
}
template <int TYPE>
__device__ __forceinline__ void widen8(const u32x4 (&r)[TYPE == DSV4_HIP_F32 ? 2 : 1], float (&f)[QU])
{
    if constexpr (TYPE == DSV4_HIP_F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = __uint_as_float(r[i >> 2][i & 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = widen16<TYPE>(r[0][i] & 0xFFFFu);
            f[2 * i + 1] = widen16<TYPE>(r[0][i] >> 16);
        }
    }
}

/* largest of the wave's values, to every lane */
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
#define QMAX(CTRL, ROWS) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, (CTRL), (ROWS), 0xF, false))
    QMAX(DPP_QUAD_1032, 0xF);
    QMAX(DPP_QUAD_2301, 0xF);
    QMAX(DPP_ROW_HALF_MIRROR, 0xF);
    QMAX(DPP_ROW_MIRROR, 0xF);
    QMAX(DPP_ROW_BCAST15, 0xA);
    QMAX(DPP_ROW_BCAST31, 0xC);
#undef QMAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

/* the code in fp64: 127 a is exact for an fp32 a, and a quotient of such
 * numbers that is not a tie is too far from one for fp64 to make it one */
__device__ __forceinline__ uint32_t code64(double a, double amax) { return (uint32_t)(int)rint(a * 127.0 / amax); }

} // namespace

/* NW waves a row, NCH units of 8 elements a lane and pass; rows of more than
 * NCH * NW * 512 elements are read again in the second pass (from L2). */
template <int TYPE, bool SWIGLU, int NW, int NCH>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void k_quant_i8(QuantI8Args a)
{
    constexpr int RPW = NW == 1 ? 4 : 1;           /* rows of a workgroup         */
    constexpr int STEP = 64 * NW * QU;
    constexpr int RW = TYPE == DSV4_HIP_F32 ? 2 : 1;
    __shared__ uint32_t smax[NW];
    __shared__ float sumax[SWIGLU ? NW : 1];
    __shared__ unsigned long long smax64[RPW];     /* SwiGLU: the fp64 maximum's bits */
    const int lane = threadIdx.x & 63, wv = wave_in_group();
    const long row = (long)blockIdx.x * RPW + (NW == 1 ? wv : 0);
    if (row >= a.n) return;                        /* whole waves; one row a workgroup has no idle waves */
    unsigned long long *m64 = &smax64[NW == 1 ? wv : 0];
    if constexpr (SWIGLU) {
        if (lane == 0 && (NW == 1 || wv == 0)) *m64 = 0;       /* seen by all after the first barrier */
    }
    const size_t off = (size_t)row * (size_t)a.ld * elem_bytes<TYPE>();
    const uint8_t *pa = (const uint8_t *)a.a + off, *pu = SWIGLU ? (const uint8_t *)a.u + off : nullptr;
    const int j0 = ((NW == 1 ? 0 : wv * 64) + lane) * QU;
    const bool once = a.k <= NCH * STEP;
    const bool unbounded = SWIGLU && dsv4_swiglu::unbounded(a.limit);
    float umax = 0.0f;                             /* unbounded: the largest |u|  */

    u32x4 ra[NCH][RW], ru[SWIGLU ? NCH : 1][RW];
    float f[NCH][QU];
    auto fetch = [&](int base) {
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int j = base + j0 + c * STEP;
            if (j < a.k) {
                load8<TYPE>(pa, j, ra[c]);
                if constexpr (SWIGLU) load8<TYPE>(pu, j, ru[c]);
            }
        }
        if (unbounded) {
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                if (base + j0 + c * STEP >= a.k) continue;
                float u[QU];
                widen8<TYPE>(ru[c], u);
#pragma unroll
                for (int i = 0; i < QU; i++) umax = fmaxf(umax, fabsf(u[i]));
            }
        }
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int j = base + j0 + c * STEP;
            if (j < a.k) {
                widen8<TYPE>(ra[c], f[c]);
                if constexpr (SWIGLU) {
                    float u[QU];
                    widen8<TYPE>(ru[c], u);
#pragma unroll
                    for (int i = 0; i < QU; i++) f[c][i] = dsv4_swiglu::value32(f[c][i], u[i], a.limit);
                }
            } else {
#pragma unroll
                for (int i = 0; i < QU; i++) f[c][i] = 0.0f;
            }
        }
    };
    /* element i of the unit at j, exactly */
    auto exact = [&](int j) -> double {
        float g, u = 0.0f;
        Elem<TYPE, 1> e;
        float t[1];
        e.load(pa + (size_t)j * elem_bytes<TYPE>());
        e.get(t);
        g = t[0];
        if constexpr (SWIGLU) {
            e.load(pu + (size_t)j * elem_bytes<TYPE>());
            e.get(t);
            u = t[0];
            return dsv4_swiglu::value64(g, u, a.limit);
        }
        return (double)g;
    };

    /* the largest magnitude, as the bits of |a|: NaN above inf above all else */
    uint32_t m = 0, top[NCH];                      /* of the row, of each unit */
    auto tops = [&]() {
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            top[c] = 0;
#pragma unroll
            for (int i = 0; i < QU; i++) top[c] = max(top[c], __float_as_uint(f[c][i]) & 0x7FFFFFFFu);
        }
    };
    for (int base = 0; base < a.k; base += NCH * STEP) {
        fetch(base);
        tops();
#pragma unroll
        for (int c = 0; c < NCH; c++) m = max(m, top[c]);
    }
    m = wave_max_u32(m);
    if (unbounded) umax = __uint_as_float(wave_max_u32(__float_as_uint(umax)));
    if constexpr (NW > 1) {
        if (lane == 0) {
            smax[wv] = m;
            if (unbounded) sumax[wv] = umax;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) m = max(m, smax[w]);
        if (unbounded) {
#pragma unroll
            for (int w = 0; w < NW; w++) umax = fmaxf(umax, sumax[w]);
        }
    }
    m = (uint32_t)__builtin_amdgcn_readfirstlane((int)m);
    const float amax = __uint_as_float(m);
    double amax64 = (double)amax;
    /* SwiGLU: a row that takes fp64 values */
    const bool wide = SWIGLU && !dsv4_swiglu::fp32_serves(amax, a.limit > 0.0f ? fminf(umax, a.limit) : umax);
    bool bad = !SWIGLU && m >= 0x7F800000u;
    if constexpr (SWIGLU) {
        /* magnitudes order as their bits do, NaN above all: one LDS maximum of
         * the few candidates */
        auto take = [&](double v) {
            v = fabs(v);
            atomicMax(m64, (unsigned long long)__double_as_longlong(v == v ? v : __builtin_inf()));
        };
        if (wide) {
            for (int j = j0; j < a.k; j += STEP)
                for (int i = 0; i < QU; i++) take(exact(j + i));
        } else {
            const float near = amax * (1.0f - 0x1p-18f);
            for (int base = 0; base < a.k; base += NCH * STEP) {
                if (!once) {
                    fetch(base);
                    tops();
                }
#pragma unroll
                for (int c = 0; c < NCH; c++) {
                    if (__uint_as_float(top[c]) >= near)
                        for (int i = 0; i < QU; i++) {
                            const int j = base + j0 + c * STEP + i;
                            float t = 0.0f;
#pragma unroll
                            for (int q = 0; q < QU; q++) t = i == q ? f[c][q] : t;
                            if (fabsf(t) >= near) take(exact(j));
                        }
                }
            }
        }
        if constexpr (NW > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        amax64 = __longlong_as_double((long long)*(volatile unsigned long long *)m64);
        bad = !(amax64 <= 1.7976931348623157e308);
    }
    if (lane == 0 && (NW == 1 || wv == 0))
        a.S[row] = bad ? __builtin_nanf("") : amax64 > 0.0 ? (SWIGLU ? (float)(amax64 / 127.0) : amax / 127.0f) : 1.0f;

    /* tiny rows are multiplied by 2^64 first (exactly), so that 127 / amax
     * stays finite and the values normal */
    const bool tiny = !SWIGLU && amax < 0x1p-64f;
    const bool sure = !bad && !wide && amax > 0.0f;    /* the codes of fp32 products */
    const float inv = !sure ? 0.0f : SWIGLU ? (float)(127.0 / amax64) : 127.0f / (tiny ? amax * 0x1p64f : amax);
    constexpr float SURE = SWIGLU ? 0.5f - 0x1.6p-14f : 0.5f - 0x1p-15f;
    int8_t *q = a.Q + (size_t)row * (size_t)a.k;
    for (int base = 0; base < a.k; base += NCH * STEP) {
        if (!once) fetch(base);
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int j = base + j0 + c * STEP;
            if (j >= a.k) continue;
            uint32_t t[QU];
            float far = 0.0f;
            if (!sure || tiny) {
#pragma unroll
                for (int i = 0; i < QU; i++) f[c][i] = sure ? __fmul_rn(f[c][i], 0x1p64f) : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < QU; i++) {
                const float v = __fmul_rn(f[c][i], inv);
                const float s = __fadd_rn(v, ROUND_MAGIC);
                t[i] = __float_as_uint(s);
                far = fmaxf(far, fabsf(__fsub_rn(v, __fsub_rn(s, ROUND_MAGIC))));
            }
            if (wide && !bad && amax64 > 0.0) {
                for (int i = 0; i < QU; i++) t[i] = code64(exact(j + i), amax64);
            } else if (far > SURE) {
                for (int i = 0; i < QU; i++) {
                    const float v = __fmul_rn(f[c][i], inv);
                    if (fabsf(__fsub_rn(v, rintf(v))) > SURE) t[i] = code64(exact(j + i), amax64);
                }
            }
            u32x2 o;                               /* the low bytes, in order */
#pragma unroll
            for (int h = 0; h < 2; h++)
                o[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[4 * h + 3], t[4 * h + 2], 0x0C0C0400u),
                                             __builtin_amdgcn_perm(t[4 * h + 1], t[4 * h], 0x0C0C0400u), 0x05040100u);
            *(DSV4_GLOBAL u32x2 *)(q + j) = o;
        }
    }
}

/* Two units a lane: the smallest number of waves that holds the row, so that
 * it is read once and many rows are in flight. us, waves x units: 4,206 rows
 * of 2,048, SwiGLU, 1 x 4 15.4, 2 x 2 14.1, 4 x 1 14.0, 8 x 1 20.4; 2,048 of
 * 4,096 bf16 2 x 4 11.7, 4 x 2 9.0, 8 x 1 8.4; 8,192 of them 23.2, 19.6, 22.3;
 * 4,096 of 8,192 fp32 4 x 4 28.8, 8 x 2 28.3, 16 x 1 31.0; 5,000 of 14,336,
 * SwiGLU, 8 x 2 (each row read three times) 156, 16 x 2 111; 24,576 of 512,
 * SwiGLU, 1 x 1 20.6, 1 x 2 22.3, 2 x 1 27. */
template <int TYPE, bool SWIGLU, int NW, int NCH>
static hipError_t quant_i8_n(const QuantI8Args &a, hipStream_t st)
{
    constexpr int RPW = NW == 1 ? 4 : 1;
    hipLaunchKernelGGL((k_quant_i8<TYPE, SWIGLU, NW, NCH>), dim3((unsigned)((a.n + RPW - 1) / RPW)),
                       dim3(NW == 1 ? 256 : 64 * NW), 0, st, a);
    return hipGetLastError();
}

template <int TYPE, bool SWIGLU>
static hipError_t quant_i8_t(const QuantI8Args &a, hipStream_t st)
{
    if (a.k <= 512) return quant_i8_n<TYPE, SWIGLU, 1, 1>(a, st);
    if (a.k <= 1024) return quant_i8_n<TYPE, SWIGLU, 1, 2>(a, st);
    if (a.k <= 2048) return quant_i8_n<TYPE, SWIGLU, 2, 2>(a, st);
    if (a.k <= 4096) return quant_i8_n<TYPE, SWIGLU, 4, 2>(a, st);
    if (a.k <= 8192) return quant_i8_n<TYPE, SWIGLU, 8, 2>(a, st);
    return quant_i8_n<TYPE, SWIGLU, 16, 2>(a, st);
}

hipError_t quant_i8_launch(const QuantI8Args &a, int type, bool swiglu, hipStream_t st)
{
    if (a.n <= 0 || a.n >= 1 << 22 || a.k <= 0 || a.k > 1 << 24 || a.k % QU) return hipErrorInvalidValue;
    switch (type) {
    case DSV4_HIP_F32: return swiglu ? quant_i8_t<DSV4_HIP_F32, true>(a, st) : quant_i8_t<DSV4_HIP_F32, false>(a, st);
    case DSV4_HIP_BF16: return swiglu ? quant_i8_t<DSV4_HIP_BF16, true>(a, st) : quant_i8_t<DSV4_HIP_BF16, false>(a, st);
    case DSV4_HIP_F16: return swiglu ? quant_i8_t<DSV4_HIP_F16, true>(a, st) : quant_i8_t<DSV4_HIP_F16, false>(a, st);
    default: return hipErrorInvalidValue;
    }
}

} // namespace dsv4
