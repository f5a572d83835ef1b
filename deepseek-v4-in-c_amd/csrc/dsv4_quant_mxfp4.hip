/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_quant_mxfp4.hip - rows (or columns) to 4-bit floating point in blocks of
 * 32 with one power of two each, the operands of the 4-bit products: tokens,
 * weights, the experts' SwiGLU output straight from the gate and up products,
 * and by columns the operands of a backward pass.
 *
 * A block's byte is 127 + e with 2^e the least power of two that keeps 6 * 2^e
 * at or above the block's largest magnitude, clamped to [0, 254]; 127 for a block
 * of zeros. A code is the e2m1 value nearest to a / 2^e, ties to the even code
 * (v_cvt_scalef32_pk_fp4_f32 rounds so; checked against comparisons with the
 * seven borders on 60,000 values and at every border and its neighbours). The
 * division is a multiplication by a power of two, exact: what leaves fp32's
 * range downwards is far below the least border. A block with a value that is
 * not finite has byte 255 and codes 0.
 *
 * EXACT CODES OF SWIGLU VALUES
 *   The fp32 values are within 8 x 2^-24 of the exact ones (dsv4_swiglu_math.h).
 *   A code is certain if the value moved by 2^-20 of itself either way has the
 *   same one, the byte if the block's largest so moved has; where not (some
 *   element in 2^17) fp64 decides. Blocks whose largest value is below 2^-60,
 *   beyond 2^120 or 2^98 times below the largest up value, where fp32 may have
 *   lost some, compute everything in fp64.
 */
#include "dsv4_elem.h"
#include "dsv4_internal.h"
#include "dsv4_swiglu_math.h"

namespace dsv4 {

namespace {

constexpr int MU = 8;                              /* elements of a lane's unit */

template <int TYPE>
__device__ __forceinline__ void load8(const uint8_t *p, u32x4 (&r)[TYPE == DSV4_HIP_F32 ? 2 : 1])
{
    r[0] = __builtin_nontemporal_load(gptr((const u32x4 *)p));
    if constexpr (TYPE == DSV4_HIP_F32) r[1] = __builtin_nontemporal_load(gptr((const u32x4 *)(p + 16)));
}
template <int TYPE>
__device__ __forceinline__ void widen8(const u32x4 (&r)[TYPE == DSV4_HIP_F32 ? 2 : 1], float (&f)[MU])
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

/* largest of the four lanes that hold a block */
__device__ __forceinline__ uint32_t quad_max(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_1032, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_2301, 0xF, 0xF, false));
}

/* the byte of a block whose largest magnitude has these fp32 bits (NaN above
 * infinity above all else): 6 = 1.5 * 2^2 */
__device__ __forceinline__ uint32_t mxfp4_byte(uint32_t m)
{
    const int b = (int)(m >> 23) - 2 + ((m & 0x7FFFFFu) > 0x400000u);
    return m >= 0x7F800000u ? 255u : m == 0u ? 127u : (uint32_t)max(b, 0);
}
/* 2^(127 - byte) for bytes up to 253, all that finite fp32 values have */
__device__ __forceinline__ float mxfp4_inverse(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }

/* eight codes of values already divided */
__device__ __forceinline__ uint32_t mxfp4_codes(const float (&v)[MU])
{
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], 1.0f, 3);
}

/* the byte and a code from fp64 values */
__device__ __forceinline__ uint32_t mxfp4_byte64(double m)
{
    if (!(m <= 1.7976931348623157e308)) return 255u;
    if (m == 0.0) return 127u;
    const uint64_t u = (uint64_t)__double_as_longlong(m);
    const int b = (int)(u >> 52) - 1023 + 127 - 2 + ((u & 0xFFFFFFFFFFFFFull) > 0x8000000000000ull);
    return (uint32_t)min(max(b, 0), 254);
}
__device__ __forceinline__ uint32_t mxfp4_code64(double v)
{
    const double a = fabs(v);
    const uint32_t c = (a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0);
    return c | (__double_as_longlong(v) < 0 ? 8u : 0u);
}

} // namespace

/* Four lanes hold a block, eight elements each; a thread takes NU units, 256
 * apart: two of 16-bit elements where the device is full, else one. us, NU 1 / 2 / 4:
 * 1,024 rows of 4,096 bf16 2.7 / 3.3 / 3.6, 1,600 4.1 / 3.9 / 4.6; 4,206 of 2,048 5.3 /
 * 4.8 / 5.2, SwiGLU 10.7 / 11.6 / 13.7; 24,576 rows 23.1 / 20.9 / 21.0, SwiGLU 43.9 /
 * 44.3 / 44.0; fp32 333 rows of 4,096 2.7 / 2.9 / 3.4, 8,192 rows 27.8 / 28.1 / 28.8.
 * Bound: HBM (24,576 rows 6.1 TB/s, SwiGLU 5.2), the vector unit for SwiGLU of fewer
 * rows (4,206: 3.6 TB/s), latency for a few. */
template <int TYPE, bool SWIGLU, int NU>
__global__ __launch_bounds__(256) void k_quant_mxfp4(QuantMxfp4Args a)
{
    constexpr int RW = TYPE == DSV4_HIP_F32 ? 2 : 1, EB = elem_bytes<TYPE>();
    const uint32_t ku = (uint32_t)a.k / MU, units = (uint32_t)((size_t)a.n * ku);
    const uint32_t u0 = blockIdx.x * (256u * NU) + threadIdx.x;
    const bool flat = a.ld == a.k, unbounded = SWIGLU && dsv4_swiglu::unbounded(a.limit);
    u32x4 ra[NU][RW], ru[SWIGLU ? NU : 1][RW];
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const uint32_t u = u0 + 256u * i;
        if (u >= units) break;
        size_t at = (size_t)u * MU;
        if (!flat) {
            const uint32_t row = u / ku;
            at = (size_t)row * (size_t)a.ld + (size_t)(u - row * ku) * MU;
        }
        load8<TYPE>((const uint8_t *)a.a + at * EB, ra[i]);
        if constexpr (SWIGLU) load8<TYPE>((const uint8_t *)a.u + at * EB, ru[i]);
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const uint32_t u = u0 + 256u * i;
        if (u >= units) break;                     /* whole blocks: units is a multiple of four */
        float f[MU], up[MU];
        widen8<TYPE>(ra[i], f);
        float gate[MU];
        uint32_t umax = 0;
        if constexpr (SWIGLU) {
            widen8<TYPE>(ru[i], up);
#pragma unroll
            for (int e = 0; e < MU; e++) {
                gate[e] = f[e];
                if (unbounded) umax = max(umax, __float_as_uint(up[e]) & 0x7FFFFFFFu);
                f[e] = dsv4_swiglu::value32(f[e], up[e], a.limit);
            }
        }
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < MU; e++) m = max(m, __float_as_uint(f[e]) & 0x7FFFFFFFu);
        m = quad_max(m);
        uint32_t byte = mxfp4_byte(m), q;
        float v[MU];
        if constexpr (!SWIGLU) {
            const float inv = mxfp4_inverse(byte);
#pragma unroll
            for (int e = 0; e < MU; e++) v[e] = __fmul_rn(f[e], inv);
            q = byte == 255u ? 0u : mxfp4_codes(v);
        } else {
            if (unbounded) umax = quad_max(umax);
            const float amax = __uint_as_float(m);
            const float um = __uint_as_float(umax);
            /* the same in the four lanes of a block, from here to the codes */
            const bool wide = !dsv4_swiglu::fp32_serves(amax, a.limit > 0.0f ? fminf(um, a.limit) : um);
            const bool far = mxfp4_byte(__float_as_uint(__fmul_rn(amax, 1.0f - 0x1p-20f))) ==
                             mxfp4_byte(__float_as_uint(__fmul_rn(amax, 1.0f + 0x1p-20f)));
            if (wide || !far) {
                double top = 0.0;
#pragma unroll 1
                for (int e = 0; e < MU; e++) {
                    float g1 = gate[0], u1 = up[0];
#pragma unroll
                    for (int j = 1; j < MU; j++) {
                        g1 = e == j ? gate[j] : g1;
                        u1 = e == j ? up[j] : u1;
                    }
                    const double d = fabs(dsv4_swiglu::value64(g1, u1, a.limit));
                    top = d == d ? (d > top ? d : top) : __builtin_inf();
                }
                top = fmax(top, __shfl_xor(top, 1, 64));
                top = fmax(top, __shfl_xor(top, 2, 64));
                byte = mxfp4_byte64(top);
            }
            const float inv = mxfp4_inverse(byte);
            float lo[MU];
#pragma unroll
            for (int e = 0; e < MU; e++) {
                v[e] = __fmul_rn(f[e], inv * (1.0f + 0x1p-20f));
                lo[e] = __fmul_rn(f[e], inv * (1.0f - 0x1p-20f));
            }
            q = mxfp4_codes(v);
            if (byte == 255u) {
                q = 0;
            } else if (wide || q != mxfp4_codes(lo)) {
                const double inv64 = __longlong_as_double((long long)(1023 + 127 - (int)byte) << 52);
                q = 0;
#pragma unroll 1
                for (int e = 0; e < MU; e++) {
                    float g1 = gate[0], u1 = up[0];
#pragma unroll
                    for (int j = 1; j < MU; j++) {
                        g1 = e == j ? gate[j] : g1;
                        u1 = e == j ? up[j] : u1;
                    }
                    q |= mxfp4_code64(dsv4_swiglu::value64(g1, u1, a.limit) * inv64) << (4 * e);
                }
            }
        }
        ((DSV4_GLOBAL uint32_t *)a.Q)[u] = q;
        if ((threadIdx.x & 3) == 0) ((DSV4_GLOBAL uint8_t *)a.S)[u / 4] = (uint8_t)byte;
    }
}

/* Columns: a wave takes 32 rows of 64 columns, one a lane, so that a block lies in
 * one lane; eight waves take as many blocks of the same columns and meet in LDS,
 * from which 128-byte pieces of a's columns leave. Every load is made, from an
 * element that is there, and what lies behind the last row is zeroed afterwards:
 * loads under conditions waited for each other. Bound: the rows' latency, then
 * HBM (1,024 rows of 4,096 bf16 3.3 us, 2,803 6.7, 24,576 of 2,048 28 us, 4.6 TB/s;
 * under conditions 9.9 and 11.6; two columns a lane 4.0, 7.4 and 27, four waves
 * 3.3, 6.7 and 29). */
template <int TYPE>
__global__ __launch_bounds__(512) void k_quant_mxfp4_t(QuantMxfp4Args a)
{
    constexpr int NC = 64, NB = 8, EB = elem_bytes<TYPE>(), LD = NB * 16 + 16;
    __shared__ __align__(16) uint8_t codes[NC * LD];
    __shared__ __align__(8) uint8_t bytes[NC][NB];
    const int lane = threadIdx.x & 63, wave = wave_in_group();
    const uint32_t ct = ((uint32_t)a.k + NC - 1) / NC;
    const int c0 = (int)(blockIdx.x % ct) * NC, b0 = (int)(blockIdx.x / ct) * NB, nb = (a.n + 31) / 32;
    const int r0 = (b0 + wave) * 32, rows = max(a.n - r0, 0);
    const uint8_t *src =
        (const uint8_t *)a.a + ((size_t)min(r0, a.n - 1) * (size_t)a.ld + min(c0 + lane, a.k - 1)) * EB;
    const size_t step = (size_t)a.ld * EB;
    uint32_t raw[32];
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const uint8_t *p = src + (size_t)min(i, max(rows - 1, 0)) * step;
        if constexpr (EB == 4) raw[i] = *gptr((const uint32_t *)p);
        else raw[i] = *gptr((const uint16_t *)p);
    }
    if (rows < 32) {
#pragma unroll
        for (int i = 0; i < 32; i++) raw[i] = i < rows ? raw[i] : 0u;
    }
    auto elem = [&](int i) -> float {
        if constexpr (EB == 4) return __uint_as_float(raw[i]);
        else return widen16<TYPE>(raw[i]);
    };
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) m = max(m, __float_as_uint(elem(i)) & 0x7FFFFFFFu);
    const uint32_t byte = mxfp4_byte(m);
    const float inv = mxfp4_inverse(byte);
    u32x4 q;
#pragma unroll
    for (int d = 0; d < 4; d++) {
        float v[MU];
#pragma unroll
        for (int e = 0; e < MU; e++) v[e] = __fmul_rn(elem(8 * d + e), inv);
        q[d] = byte == 255u ? 0u : mxfp4_codes(v);
    }
    *(u32x4 *)(codes + lane * LD + 16 * wave) = q;
    bytes[lane][wave] = (uint8_t)byte;
    __syncthreads();
    const int col = threadIdx.x / NB, b = threadIdx.x % NB;
    if (c0 + col >= a.k || b0 + b >= nb) return;
    const size_t at = (size_t)(c0 + col) * nb + b0 + b;
    *(DSV4_GLOBAL u32x4 *)(a.Q + 16 * at) = *(const u32x4 *)(codes + col * LD + 16 * b);
    ((DSV4_GLOBAL uint8_t *)a.S)[at] = bytes[col][b];
}

template <int TYPE>
static hipError_t quant_mxfp4_t(const QuantMxfp4Args &a, Mxfp4Rows rows, hipStream_t st)
{
    if (rows == MXFP4_COLUMNS) {
        const size_t groups = (((size_t)a.n + 255) / 256) * (((size_t)a.k + 63) / 64);
        if (groups >= 1u << 23) return hipErrorInvalidConfiguration;
        hipLaunchKernelGGL(k_quant_mxfp4_t<TYPE>, dim3((unsigned)groups), dim3(512), 0, st, a);
        return hipGetLastError();
    }
    const size_t units = (size_t)a.n * (a.k / MU);
    if (units >> 32) return hipErrorInvalidConfiguration;
    if (rows == MXFP4_SWIGLU)
        hipLaunchKernelGGL((k_quant_mxfp4<TYPE, true, 1>), dim3((unsigned)((units + 255) / 256)), dim3(256), 0, st, a);
    else if (TYPE != DSV4_HIP_F32 && units > 5u << 17)
        hipLaunchKernelGGL((k_quant_mxfp4<TYPE, false, 2>), dim3((unsigned)((units + 511) / 512)), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_quant_mxfp4<TYPE, false, 1>), dim3((unsigned)((units + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t quant_mxfp4_launch(const QuantMxfp4Args &a, int type, Mxfp4Rows rows, hipStream_t st)
{
    if (a.n <= 0 || a.k <= 0 || (rows != MXFP4_COLUMNS && a.k % 32)) return hipErrorInvalidValue;
    switch (type) {
    case DSV4_HIP_F32: return quant_mxfp4_t<DSV4_HIP_F32>(a, rows, st);
    case DSV4_HIP_BF16: return quant_mxfp4_t<DSV4_HIP_BF16>(a, rows, st);
    case DSV4_HIP_F16: return quant_mxfp4_t<DSV4_HIP_F16>(a, rows, st);
    default: return hipErrorInvalidValue;
    }
}

} // namespace dsv4
