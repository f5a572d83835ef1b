/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_gemm_i8.hip - products of 8-bit integers with a scale for each token
 * and each weight row:
 *   C[m][n] = Sa[m] * Sw[n] * sum_k Aq[m][k] * W[n][k]
 * and the same for every expert's bucket of rows (its own W and Sw, rows
 * taken from the tokens through row_tok).
 *
 * The sum is exact in 32-bit integers for K <= 131,056 (codes -128..127), in
 * any order, so every form and split gives the same bits. The result is
 * ((float)sum * Sa[m]) * Sw[n] in fp32, rounded once more to a 16-bit output.
 *
 * v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive codes of row l % 16 of A
 * and of column l % 16 of B, element e of lane l of the result is row
 * 4 (l / 16) + e, column l % 16. Weight rows are the A operand, tokens the B
 * operand. Any order of k works as long as both operands use the same one, so
 * the four lane groups may take their 16 codes from wherever loads like best.
 */
#include "dsv4_elem.h"
#include "dsv4_internal.h"

namespace dsv4 {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr uint32_t I8_OOB = 0x80000000u;           /* beyond every buffer: reads zeros */

__device__ __forceinline__ __amdgpu_buffer_rsrc_t i8_rsrc(const void *p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)bytes, 0x00020000);
}
/* The whole offset goes into the per-lane part: the range check subtracts the
 * scalar part from the buffer's size, which wraps for a buffer shorter than
 * that (a single row). */
template <int CPOL>
__device__ __forceinline__ v4i i8_ld16(__amdgpu_buffer_rsrc_t r, uint32_t voff)
{
    return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, 0, CPOL));
}

/* what one workgroup multiplies: rows r0 .. r0 + rows of the product against
 * matrix w (scales s) */
struct Tile {
    const uint8_t *w;
    const float *s;
    int r0, rows;
    bool bad;                                      /* the table's entry is not an int8 N x K matrix */
};

/* Tile `t` of the buckets ex_off[0 .. E], each cut into tiles of TR rows;
 * rows == 0 past the last tile. Every wave finds it by itself: a lane counts
 * the tiles of E / 64 experts, a scan over the lanes finds the one that holds
 * t. Offsets are clamped to [0, R], so no table makes a row out of range. */
template <int TR>
__device__ __forceinline__ Tile bucket_tile(const I8Args &a, int t, int lane)
{
    const int E = a.n_experts, per = (E + 63) / 64;
    auto clampr = [&](int v) { return min(max(v, 0), a.M); };
    int mine = 0;
    int lo = lane * per < E ? clampr(a.ex_off[lane * per]) : 0;
    for (int i = 0; i < per; i++) {
        const int e = lane * per + i;
        if (e < E) {
            const int hi = clampr(a.ex_off[e + 1]);
            mine += (max(hi - lo, 0) + TR - 1) / TR;
            lo = hi;
        }
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    Tile o;
    o.w = nullptr; o.s = nullptr; o.r0 = 0; o.rows = 0; o.bad = false;
    const uint64_t past = __ballot(incl > t);
    if (!past) return o;
    const int L = __builtin_ctzll(past);
    int left = t - __builtin_amdgcn_readlane(incl - mine, L);
    int e = L * per;
    lo = clampr(a.ex_off[e]);
    for (;; e++) {                                 /* ends within the lane's experts: they hold tile t */
        const int hi = clampr(a.ex_off[e + 1]);
        const int n = max(hi - lo, 0), tiles = (n + TR - 1) / TR;
        if (left < tiles || e + 1 >= E) {
            o.r0 = lo + left * TR;
            o.rows = min(TR, n - left * TR);
            break;
        }
        left -= tiles;
        lo = hi;
    }
    const DSV4QMat m = ld_uniform(a.table, __builtin_amdgcn_readfirstlane(e));
    o.w = (const uint8_t *)m.w;
    o.s = (const float *)m.s;
    o.bad = m.wdt != DSV4_WI8 || m.rows != a.N || m.cols != a.K || !m.w || !m.s || ((uintptr_t)m.w & 15u) ||
            ((uintptr_t)m.s & 3u);
    o.r0 = __builtin_amdgcn_readfirstlane(o.r0);
    o.rows = __builtin_amdgcn_readfirstlane(o.rows);
    return o;
}

/* one result: element n of row r */
template <int OUT>
__device__ __forceinline__ void i8_store(void *C, size_t i, float v)
{
    if constexpr (OUT == DSV4_HIP_F32) ((float *)C)[i] = v;
    else ((uint16_t *)C)[i] = (uint16_t)narrow16<OUT>(v);
}

} // namespace

/* ------------------------------------------------------- few rows -------
 * A workgroup of four waves takes 16 weight rows and up to 16 TT rows of
 * tokens; the waves share out K in blocks of 128 and add their sums in LDS.
 * Both operands go straight to registers. Bound: the weight stream. */
template <int TT, bool GROUPED, int OUT>
__global__ __launch_bounds__(256) void k_i8_stream(I8Args a)
{
    constexpr int NW = 4, B = 2;                   /* waves along K, blocks of 128 in flight a wave */
    __shared__ int sum[NW][TT][256];
    const int lane = threadIdx.x & 63, wave = wave_in_group();
    const int r = lane & 15, g = lane >> 4;
    const int slabs = (a.N + 15) / 16, tile = blockIdx.x / slabs, n0 = (blockIdx.x - tile * slabs) * 16;
    Tile t;
    if constexpr (GROUPED) {
        t = bucket_tile<16 * TT>(a, tile, lane);
        if (t.rows <= 0) return;
    } else {
        t.w = a.W; t.s = a.Sw; t.bad = false;
        t.r0 = tile * 16 * TT;
        t.rows = min(16 * TT, a.M - t.r0);
    }
    if (GROUPED && t.bad) {
        if (threadIdx.x == 0) atomicOr(a.status, ST_BAD_DESCRIPTOR);
        for (int i = threadIdx.x; i < t.rows * 16; i += 256)
            if (n0 + (i & 15) < a.N) i8_store<OUT>(a.C, (size_t)(t.r0 + i / 16) * a.N + n0 + (i & 15), __builtin_nanf(""));
        return;
    }
    const uint32_t K = (uint32_t)a.K;
    const __amdgpu_buffer_rsrc_t rw = i8_rsrc(t.w + (size_t)n0 * K, (uint32_t)min(16, a.N - n0) * K);
    const uint8_t *xb = GROUPED ? a.Aq : a.Aq + (size_t)t.r0 * K;
    const __amdgpu_buffer_rsrc_t rx = i8_rsrc(xb, GROUPED ? (uint32_t)a.n_a * K : (uint32_t)t.rows * K);
    /* source row of product row i of the tile; -1 where there is none */
    auto src_of = [&](int i) -> int {
        if (i >= t.rows) return -1;
        if (!GROUPED) return i;
        const int s = a.row_tok ? a.row_tok[t.r0 + i] : t.r0 + i;
        return (unsigned)s < (unsigned)a.n_a ? s : -1;
    };
    uint32_t xo[TT];
#pragma unroll
    for (int u = 0; u < TT; u++) {
        const int s = src_of(16 * u + r);
        xo[u] = s < 0 ? I8_OOB : (uint32_t)s * K + 16u * g;
    }
    const uint32_t wo = (uint32_t)r * K + 16u * g;
    const int nblk = (a.K + 127) / 128;
    v4i acc[TT];
#pragma unroll
    for (int u = 0; u < TT; u++) acc[u] = v4i{0, 0, 0, 0};
    /* codes past K: the tokens' read as zeros, whatever the weights' are */
    for (int b0 = wave; b0 < nblk; b0 += NW * B) {
        v4i w[B][2], x[B][2][TT];
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int c = (b0 + NW * b) * 128 + 64 * h;
                const bool in = c + 16 * g < a.K;
                w[b][h] = i8_ld16<2>(rw, in ? wo + (uint32_t)c : I8_OOB);
#pragma unroll
                for (int u = 0; u < TT; u++) x[b][h][u] = i8_ld16<0>(rx, in && xo[u] != I8_OOB ? xo[u] + (uint32_t)c : I8_OOB);
            }
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int u = 0; u < TT; u++)
                    acc[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[b][h], x[b][h][u], acc[u], 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < TT; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) sum[wave][u][(4 * g + e) * 16 + r] = acc[u][e];
    __syncthreads();
    /* thread: weight row threadIdx % 16 of the workgroup's, row threadIdx / 16 */
    const int n = threadIdx.x & 15, m16 = threadIdx.x >> 4;
    if (n0 + n >= a.N) return;
    const float sw = t.s[n0 + n];
#pragma unroll
    for (int u = 0; u < TT; u++) {
        const int i = 16 * u + m16;
        if (i >= t.rows) continue;
        int v = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) v += sum[w][u][n * 16 + m16];
        const int s = src_of(i);
        float f = __builtin_nanf("");
        if (s >= 0) f = (float)v * (GROUPED ? a.Sa[s] : a.Sa[t.r0 + s]) * sw;
        else if (n == 0) atomicOr(a.status, ST_BAD_EXPERT_ID);
        i8_store<OUT>(a.C, (size_t)(t.r0 + i) * a.N + n0 + n, f);
    }
}

template <bool GROUPED, int OUT>
static hipError_t i8_stream(const I8Args &a, hipStream_t st)
{
    constexpr int TT = 4, TR = 16 * TT;
    const long tiles = GROUPED ? a.M / TR + (a.n_experts < a.M ? a.n_experts : a.M) : (a.M + TR - 1) / TR;
    const long groups = tiles * ((a.N + 15) / 16);
    if (groups >= 1L << 24) return hipErrorInvalidConfiguration;   /* 2^32 threads */
    hipLaunchKernelGGL((k_i8_stream<TT, GROUPED, OUT>), dim3((unsigned)groups), dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t gemm_i8_launch(const I8Args &a, int out_type, hipStream_t st)
{
    if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.K % 16) return hipErrorInvalidValue;
    const bool grouped = a.table != nullptr;
    switch (out_type) {
    case DSV4_HIP_F32: return grouped ? i8_stream<true, DSV4_HIP_F32>(a, st) : i8_stream<false, DSV4_HIP_F32>(a, st);
    case DSV4_HIP_BF16: return grouped ? i8_stream<true, DSV4_HIP_BF16>(a, st) : i8_stream<false, DSV4_HIP_BF16>(a, st);
    case DSV4_HIP_F16: return grouped ? i8_stream<true, DSV4_HIP_F16>(a, st) : i8_stream<false, DSV4_HIP_F16>(a, st);
    default: return hipErrorInvalidValue;
    }
}

} // namespace dsv4
