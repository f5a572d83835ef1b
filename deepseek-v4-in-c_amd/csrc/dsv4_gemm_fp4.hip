/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_gemm_fp4.hip - products of 4-bit rows, both operands e2m1 codes with one
 * E8M0 scale for 32 values along the sum:
 *   C[m][n] = sum_b 2^(sa[m][b] - 127) 2^(sw[n][b] - 127) sum_{k in b} a[m][k] w[n][k]
 * and the same for every expert's bucket of rows (its own matrix, rows taken
 * from the tokens through row_tok).
 *
 * The matrix instructions take codes and scale bytes as they are stored: no
 * value is decoded, the sum stays in their fp32 accumulators, each result is
 * rounded once more for a 16-bit output. A scale byte of 255 is NaN, and so is
 * every result that it meets. Products of codes are multiples of 1/4 up to 36,
 * so within a block, and over blocks of like scales, sums are exact; the whole
 * is nearer to the exact sum than fp32 additions one after the other (4,096
 * values, scales over 18 powers of two: relative L2 1.3e-7 against 4.9e-7).
 *
 * v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds the 32 codes (16 bytes, low
 * nibble first) of row l % 16, block l / 16, and their scale in the byte of a
 * register that the instruction names; element e of lane l of the result is row
 * 4 (l / 16) + e of A, row l % 16 of B. v_mfma_scale_f32_32x32x64_f8f6f4: row l %
 * 32, block l / 32; element e is row 8 (e / 4) + 4 (l / 32) + e % 4 of A, row l %
 * 32 of B. Weight rows are the A operand, tokens the B operand. Registers alone
 * reach 5.3 PFLOP/s with the first and 6.8 with the second (10 nominal).
 *
 * Codes past a row's end (K no multiple of a load's) come as zeros for the
 * tokens, and scales there as finite ones, so whatever the weights' side reads
 * adds nothing.
 */
#include "dsv4_bucket.h"
#include "dsv4_elem.h"

namespace dsv4 {

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));
template <int N> struct IC { static constexpr int value = N; };

using Fp4Bucket = Bucket<uint8_t>;

/* whether a table's entry is an FP4 N x K matrix */
__device__ __forceinline__ auto fp4_matrix(const Fp4Args &a)
{
    return [&a](const DSV4QMat &m) {
        return m.wdt == DSV4_WFP4 && m.rows == a.N && m.cols == a.K && m.blk_r == 1 && m.blk_c == 32 && m.w && m.s &&
               !((uintptr_t)m.w & 15u);
    };
}

/* W scale bytes of a row from block b on (nb blocks a row), W = 8 or 16; blocks past
 * the row's end 0. Rows of scales have any alignment. The last bytes come with those
 * before them, shifted: a byte a time they waited for each other (1 row of 2048 x
 * 2816 3.8 us, 3.1 so). */
template <int W> struct Fp4Scales;
template <> struct Fp4Scales<8> { typedef u32x2 type; typedef uint64_t bits; };
template <> struct Fp4Scales<16> { typedef u32x4 type; typedef unsigned __int128 bits; };
template <int W>
__device__ __forceinline__ typename Fp4Scales<W>::type fp4_scales(const uint8_t *row, int b, int nb)
{
    using T = typename Fp4Scales<W>::type;
    using B = typename Fp4Scales<W>::bits;
    typedef T at_any __attribute__((aligned(1)));
    if (b + W <= nb) return *(const DSV4_GLOBAL at_any *)(row + b);
    if (b >= nb) return T(0);
    if (nb >= W) {
        const T v = *(const DSV4_GLOBAL at_any *)(row + nb - W);
        return __builtin_bit_cast(T, __builtin_bit_cast(B, v) >> (8 * (b + W - nb)));
    }
    uint32_t v[W];
#pragma unroll
    for (int i = 0; i < W; i++) v[i] = gptr(row)[min(b + i, nb - 1)];
    T o(0);
#pragma unroll
    for (int i = 0; i < W; i++) o[i / 4] |= b + i < nb ? v[i] << (8 * (i & 3)) : 0u;
    return o;
}

__device__ __forceinline__ v8i fp4_operand(const v4i &v)
{
    return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}
__device__ __forceinline__ f32x4 fp4_mfma16(const v4i &w, const v4i &x, f32x4 c, uint32_t sw, uint32_t sx)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(w), fp4_operand(x), c, 4, 4, 0, (int)sw, 0, (int)sx);
}
/* B: which byte of the scale registers */
template <int B>
__device__ __forceinline__ f32x16 fp4_mfma32(const v4i &w, const v4i &x, f32x16 c, uint32_t sw, uint32_t sx)
{
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(w), fp4_operand(x), c, 4, 4, B, (int)sw, B, (int)sx);
}

/* two results as 16-bit elements, rounded to nearest even */
template <int OUT>
__device__ __forceinline__ uint32_t fp4_pack(float a, float b)
{
    if constexpr (OUT == DSV4_HIP_BF16) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    }
}

/* one result: element i of C */
template <int OUT>
__device__ __forceinline__ void fp4_store(void *C, size_t i, float v)
{
    if constexpr (OUT == DSV4_HIP_F32) ((float *)C)[i] = v;
    else ((uint16_t *)C)[i] = (uint16_t)narrow16<OUT>(v);
}

/* rows of an expert whose table entry is no matrix of the product */
template <int OUT>
__device__ __forceinline__ void fp4_bad(const Fp4Args &a, const Fp4Bucket &t, int n0, int nf, int threads)
{
    if (threadIdx.x == 0) atomicOr(a.status, ST_BAD_DESCRIPTOR);
    for (int i = threadIdx.x; i < t.rows * nf; i += threads)
        fp4_store<OUT>(a.C, (size_t)(t.r0 + i / nf) * a.N + n0 + i % nf, __builtin_nanf(""));
}

/* the row of Aq that row i of the tile multiplies (from the tile's first on for
 * one matrix); -1: none */
template <bool GROUPED>
__device__ __forceinline__ int fp4_source(const Fp4Args &a, const Fp4Bucket &t, int i)
{
    if (i >= t.rows) return -1;
    if (!GROUPED) return i;
    const int s = a.row_tok ? a.row_tok[t.r0 + i] : t.r0 + i;
    return (unsigned)s < (unsigned)a.n_a ? s : -1;
}

} // namespace

/* --------------------------------------------------- K over the waves ---
 * A workgroup takes 16 features by 16 rows of one matrix, and its eight waves
 * share out K in pieces of 512 values: operands go straight to registers, a
 * whole piece's loads before its first product, and the sums meet in LDS, added
 * in wave order. No wave waits for another before the end, so a product too
 * small to fill the device costs one latency of its loads, not one a stage.
 * Bound: that latency (one token of 4096 x 4096 3.4 us, with weights from HBM 4.1, the
 * weights alone 1.4 at 6.2 TB/s; 64 x 32 tiles 6.1); with many rows the loads, 64 bytes of a row each. */
template <int OUT>
__global__ __launch_bounds__(512) void k_fp4_split(Fp4Args a)
{
    constexpr int NW = 8;
    __shared__ float sum[NW][256];
    const int lane = threadIdx.x & 63, wave = wave_in_group(), r16 = lane & 15, g = lane >> 4;
    const int nt = (a.N + 15) / 16, tile = blockIdx.x / nt, n0 = (blockIdx.x - tile * nt) * 16;
    const int r0 = tile * 16, rows = min(16, a.M - r0), nf = min(16, a.N - n0);
    const uint32_t KB = (uint32_t)a.K / 2;
    const int nb = a.K / 32;
    const __amdgpu_buffer_rsrc_t rw = buf_rsrc(a.W + (size_t)n0 * KB, (uint32_t)nf * KB);
    const __amdgpu_buffer_rsrc_t rx = buf_rsrc(a.Aq + (size_t)r0 * KB, (uint32_t)rows * KB);
    /* rows past the last: the last again, not stored */
    const int wr = min(r16, nf - 1), xr = min(r16, rows - 1);
    const uint8_t *ws = a.Sw + (size_t)(n0 + wr) * nb, *xs = a.As + (size_t)(r0 + xr) * nb;
    f32x4 acc = {0, 0, 0, 0};
    for (int p = wave; 16 * p < nb; p += NW) {
        v4i w[4], x[4];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const uint32_t at = 256u * p + 64u * s + 16u * g;
            const bool in = 16 * p + 4 * s + g < nb;
            w[s] = buf_ld16<0>(rw, in ? (uint32_t)wr * KB + at : BUF_OOB);
            x[s] = buf_ld16<0>(rx, in ? (uint32_t)xr * KB + at : BUF_OOB);
        }
        const u32x4 sw = fp4_scales<16>(ws, 16 * p, nb), sx = fp4_scales<16>(xs, 16 * p, nb);
#pragma unroll
        for (int s = 0; s < 4; s++) acc = fp4_mfma16(w[s], x[s], acc, sw[s] >> (8 * g), sx[s] >> (8 * g));
    }
    *(f32x4 *)&sum[wave][r16 * 16 + 4 * g] = acc;
    __syncthreads();
    const int o = threadIdx.x, n = o % 16, i = o / 16;
    if (i >= rows || n >= nf) return;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) v += sum[w][o];
    fp4_store<OUT>(a.C, (size_t)(r0 + i) * a.N + n0 + n, v);
}

/* ------------------------------------------- stages over the waves -----
 * A workgroup takes 32 features by 32 rows of one matrix, and its four waves
 * share out the stages of 256 values, each with a stage's place of its own in
 * LDS and all of the tile's results in registers: no wave waits for another
 * before the sums meet in LDS, added in wave order. A stage's loads are asked for
 * when the one before is in registers; other workgroups, four to a CU (103 registers;
 * LDS has room for five), hide their latency better than a second place does (64 x 4096 x 4096 4.5 us with either, 128 x
 * 4096 x 1024 4.5 against 3.2; eight waves 4.4 and 4.3; 64 rows a tile 5.9 and 3.6).
 * Bound: latency of launch, a few stages and the sums, then a CU's loads
 * (128 KB of operands a 32 x 32 tile at K = 4096). */
template <int OUT>
__global__ __launch_bounds__(256) void k_fp4_team(Fp4Args a)
{
    constexpr int NW = 4, F = 32, T = 32, LW = F / 8, LX = T / 8, LD = F + 4, STAGE = (F + T) * 128;
    static_assert(T * LD * 4 <= STAGE, "the sums take the stage's place");
    __shared__ __align__(16) uint8_t lds[NW * STAGE];
    const int lane = threadIdx.x & 63, wave = wave_in_group(), rr = lane & 31, g = lane >> 5;
    const int mt = (a.M + T - 1) / T, nt = (a.N + F - 1) / F, total = mt * nt, nb = a.K / 32;
    /* each XCD a contiguous run of tiles, row tiles first: it reads a weight once */
    const int per = total / 8, rest = total % 8, x = blockIdx.x % 8, y = blockIdx.x / 8;
    const int id = x * per + min(x, rest) + y, n0 = id / mt * F, r0 = id % mt * T;
    const int rows = min(T, a.M - r0), nf = min(F, a.N - n0);
    const uint32_t KB = (uint32_t)a.K / 2;
    const int nreal = (a.K + 255) / 256;
    const __amdgpu_buffer_rsrc_t rw = buf_rsrc(a.W + (size_t)n0 * KB, (uint32_t)nf * KB);
    const __amdgpu_buffer_rsrc_t rx = buf_rsrc(a.Aq + (size_t)r0 * KB, (uint32_t)rows * KB);
    uint8_t *const buf = lds + wave * STAGE;
    auto swz = [](int r, int c) { return c ^ ((r >> 1) & 7); };
    uint32_t wo[LW], xo[LX], xl[LX];               /* xl: of the last stage, pieces past K out of range */
#pragma unroll
    for (int i = 0; i < LW; i++) {
        const int r = 8 * i + lane / 8;
        wo[i] = r < nf ? (uint32_t)r * KB + 16u * (uint32_t)swz(r, lane & 7) : BUF_OOB;
    }
#pragma unroll
    for (int i = 0; i < LX; i++) {
        const int r = 8 * i + lane / 8, c = swz(r, lane & 7);
        xo[i] = r < rows ? (uint32_t)r * KB + 16u * (uint32_t)c : BUF_OOB;
        xl[i] = 8 * (nreal - 1) + c < nb ? xo[i] : BUF_OOB;
    }
    /* rows past the last: the last one's scales, not stored */
    const uint8_t *const ws = a.Sw + (size_t)(n0 + min(rr, nf - 1)) * nb;
    const uint8_t *const xs = a.As + (size_t)(r0 + min(rr, rows - 1)) * nb;
    u32x2 bw, bx;                                  /* the eight scale bytes of a stage */
    auto ask = [&](int st) {
        bw = fp4_scales<8>(ws, 8 * st, nb);
        bx = fp4_scales<8>(xs, 8 * st, nb);
#pragma unroll
        for (int i = 0; i < LW; i++) buf_dma16<0>(rw, wo[i] + 128u * (uint32_t)st, 0, buf + 1024 * i);
#pragma unroll
        for (int i = 0; i < LX; i++)
            buf_dma16<0>(rx, (st < nreal - 1 ? xo[i] : xl[i]) + 128u * (uint32_t)st, 0, buf + 128 * F + 1024 * i);
    };
    const uint32_t pick = g ? 0x07050301u : 0x06040200u;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0.0f;
    if (wave < nreal) ask(wave);
    for (int st = wave; st < nreal; st += NW) {
        wait_vm<0>();
        asm volatile("" ::: "memory");
        v4i w[4], v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            w[k] = *(const v4i *)(buf + rr * 128 + 16 * swz(rr, 2 * k + g));
            v[k] = *(const v4i *)(buf + 128 * (F + rr) + 16 * swz(rr, 2 * k + g));
        }
        const uint32_t sw = __builtin_amdgcn_perm(bw.y, bw.x, pick);
        const uint32_t sx = __builtin_amdgcn_perm(bx.y, bx.x, pick);
        __builtin_amdgcn_s_waitcnt(0xC07F);        /* the operands are in registers: the place is free */
        asm volatile("" ::: "memory");
        if (st + NW < nreal) ask(st + NW);
        acc = fp4_mfma32<0>(w[0], v[0], acc, sw, sx);
        acc = fp4_mfma32<1>(w[1], v[1], acc, sw, sx);
        acc = fp4_mfma32<2>(w[2], v[2], acc, sw, sx);
        acc = fp4_mfma32<3>(w[3], v[3], acc, sw, sx);
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {
        f32x4 o;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = acc[4 * q + e];
        *(f32x4 *)(buf + 4 * (rr * LD + 8 * q + 4 * g)) = o;
    }
    __syncthreads();
    static_assert(T * F == 4 * 64 * NW, "four results a thread");
    const int m = threadIdx.x / (F / 4), n = threadIdx.x % (F / 4) * 4;
    if (m >= rows || n >= nf) return;
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NW; k++) {
        const f32x4 t = *(const f32x4 *)(lds + k * STAGE + 4 * (m * LD + n));
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += t[e];
    }
    const size_t at = (size_t)(r0 + m) * a.N + n0 + n;
    if (n + 4 > nf) {
        for (int e = 0; e < nf - n; e++) fp4_store<OUT>(a.C, at + e, v[e]);
    } else if constexpr (OUT == DSV4_HIP_F32) {
        typedef f32x4 any __attribute__((aligned(4)));
        *(DSV4_GLOBAL any *)((float *)a.C + at) = v;
    } else {
        typedef u32x2 any __attribute__((aligned(2)));
        *(DSV4_GLOBAL any *)((uint16_t *)a.C + at) = u32x2{fp4_pack<OUT>(v[0], v[1]), fp4_pack<OUT>(v[2], v[3])};
    }
}

/* ------------------------------------------------------- many rows ------
 * A workgroup takes F features by T rows, its WR x WT waves each F / WR by T / WT
 * of them in 32 x 32 results. K goes in stages of 256 values, a staged row a
 * 128-byte line: both operands by loads straight to LDS into a ring of NST
 * stages (16-byte pieces XOR-swizzled by row), a wave reading the operands of
 * the next 64 values while it multiplies these. The scales of two stages, 16
 * bytes a row, go through a thread's registers (rows of scales have any
 * alignment) into one of two LDS tables; a lane picks the four bytes of its
 * block in each step with one permutation. One barrier a stage: after it every
 * wave's loads of the next stage have landed and no wave still reads this one,
 * so the stage NST ahead takes its place. The tile leaves through LDS as whole
 * 16-byte pieces of rows.
 * Bound, 256 x 256: the matrix instructions at the clock that power allows (4096^3
 * 36.5 to 39.4 us from card to card, 3.5 to 3.8 PFLOP/s; of it 9 us first loads and the
 * way out, as one workgroup has the CU). 128 x 128: a CU's loads, 32 KB a stage in 0.52 us (63 GB/s, alone
 * they reach 80): 2,803 x 1024 x 4096 13 us, in 128 x 96 tiles, which fill more of the
 * CUs, 12, 5 of them launch, first loads and the way out. Buckets: the weights'
 * stream (7 tokens, top 6 of 256 experts 2048 x 4096 35 us, 5.0 TB/s), with many rows
 * beside it the tokens and the results (4,096 tokens, Zipf, 300 us, 4.2 TB/s; without
 * products 294, without either of the two 276). */
template <int F, int T, int WR, int WT, int NST_> struct Fp4Tile {
    static constexpr int NWAVE = WR * WT, NT = 64 * NWAVE, NST = NST_;
    static constexpr int WI = F / WR / 32, U = T / WT / 32;
    static constexpr bool DEEP = WI * U <= 2;          /* few products a step: latencies of LDS show */
    static constexpr int OFF_X = F * 128, STAGE = (F + T) * 128;
    static constexpr int LW = F / 8 / NWAVE, LX = T / 8 / NWAVE, VM = LW + LX;
    static constexpr int RING = NST * STAGE, TABLE = NT * 16;
    static constexpr int out_ld(int eb) { return F * eb + 16; }
    /* tokens that leave together, whole row groups of every wave */
    static constexpr int out_rows(int eb)
    {
        int parts = 1;
        while (T / parts * out_ld(eb) > 160 * 1024 || T % (32 * WT * parts)) parts++;
        return T / parts;
    }
    static constexpr int lds(int eb)
    {
        return RING + 2 * TABLE > out_rows(eb) * out_ld(eb) ? RING + 2 * TABLE : out_rows(eb) * out_ld(eb);
    }
    static_assert(LW * NWAVE * 8 == F && LX * NWAVE * 8 == T && F + T <= NT && (NST - 1) * VM < 64 &&
                      lds(4) <= 160 * 1024 && WI >= 1 && U >= 1, "tile");
};

template <int F, int T, int WR, int WT, int NST, bool GROUPED, bool STREAM, int OUT>
__device__ __forceinline__ void fp4_tile_sum(const Fp4Args &a, const Fp4Bucket &t, int n0)
{
    using C = Fp4Tile<F, T, WR, WT, NST>;
    constexpr int U = C::U, WI = C::WI;
    extern __shared__ __align__(16) uint8_t lds[];
    uint8_t *const table = lds + C::RING;
    const int lane = threadIdx.x & 63, wave = wave_in_group();
    const int rr = lane & 31, g = lane >> 5, wr = wave % WR, wt = wave / WR;
    const int nb = a.K / 32;
    const int nf = min(F, a.N - n0);
    if (GROUPED && t.bad) {
        fp4_bad<OUT>(a, t, n0, nf, C::NT);
        return;
    }
    const uint32_t KB = (uint32_t)a.K / 2;
    /* stages, whole pairs of them: a way out between the two, or the last one
     * after the loop, cost registers that the large tiles do not have */
    const int nst = (a.K + 511) / 512 * 2;
    const size_t x0 = GROUPED ? 0 : (size_t)t.r0;
    const uint8_t *const wb = t.w + (size_t)n0 * KB, *const xb = a.Aq + x0 * KB;
    const uint32_t wlen = (uint32_t)nf * KB, xlen = (GROUPED ? (uint32_t)a.n_a : (uint32_t)t.rows) * KB;
    auto swz = [](int r, int c) { return c ^ ((r >> 1) & 7); };
    const int nreal = (a.K + 255) / 256;           /* stages with values */
    uint32_t wo[C::LW], xo[C::LX], xl[C::LX];      /* xl: of the last of them, pieces past K out of range */
#pragma unroll
    for (int i = 0; i < C::LW; i++) {
        const int r = 8 * (C::LW * wave + i) + lane / 8;
        wo[i] = (uint32_t)r * KB + 16u * (uint32_t)swz(r, lane & 7);
    }
    /* the weights of the ring's first stages before the tokens are looked up
     * (24,576 rows on 256 experts 2 %; where a tile is short it costs more: 42 rows 5 %) */
    constexpr bool AHEAD = GROUPED && F == 256;
    if constexpr (AHEAD) {
#pragma unroll
        for (int s = 0; s < NST; s++)
#pragma unroll
            for (int i = 0; i < C::LW; i++)
                buf_dma16<STREAM ? 2 : 0>(buf_rsrc(wb, s < nreal ? wlen : 0u), wo[i], s < nreal ? 128 * s : 0,
                                          lds + s * C::STAGE + 1024 * (C::LW * wave + i));
        asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int i = 0; i < C::LX; i++) {
        const int r = 8 * (C::LX * wave + i) + lane / 8, c = swz(r, lane & 7), s = fp4_source<GROUPED>(a, t, r);
        xo[i] = s < 0 ? BUF_OOB : (uint32_t)s * KB + 16u * (uint32_t)c;
        xl[i] = 8 * (nreal - 1) + c < nb ? xo[i] : BUF_OOB;
    }
    /* the row whose scales this thread fetches. Rows past the last weight row take
     * its, and so do tokens that are not there and threads without a row: what
     * they give is not stored, or multiplies zeros */
    const uint8_t *srow = t.s + (size_t)(n0 + min((int)threadIdx.x, nf - 1)) * nb;
    if ((int)threadIdx.x >= F && (int)threadIdx.x < F + T) {
        const int s = fp4_source<GROUPED>(a, t, (int)threadIdx.x - F);
        if (s >= 0) srow = a.As + (x0 + s) * (size_t)nb;
    }
    /* the scales of stages 2 pair and 2 pair + 1; of the last pair, which may end
     * inside 16, from the start. No branch, and few instructions: in the loop a
     * wave's own instructions are what small tiles wait for. */
    const int last = nst / 2 - 1;
    const u32x4 ends = fp4_scales<16>(srow, 16 * last, nb);
    auto fetch_scales = [&](int pair) -> u32x4 {   /* w: 16 bytes that are there */
        return *(const DSV4_GLOBAL u32x4_any *)(nb < 16 ? t.w : srow + min(16 * pair, nb - 16));
    };
    auto put_scales = [&](int pair, const u32x4 &v) {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = pair == last ? ends[j] : v[j];
        *(u32x4 *)(table + (pair & 1) * C::TABLE + 16 * threadIdx.x) = o;
    };
    /* load i of a wave's share of stage st; past the end zeros, no traffic (an
     * empty buffer, and no scalar offset: the range check takes it off the size) */
    auto issue = [&](int st, int slot, int i) {
        const bool in = st < nreal;
        const int so = in ? 128 * st : 0;
        uint8_t *buf = lds + slot * C::STAGE;
        if (i < C::LW) {
            buf_dma16<STREAM ? 2 : 0>(buf_rsrc(wb, in ? wlen : 0u), wo[min(i, C::LW - 1)], so, buf + 1024 * (C::LW * wave + i));
        } else {
            const int j = max(0, min(i - C::LW, C::LX - 1));
            buf_dma16<0>(buf_rsrc(xb, in ? xlen : 0u), st < nreal - 1 ? xo[j] : xl[j], so,
                      buf + C::OFF_X + 1024 * (C::LX * wave + j));
        }
    };
    const u32x4 first = fetch_scales(0);
    u32x4 held = fetch_scales(1);
#pragma unroll
    for (int s = 0; s < NST; s++)
#pragma unroll
        for (int i = AHEAD ? C::LW : 0; i < C::VM; i++) issue(s, s, i);
    put_scales(0, first);

    struct Op { v4i w[WI], x[U]; };
    struct Sc { uint32_t w[WI], x[U]; };
    /* a wave's row groups are WT apart, so that a bucket's last few rows keep as
     * many waves busy as they can */
    auto read_w = [&](Op &o, const uint8_t *buf, int i, int s) {
        const int r = 32 * (WI * wr + i) + rr;
        o.w[i] = *(const v4i *)(buf + r * 128 + 16 * swz(r, 2 * s + g));
    };
    auto read_x = [&](Op &o, const uint8_t *buf, int u, int s) {
        const int r = 32 * (WT * u + wt) + rr;
        o.x[u] = *(const v4i *)(buf + C::OFF_X + r * 128 + 16 * swz(r, 2 * s + g));
    };
    const uint32_t pick = g ? 0x07050301u : 0x06040200u;
    f32x16 acc[WI][U];
#pragma unroll
    for (int i = 0; i < WI; i++)
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][u][e] = 0.0f;
    int slot = 0;
    /* AHEAD: the first stages' tokens come last, all but the last stage's are waited
     * for here, as the waits of the loop count whole stages */
    wait_vm<AHEAD ? C::LX : (NST - 1) * C::VM>();
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    /* the whole sum of a wave with UA row groups that hold rows */
    auto multiply = [&](auto ACTIVE) {
        constexpr int UA = decltype(ACTIVE)::value, N = WI * UA, R = WI + UA;
        /* the scales of stage st: byte s of a row's register is step s's */
        auto read_scales = [&](Sc &o, int st) {
            const uint8_t *p = table + (st / 2 & 1) * C::TABLE + 8 * (st & 1);
#pragma unroll
            for (int i = 0; i < WI; i++) {
                const u32x2 v = *(const u32x2 *)(p + 16 * (32 * (WI * wr + i) + rr));
                o.w[i] = __builtin_amdgcn_perm(v.y, v.x, pick);
            }
#pragma unroll
            for (int u = 0; u < UA; u++) {
                const u32x2 v = *(const u32x2 *)(p + 16 * (F + 32 * (WT * u + wt) + rr));
                o.x[u] = __builtin_amdgcn_perm(v.y, v.x, pick);
            }
        };
        /* the products of `cur` (step S), the reads of `nxt` (step s of the stage
         * in buf) and, with `load`, stage st's loads into slot `to`, spread among
         * them */
        auto step = [&](auto S, const Op &cur, const Sc &sc, Op &nxt, const uint8_t *buf, int s, bool load, int st, int to) {
            if constexpr (UA == 0) {
                if (load) {
#pragma unroll
                    for (int l = 0; l < C::VM; l++) issue(st, to, l);
                }
            }
#pragma unroll
            for (int q = 0; q < N; q++) {
                const int i = q % WI, u = q / WI;
                acc[i][u] = fp4_mfma32<decltype(S)::value>(cur.w[i], cur.x[u], acc[i][u], sc.w[i], sc.x[u]);
                if (N >= 8 && q == 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < R; j++)
                    if (j * N / (R + 1) == q) {
                        if (j < WI) read_w(nxt, buf, j, s);
                        else read_x(nxt, buf, j - WI, s);
                    }
                if (load) {
#pragma unroll
                    for (int l = 0; l < C::VM; l++)
                        if (l * N / C::VM == q) issue(st, to, l);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        /* stage st, the first or second of its pair. Nothing here branches: the
         * compiler would move products over the barrier into another block. */
        auto meet = [&](auto SECOND, int st) {
            if constexpr (decltype(SECOND)::value)
                put_scales(st / 2 + 1, held);
            __builtin_amdgcn_s_waitcnt(0xC07F);    /* this stage's operands are in registers */
            wait_vm<(NST - 2) * C::VM>();          /* the wave's loads of the next have landed */
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if constexpr (decltype(SECOND)::value) held = fetch_scales(st / 2 + 2);
        };
        if constexpr (C::DEEP) {
            /* the operands of a whole stage ahead */
            struct Ops { Op s[4]; } o0, o1;
            Sc c0, c1;
            auto read = [&](Ops &o, const uint8_t *buf, int k) {   /* the k-th of 4 R */
                if (k % R < WI) read_w(o.s[k / R], buf, k % R, k / R);
                else read_x(o.s[k / R], buf, k % R - WI, k / R);
            };
            auto stage = [&](auto SECOND, int st, const Ops &cur, const Sc &sc, Ops &nxt, Sc &sn) {
                meet(SECOND, st);
                const int free = slot;
                slot = slot + 1 == NST ? 0 : slot + 1;
                const uint8_t *buf = lds + slot * C::STAGE;
                if constexpr (UA == 0) {
#pragma unroll
                    for (int l = 0; l < C::VM; l++) issue(st + NST, free, l);
                } else {
                    read_scales(sn, st + 1);
#pragma unroll
                    for (int q = 0; q < 4 * N; q++) {
                        const int s = q / N, i = q % N % WI, u = q % N / WI;
                        acc[i][u] = s == 0   ? fp4_mfma32<0>(cur.s[s].w[i], cur.s[s].x[u], acc[i][u], sc.w[i], sc.x[u])
                                    : s == 1 ? fp4_mfma32<1>(cur.s[s].w[i], cur.s[s].x[u], acc[i][u], sc.w[i], sc.x[u])
                                    : s == 2 ? fp4_mfma32<2>(cur.s[s].w[i], cur.s[s].x[u], acc[i][u], sc.w[i], sc.x[u])
                                             : fp4_mfma32<3>(cur.s[s].w[i], cur.s[s].x[u], acc[i][u], sc.w[i], sc.x[u]);
#pragma unroll
                        for (int k = 0; k < 4 * R; k++)
                            if (k / (R / N + 1) == q || (q == 4 * N - 1 && k / (R / N + 1) > q)) read(nxt, buf, k);
#pragma unroll
                        for (int l = 0; l < C::VM; l++)
                            if (l * 4 * N / C::VM == q) issue(st + NST, free, l);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            };
            if constexpr (UA > 0) {
#pragma unroll
                for (int k = 0; k < 4 * R; k++) read(o0, lds, k);
                read_scales(c0, 0);
            }
            for (int st = 0; st < nst; st += 2) {
                stage(IC<0>{}, st, o0, c0, o1, c1);
                stage(IC<1>{}, st + 1, o1, c1, o0, c0);
            }
        } else {
            /* those of the next 64 values */
            Op o0, o1;
            Sc sc;
            if constexpr (UA > 0) {
#pragma unroll
                for (int i = 0; i < WI; i++) read_w(o0, lds, i, 0);
#pragma unroll
                for (int u = 0; u < UA; u++) read_x(o0, lds, u, 0);
                read_scales(sc, 0);
            }
            auto stage = [&](auto SECOND, int st) {
                const uint8_t *buf = lds + slot * C::STAGE;
                step(IC<0>{}, o0, sc, o1, buf, 1, false, 0, 0);
                step(IC<1>{}, o1, sc, o0, buf, 2, false, 0, 0);
                step(IC<2>{}, o0, sc, o1, buf, 3, false, 0, 0);
                meet(SECOND, st);
                const int free = slot;
                slot = slot + 1 == NST ? 0 : slot + 1;
                Sc sn;
                if constexpr (UA > 0) read_scales(sn, st + 1);
                step(IC<3>{}, o1, sc, o0, lds + slot * C::STAGE, 0, true, st + NST, free);
                sc = sn;
            };
            for (int st = 0; st < nst; st += 2) {
                stage(IC<0>{}, st);
                stage(IC<1>{}, st + 1);
            }
        }
    };
    if constexpr (GROUPED && U <= 2) {
        /* row groups of the wave that begin before the bucket's end */
        const int ua = (t.rows - 32 * wt + 32 * WT - 1) / (32 * WT);
        if (ua >= U) multiply(IC<U>{});
        else if (U == 2 && ua == 1) multiply(IC<U / 2>{});
        else multiply(IC<0>{});
    } else {
        multiply(IC<U>{});
    }
    /* the loads past the end, then the ring becomes the output tile */
    __builtin_amdgcn_s_waitcnt(0xC07F);
    wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    constexpr int EB = elem_bytes<OUT>(), LD = C::out_ld(EB), ROWS = C::out_rows(EB), PMAX = F * EB / 16;
    const int pieces = nf * EB / 16;
    const size_t ld = (size_t)a.N * EB;
    const bool whole = (((uintptr_t)a.C | ld) & 15u) == 0;   /* n0 and nf are whole pieces then too */
    typedef u32x4 piece __attribute__((aligned(2)));
#pragma unroll
    for (int m0 = 0; m0 < T; m0 += ROWS) {
#pragma unroll
        for (int u = m0 / (32 * WT); u < (m0 + ROWS) / (32 * WT); u++) {
            const int m = 32 * (WT * u + wt) + rr;
            const bool none = GROUPED && m < t.rows && fp4_source<GROUPED>(a, t, m) < 0;
            if (none && wr == 0 && g == 0) atomicOr(a.status, ST_BAD_EXPERT_ID);
#pragma unroll
            for (int i = 0; i < WI; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint8_t *o = lds + (m - m0) * LD + (32 * (WI * wr + i) + 8 * q + 4 * g) * EB;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = none ? __builtin_nanf("") : acc[i][u][4 * q + e];
                    if constexpr (OUT == DSV4_HIP_F32) {
                        *(f32x4 *)o = f32x4{v[0], v[1], v[2], v[3]};
                    } else {
                        u32x2 p;
                        p.x = fp4_pack<OUT>(v[0], v[1]);
                        p.y = fp4_pack<OUT>(v[2], v[3]);
                        *(u32x2 *)o = p;
                    }
                }
        }
        __syncthreads();
        uint8_t *out = (uint8_t *)a.C + ((size_t)(t.r0 + m0) * a.N + n0) * EB;
        const int rows = min(ROWS, t.rows - m0);
        for (int i = threadIdx.x; i < rows * PMAX; i += C::NT) {
            const int m = i / PMAX, p = i % PMAX;
            const uint8_t *src = lds + m * LD + 16 * p;
            uint8_t *dst = out + m * ld + 16 * p;
            if (p < pieces) {
                if (whole) __builtin_nontemporal_store(*(const u32x4 *)src, (DSV4_GLOBAL u32x4 *)dst);
                else *(DSV4_GLOBAL piece *)dst = *(const u32x4 *)src;
            } else {
                for (int b = 0; b < nf * EB - 16 * p; b += EB) {
                    if constexpr (EB == 4) *(DSV4_GLOBAL float *)(dst + b) = *(const float *)(src + b);
                    else *(DSV4_GLOBAL uint16_t *)(dst + b) = *(const uint16_t *)(src + b);
                }
            }
        }
        if (m0 + ROWS < T) __syncthreads();
    }
}

template <int F, int T, int WR, int WT, int NST, bool GROUPED, bool STREAM, int OUT>
__global__ __launch_bounds__((Fp4Tile<F, T, WR, WT, NST>::NT)) void k_fp4_tile(Fp4Args a)
{
    const int nt = (a.N + F - 1) / F;
    Fp4Bucket t;
    int n0;
    if constexpr (GROUPED) {
        int f = blockIdx.x % nt;
        if constexpr (F == 256) t = bucket_tile<T, uint8_t>(a, blockIdx.x, threadIdx.x & 63, fp4_matrix(a), nt, &f);
        else t = bucket_tile<T, uint8_t>(a, blockIdx.x / nt, threadIdx.x & 63, fp4_matrix(a));
        n0 = f * F;
        if (t.rows <= 0) return;
    } else {
        /* each XCD a contiguous run of tiles, eight row tiles by their feature
         * tiles at a time */
        const int mt = (a.M + T - 1) / T, total = mt * nt;
        const int per = total / 8, rest = total % 8, x = blockIdx.x % 8, y = blockIdx.x / 8;
        const int id = x * per + min(x, rest) + y;
        const int grp = id / (8 * nt), gm = min(8, mt - 8 * grp), in = id - grp * 8 * nt;
        t.w = a.W; t.s = a.Sw; t.e = 0; t.bad = false;
        t.r0 = (8 * grp + in % gm) * T;
        t.rows = min(T, a.M - t.r0);
        n0 = in / gm * F;
    }
    fp4_tile_sum<F, T, WR, WT, NST, GROUPED, STREAM, OUT>(a, t, n0);
}

/* Buckets of many rows: 256 features by the 256 rows of a bucket's whole tiles, a
 * last tile of up to 128 rows in the smaller form with its deeper ring: a weight is
 * read once for 256 rows (24,576 rows, Zipf, on 256 experts 2048 x 4096 319 us by 128
 * rows, 300 so). */
template <int OUT>
__global__ __launch_bounds__(512) void k_fp4_buckets(Fp4Args a)
{
    const int nt = (a.N + 255) / 256;
    int f = 0;
    const Fp4Bucket t = bucket_tile<256, uint8_t>(a, blockIdx.x, threadIdx.x & 63, fp4_matrix(a), nt, &f);
    if (t.rows <= 0) return;
    if (t.rows > 128) fp4_tile_sum<256, 256, 4, 2, 2, true, false, OUT>(a, t, 256 * f);
    else fp4_tile_sum<256, 128, 4, 2, 3, true, false, OUT>(a, t, 256 * f);
}

template <int F, int T, int WR, int WT, int NST, bool GROUPED, bool STREAM, int OUT>
static hipError_t fp4_tile(const Fp4Args &a, unsigned groups, hipStream_t st)
{
    using C = Fp4Tile<F, T, WR, WT, NST>;
    constexpr int lds = C::lds(elem_bytes<OUT>());
    static uint64_t done = 0;
    const hipError_t e = allow_lds((const void *)k_fp4_tile<F, T, WR, WT, NST, GROUPED, STREAM, OUT>, lds, done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_fp4_tile<F, T, WR, WT, NST, GROUPED, STREAM, OUT>), dim3(groups), dim3(C::NT), lds, st, a);
    return hipGetLastError();
}

template <int OUT>
static hipError_t fp4_buckets(const Fp4Args &a, unsigned groups, hipStream_t st)
{
    constexpr int small = Fp4Tile<256, 128, 4, 2, 3>::lds(elem_bytes<OUT>()), large = Fp4Tile<256, 256, 4, 2, 2>::lds(elem_bytes<OUT>());
    constexpr int lds = small > large ? small : large;
    static uint64_t done = 0;
    const hipError_t e = allow_lds((const void *)k_fp4_buckets<OUT>, lds, done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_fp4_buckets<OUT>, dim3(groups), dim3(512), lds, st, a);
    return hipGetLastError();
}

template <int OUT>
static hipError_t fp4_one(const Fp4Args &a, hipStream_t st)
{
    const Fp4Form form = fp4_form(a.M, a.N, a.K);
    const long waves = fp4_waves(form, a.M, a.N, 0);
    if (waves > FP4_MAX_WAVES) return hipErrorInvalidConfiguration;
    const unsigned groups = (unsigned)(waves / fp4_shape(form).waves);
    switch (form) {
    case FP4_SPLIT:
        hipLaunchKernelGGL(k_fp4_split<OUT>, dim3(groups), dim3(512), 0, st, a);
        return hipGetLastError();
    case FP4_TEAM:
        hipLaunchKernelGGL(k_fp4_team<OUT>, dim3(groups), dim3(256), 0, st, a);
        return hipGetLastError();
    case FP4_64x64: return fp4_tile<64, 64, 2, 2, 3, false, false, OUT>(a, groups, st);
    case FP4_128x64: return fp4_tile<128, 64, 2, 2, 3, false, false, OUT>(a, groups, st);
    case FP4_128x96: return fp4_tile<128, 96, 4, 1, 3, false, false, OUT>(a, groups, st);
    case FP4_128x128: return fp4_tile<128, 128, 2, 2, 2, false, false, OUT>(a, groups, st);
    case FP4_128x128_W8: return fp4_tile<128, 128, 4, 2, 3, false, false, OUT>(a, groups, st);
    case FP4_256x128: return fp4_tile<256, 128, 4, 2, 3, false, false, OUT>(a, groups, st);
    case FP4_256x192: return fp4_tile<256, 192, 4, 2, 2, false, false, OUT>(a, groups, st);
    default: return fp4_tile<256, 256, 4, 2, 2, false, false, OUT>(a, groups, st);
    }
}

template <bool STREAM, int OUT>
static hipError_t fp4_grouped(const Fp4Args &a, hipStream_t st)
{
    const Fp4Form form = fp4_grouped_form(a.M, a.N, a.K, a.n_experts);
    const long waves = fp4_waves(form, a.M, a.N, a.n_experts);
    if (waves > FP4_MAX_WAVES) return hipErrorInvalidConfiguration;
    const unsigned groups = (unsigned)(waves / fp4_shape(form).waves);
    switch (form) {
    case FP4_64x32: return fp4_tile<64, 32, 2, 1, 4, true, STREAM, OUT>(a, groups, st);
    case FP4_128x32: return fp4_tile<128, 32, 4, 1, 3, true, STREAM, OUT>(a, groups, st);
    case FP4_128x64: return fp4_tile<128, 64, 2, 2, 3, true, STREAM, OUT>(a, groups, st);
    case FP4_256x128: return fp4_tile<256, 128, 4, 2, 3, true, false, OUT>(a, groups, st);
    default: return fp4_buckets<OUT>(a, groups, st);
    }
}

template <int OUT>
static hipError_t fp4_launch(const Fp4Args &a, hipStream_t st)
{
    if (!a.table) return fp4_one<OUT>(a, st);
    return fp4_stream(a.M, a.N, a.K, a.n_experts) ? fp4_grouped<true, OUT>(a, st) : fp4_grouped<false, OUT>(a, st);
}

hipError_t gemm_fp4_launch(const Fp4Args &a, int out_type, hipStream_t st)
{
    if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.K % 32) return hipErrorInvalidValue;
    switch (out_type) {
    case DSV4_HIP_F32: return fp4_launch<DSV4_HIP_F32>(a, st);
    case DSV4_HIP_BF16: return fp4_launch<DSV4_HIP_BF16>(a, st);
    case DSV4_HIP_F16: return fp4_launch<DSV4_HIP_F16>(a, st);
    default: return hipErrorInvalidValue;
    }
}

} // namespace dsv4
