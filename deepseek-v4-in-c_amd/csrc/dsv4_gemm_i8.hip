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
    int e;                                         /* its expert */
    bool bad;                                      /* the table's entry is not an int8 N x K matrix */
};

/* Row tile `t` of the buckets ex_off[0 .. E], each cut into tiles of TR rows;
 * rows == 0 past the last one. Every wave finds it by itself: a lane counts the
 * tiles of E / 64 experts, a scan over the lanes finds the one that holds t, a
 * scan of its experts' tiles the expert. Offsets are clamped to [0, M], so no
 * table makes a row out of range.
 *
 * With nt, `t` is the workgroup of a launch over nt feature tiles, *f the one it
 * takes: workgroups go round the eight XCDs, and each XCD gets a contiguous
 * eighth of the (row, feature) tiles, an expert's in groups of eight row tiles by
 * its feature tiles. So an XCD's L2 fetches an expert's tokens once for all
 * features and a popular expert's weights once for eight row tiles. us in 256 x
 * 128 tiles, against feature tiles dealt out to the XCDs: 24,576 rows of 256
 * experts 2048 x 4096 453 -> 429, with Zipf 520 -> 484, 6,144 rows of 64 of them
 * 116 -> 106; groups of all row tiles by one feature tile after the other 485 and
 * no groups 345 rather than 327 at 24,576 rows of 64 experts 4096 x 2048, Zipf. */
template <int TR>
__device__ __forceinline__ Tile bucket_tile(const I8Args &a, int t, int lane, int nt = 0, int *f = nullptr)
{
    const int E = a.n_experts, per = (E + 63) / 64;
    auto clampr = [&](int v) { return min(max(v, 0), a.M); };
    int mine = 0;
    const auto off = gptr(a.ex_off);
    int lo = clampr(off[min(lane * per, E)]);
    for (int i = 0; i < per; i += 4) {             /* four loads in flight */
        int hi[4];
#pragma unroll
        for (int j = 0; j < 4; j++) hi[j] = off[min(lane * per + min(i + j + 1, per), E)];
#pragma unroll
        for (int j = 0; j < 4; j++) {              /* past the lane's experts: empty buckets */
            hi[j] = clampr(hi[j]);
            mine += (max(hi[j] - lo, 0) + TR - 1) / TR;
            lo = hi[j];
        }
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    Tile o;
    o.w = nullptr; o.s = nullptr; o.r0 = 0; o.rows = 0; o.e = 0; o.bad = false;
    int in = 0;
    if (nt) {
        /* a sum that wraps comes from falling offsets: never more tiles than there are */
        const uint32_t tiles = min((uint32_t)__builtin_amdgcn_readlane(incl, 63), gridDim.x / (uint32_t)nt);
        const int total = (int)tiles * nt, x = t % 8, y = t / 8;
        if (t >= total) return o;
        const int id = x * (total / 8) + min(x, total % 8) + y;
        t = id / nt;
        in = id - t * nt;
    }
    const uint64_t past = __ballot(incl > t);
    if (!past) return o;
    const int L = __builtin_ctzll(past);
    int left = t - __builtin_amdgcn_readlane(incl - mine, L);
    /* its experts, one a lane */
    const int mylo = clampr(off[min(L * per + min(lane, per), E)]);
    const int n = max(__shfl_down(mylo, 1, 64) - mylo, 0), tiles = lane < per ? (n + TR - 1) / TR : 0;
    int upto = tiles;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {             /* per <= 16 */
        const int v = __shfl_up(upto, d, 64);
        if (lane >= d) upto += v;
    }
    const uint64_t holds = __ballot(lane < per && upto > left);
    if (!holds) return o;
    const int i = __builtin_ctzll(holds), mine_i = __builtin_amdgcn_readlane(tiles, i);
    left -= __builtin_amdgcn_readlane(upto, i) - mine_i;
    if (nt) {
        constexpr int GROUP = 8;
        in += left * nt;                           /* among the expert's tiles */
        const int g0 = in / (GROUP * nt) * GROUP, rows = min(GROUP, mine_i - g0);
        in -= g0 * nt;
        left = g0 + in % rows;
        *f = in / rows;
    }
    o.r0 = __builtin_amdgcn_readlane(mylo, i) + left * TR;
    o.rows = min(TR, __builtin_amdgcn_readlane(n, i) - left * TR);
    o.e = L * per + i;
    const DSV4QMat m = ld_uniform(a.table, o.e);
    o.w = (const uint8_t *)m.w;
    o.s = (const float *)m.s;
    o.bad = m.wdt != DSV4_WI8 || m.rows != a.N || m.cols != a.K || !m.w || !m.s || ((uintptr_t)m.w & 15u) ||
            ((uintptr_t)m.s & 3u);
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
 * Weights as whole 128-byte lines: an instruction takes 128 codes of 8 weight
 * rows, lane l (row l % 8) its 16 codes from 64 (l / 8 % 2) + 16 (l / 16).
 * Rows 0 - 7 of the MFMA's A operand are then the 8 weight rows at the block's
 * first 64 codes, rows 8 - 15 the same rows at its last 64; the B operand holds
 * 8 tokens the same way, and of the 16 x 16 result the two quadrants that
 * multiply equal codes count. A workgroup takes 8 RT weight rows by 8 TT
 * tokens, its waves share out K in blocks of 128, B of them in flight, and add
 * up in LDS. Bound: the weight stream, and below some 20 MB its latency: one
 * token of 4096 x 4096 5.2 us (3.2 TB/s), 247 experts of 2048 x 4096 with three
 * rows each 321 us (6.5 TB/s). Whole lines matter: 16 rows x 64 bytes an
 * instruction took 5.9 and 594 us. */
template <int RT, int TT, int NW, int B, bool GROUPED, int OUT>
__global__ __launch_bounds__(64 * NW) void k_i8_pair(I8Args a)
{
    constexpr int TR = 8 * TT, FR = 8 * RT;
    __shared__ int sum[NW][2][TT * RT][64];
    const int lane = threadIdx.x & 63, wave = wave_in_group();
    const int r8 = lane & 7, half = (lane >> 3) & 1, g = lane >> 4;
    const int slabs = (a.N + FR - 1) / FR, tile = blockIdx.x / slabs, n0 = (blockIdx.x - tile * slabs) * FR;
    Tile t;
    if constexpr (GROUPED) {
        t = bucket_tile<TR>(a, tile, lane);
        if (t.rows <= 0) return;
    } else {
        t.w = a.W; t.s = a.Sw; t.e = 0; t.bad = false;
        t.r0 = tile * TR;
        t.rows = min(TR, a.M - t.r0);
    }
    const int nf = min(FR, a.N - n0);
    if (GROUPED && t.bad) {
        if (threadIdx.x == 0) atomicOr(a.status, ST_BAD_DESCRIPTOR);
        for (int i = threadIdx.x; i < t.rows * nf; i += 64 * NW)
            i8_store<OUT>(a.C, (size_t)(t.r0 + i / nf) * a.N + n0 + i % nf, __builtin_nanf(""));
        return;
    }
    const uint32_t K = (uint32_t)a.K;
    const __amdgpu_buffer_rsrc_t rw = i8_rsrc(t.w + (size_t)n0 * K, (uint32_t)nf * K);
    const uint8_t *xb = GROUPED ? a.Aq : a.Aq + (size_t)t.r0 * K;
    const __amdgpu_buffer_rsrc_t rx = i8_rsrc(xb, GROUPED ? (uint32_t)a.n_a * K : (uint32_t)t.rows * K);
    auto src_of = [&](int i) -> int {
        if (i >= t.rows) return -1;
        if (!GROUPED) return i;
        const int s = a.row_tok ? a.row_tok[t.r0 + i] : t.r0 + i;
        return (unsigned)s < (unsigned)a.n_a ? s : -1;
    };
    const uint32_t kc = 64u * half + 16u * g;
    uint32_t xo[TT], wo[RT];
#pragma unroll
    for (int u = 0; u < TT; u++) {
        const int s = src_of(8 * u + r8);
        xo[u] = s < 0 ? I8_OOB : (uint32_t)s * K + kc;
    }
#pragma unroll
    for (int i = 0; i < RT; i++) wo[i] = (uint32_t)(8 * i + r8) * K + kc;
    const int nblk = (a.K + 127) / 128;
    v4i acc[RT][TT];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int u = 0; u < TT; u++) acc[i][u] = v4i{0, 0, 0, 0};
    for (int b0 = wave; b0 < nblk; b0 += NW * B) {
        v4i w[B][RT], x[B][TT];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const uint32_t c = (uint32_t)(b0 + NW * b) * 128u;
            const bool in = c + kc < K;
#pragma unroll
            for (int i = 0; i < RT; i++) w[b][i] = i8_ld16<2>(rw, in ? wo[i] + c : I8_OOB);
#pragma unroll
            for (int u = 0; u < TT; u++) x[b][u] = i8_ld16<0>(rx, in && xo[u] != I8_OOB ? xo[u] + c : I8_OOB);
        }
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int u = 0; u < TT; u++)
                    acc[i][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[b][i], x[b][u], acc[i][u], 0, 0, 0);
    }
    /* element e of lane l: weight row 4 (g % 2) + e at half g / 2, token l % 8
     * at half l / 8 % 2 */
    if (half == g >> 1) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int u = 0; u < TT; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum[wave][half][i * TT + u][r8 * 8 + 4 * (g & 1) + e] = acc[i][u][e];
    }
    __syncthreads();
    for (int o = threadIdx.x; o < TR * FR; o += 64 * NW) {
        const int n = o % FR, i = o / FR;
        if (i >= t.rows || n >= nf) continue;
        int v = 0;
#pragma unroll
        for (int w = 0; w < NW; w++)
#pragma unroll
            for (int h = 0; h < 2; h++) v += sum[w][h][(n / 8) * TT + i / 8][(i & 7) * 8 + (n & 7)];
        const int s = src_of(i);
        float f = __builtin_nanf("");
        if (s >= 0) f = (float)v * (GROUPED ? a.Sa[s] : a.Sa[t.r0 + s]) * t.s[n0 + n];
        else if (n == 0) atomicOr(a.status, ST_BAD_EXPERT_ID);
        i8_store<OUT>(a.C, (size_t)(t.r0 + i) * a.N + n0 + n, f);
    }
}

template <int RT, int TT, int NW, int B, bool GROUPED, int OUT>
static hipError_t i8_pair(const I8Args &a, hipStream_t st)
{
    const long groups = i8_waves(I8_PAIR, a.M, a.N, GROUPED ? a.n_experts : 0) / NW;
    hipLaunchKernelGGL((k_i8_pair<RT, TT, NW, B, GROUPED, OUT>), dim3((unsigned)groups), dim3(64 * NW), 0, st, a);
    return hipGetLastError();
}

/* bytes between rows of a tile of F features on its way out through LDS: 16
 * more than the row, so that the 16 rows of a store spread over the banks */
constexpr int i8_out_ld(int F, int eb) { return F * eb + 16; }

/* A workgroup's sums, acc[i][u] the wave's 16 features from f0 + 16 i by 16 rows
 * from m0 + 16 u, scaled, rounded, put together in LDS (free by now) and
 * written as 16-byte pieces: past the caches where C's rows consist of such; of
 * other rows from each row's first element, unaligned, the last few elements by
 * themselves (element by element throughout, us -> this: 299 rows 20543 x 224
 * bf16 14.3 -> 11.9, 2,787 rows 2691 x 128 fp32 12.3 -> 10.9; aligned 10.0 and
 * 10.7 at 20544 and 2688). */
template <int F, bool GROUPED, int OUT, int NTHREADS, int WI, int U, class SRC>
__device__ __forceinline__ void i8_leave(const I8Args &a, const Tile &t, int n0, int nf, uint8_t *lds,
                                         const v4i (&acc)[WI][U], int f0, int m0, SRC src_of)
{
    constexpr int EB = elem_bytes<OUT>(), LD = i8_out_ld(F, EB);
    const int lane = threadIdx.x & 63, rr = lane & 15, gq = lane >> 4;
    float sw[WI][4];
#pragma unroll
    for (int i = 0; i < WI; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int n = f0 + 16 * i + 4 * gq + e;
            sw[i][e] = n < nf ? gptr(t.s)[n0 + n] : 0.0f;
        }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int m = m0 + 16 * u + rr, s = src_of(m);
        const float sa = s >= 0 ? gptr(a.Sa)[GROUPED ? s : t.r0 + s] : __builtin_nanf("");
        if (GROUPED && s < 0 && m < t.rows && f0 == 0 && gq == 0) atomicOr(a.status, ST_BAD_EXPERT_ID);
#pragma unroll
        for (int i = 0; i < WI; i++) {
            uint8_t *o = lds + m * LD + (f0 + 16 * i + 4 * gq) * EB;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = (float)acc[i][u][e] * sa * sw[i][e];
            if constexpr (OUT == DSV4_HIP_F32) {
                *(f32x4 *)o = f32x4{v[0], v[1], v[2], v[3]};
            } else {
                uint2 p;
                p.x = narrow16<OUT>(v[0]) | (narrow16<OUT>(v[1]) << 16);
                p.y = narrow16<OUT>(v[2]) | (narrow16<OUT>(v[3]) << 16);
                *(uint2 *)o = p;
            }
        }
    }
    __syncthreads();
    uint8_t *out = (uint8_t *)a.C + ((size_t)t.r0 * a.N + n0) * EB;
    const size_t ld = (size_t)a.N * EB;
    const int pieces = nf * EB / 16;
    constexpr int PMAX = F * EB / 16;
    if ((((uintptr_t)a.C | ld) & 15u) == 0) {      /* n0 and nf are whole pieces then too */
        for (int i = threadIdx.x; i < t.rows * PMAX; i += NTHREADS) {
            const int m = i / PMAX, p = i % PMAX;
            if (p < pieces)
                __builtin_nontemporal_store(*(const u32x4 *)(lds + m * LD + 16 * p), (DSV4_GLOBAL u32x4 *)(out + m * ld + 16 * p));
        }
    } else {
        typedef u32x4 piece __attribute__((aligned(2)));
        for (int i = threadIdx.x; i < t.rows * PMAX; i += NTHREADS) {
            const int m = i / PMAX, p = i % PMAX;
            const uint8_t *src = lds + m * LD + 16 * p;
            uint8_t *dst = out + m * ld + 16 * p;
            if (p < pieces) {
                *(DSV4_GLOBAL piece *)dst = *(const u32x4 *)src;
            } else {
                for (int b = 0; b < nf * EB - 16 * p; b += EB) {
                    if constexpr (EB == 4) *(DSV4_GLOBAL float *)(dst + b) = *(const float *)(src + b);
                    else *(DSV4_GLOBAL uint16_t *)(dst + b) = *(const uint16_t *)(src + b);
                }
            }
        }
    }
}

/* ------------------------------------------------------ many rows -------
 * A workgroup takes F features by 16 T rows, wave (wr, wt) F / 4 features by
 * 16 T / WT rows. K goes in blocks of 128 codes, one staged row a 128-byte
 * line: both operands by loads straight to LDS into a ring of NST blocks (16-
 * byte pieces XOR-swizzled by row), a wave reading the operands of the next 64
 * codes while it multiplies these. One barrier a stage of KB blocks: after it
 * every wave's loads of the next stage have landed and no wave still reads this
 * one, so the stage NST ahead takes its place. Loads past K read nothing and
 * multiply as zeros. The tile leaves through LDS as whole 16-byte pieces of rows,
 * written past the caches (16 MB of bf16 36.7 -> 35.6 us of the call).
 * Bound: 256 x 128 tiles keep the MFMA units busy in 37 % of the cycles (2,048 x
 * 4096 x 4096 34 us, 2.0 POP/s, of 5 nominal and 4.3 that products of registers
 * alone reach; the library's int8 product takes 41.7), the rest are barriers and
 * LDS; its XCDs fetch 8.4 MB each, eight row tiles by four feature tiles' operands,
 * 67 MB for 25. Experts' buckets the HBM stream beside that (24,576 rows of 256
 * experts, Zipf, 483 us, even 430; 359 with every table entry the same matrix, 316
 * for the weights alone); few rows the chain of stages (16 to 128 rows of 4096 x
 * 4096 7 to 8 us; K split over teams of waves gained nothing, weights straight to
 * registers lost 10 to 20 %). */
template <int F, int T, int KB, int NST_> struct I8Tile {
    static constexpr int WT = T >= 4 ? 2 : 1, NWAVE = 4 * WT, U = T / WT, WI = F / 64;
    static constexpr int OFF_X = F * 128, SUB = OFF_X + 16 * T * 128, STAGE = KB * SUB;
    static constexpr int NST = NST_;
    static constexpr int LW = F / 8 / NWAVE, LX = 2 * T / NWAVE, VM = KB * (LW + LX);
    static constexpr int RING = NST * STAGE;
    static constexpr int OUTB(int eb) { return 16 * T * i8_out_ld(F, eb); }
    static constexpr int lds(int eb) { return RING > OUTB(eb) ? RING : OUTB(eb); }
    static_assert(LX * NWAVE == 2 * T && LW * NWAVE * 8 == F && (NST - 1) * VM < 64 && lds(4) <= 160 * 1024, "ring");
};

typedef __attribute__((address_space(3))) void i8_lds;

__device__ __forceinline__ void i8_dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, int soff, uint8_t *dst)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (i8_lds *)dst, 16, (int)voff, soff, 0, 0);
}
template <int N>
__device__ __forceinline__ void i8_wait_vm()
{
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

template <int F, int T, int KB, int NST, bool GROUPED, int OUT>
__global__ __launch_bounds__((64 * I8Tile<F, T, KB, NST>::NWAVE)) void k_i8_tile(I8Args a)
{
    using C = I8Tile<F, T, KB, NST>;
    constexpr int U = C::U, WI = C::WI, TR = 16 * T;
    /* buckets of many rows: an XCD's workgroups share an expert (bucket_tile).
     * Smaller tiles, dealt out / shared, us: 9,216 rows of 256 experts 2048 x 4096 in
     * 128 x 64 411 / 425, 3,582 of 256 4096 x 2048 in 64 x 32 397 / 408, 1,200 of 16
     * 1024 x 2048 in 128 x 64 11.4 / 11.7. */
    constexpr bool SHARED = GROUPED && F == 256;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = wave_in_group();
    const int rr = lane & 15, gq = lane >> 4, wr = wave & 3, wt = wave >> 2;
    const int nt = (a.N + F - 1) / F, nblk = (a.K + 127) / 128, nst = (nblk + KB - 1) / KB;
    Tile t;
    int n0;
    if constexpr (GROUPED) {
        int f = blockIdx.x % nt;
        if constexpr (SHARED) t = bucket_tile<TR>(a, blockIdx.x, lane, nt, &f);
        else t = bucket_tile<TR>(a, blockIdx.x / nt, lane);
        n0 = f * F;
        if (t.rows <= 0) return;
    } else {
        /* each XCD a contiguous run of tiles, eight row tiles by their feature
         * tiles at a time */
        const int mt = (a.M + TR - 1) / TR, total = mt * nt;
        const int per = total / 8, rest = total % 8, x = blockIdx.x % 8, y = blockIdx.x / 8;
        const int id = x * per + min(x, rest) + y;
        const int grp = id / (8 * nt), gm = min(8, mt - 8 * grp), in = id - grp * 8 * nt;
        t.w = a.W; t.s = a.Sw; t.e = 0; t.bad = false;
        t.r0 = (8 * grp + in % gm) * TR;
        t.rows = min(TR, a.M - t.r0);
        n0 = in / gm * F;
    }
    const int nf = min(F, a.N - n0);
    const uint32_t K = (uint32_t)a.K;
    const __amdgpu_buffer_rsrc_t rw = i8_rsrc(t.w + (size_t)n0 * K, (uint32_t)nf * K);
    const uint8_t *xb = GROUPED ? a.Aq : a.Aq + (size_t)t.r0 * K;
    const __amdgpu_buffer_rsrc_t rx = i8_rsrc(xb, GROUPED ? (uint32_t)a.n_a * K : (uint32_t)t.rows * K);
    auto src_of = [&](int i) -> int {              /* row of Aq from xb on; -1: none */
        if (i >= t.rows) return -1;
        if (!GROUPED) return i;
        const int s = a.row_tok ? a.row_tok[t.r0 + i] : t.r0 + i;
        return (unsigned)s < (unsigned)a.n_a ? s : -1;
    };
    auto swz = [](int r, int c) { return c ^ ((r >> 1) & 7); };
    uint32_t wo[C::LW], xo[C::LX], xl[C::LX];      /* xl: of the last block, pieces past K out of range */
#pragma unroll
    for (int i = 0; i < C::LW; i++) {
        const int r = 8 * (C::LW * wave + i) + lane / 8;
        wo[i] = (uint32_t)r * K + 16u * (uint32_t)swz(r, lane & 7);
    }
#pragma unroll
    for (int i = 0; i < C::LX; i++) {
        const int r = 8 * (C::LX * wave + i) + lane / 8, c = swz(r, lane & 7), s = src_of(r);
        xo[i] = s < 0 ? I8_OOB : (uint32_t)s * K + 16u * (uint32_t)c;
        xl[i] = (nblk - 1) * 128 + 16 * c < a.K ? xo[i] : I8_OOB;
    }
    if (GROUPED && t.bad) {
        if (threadIdx.x == 0) atomicOr(a.status, ST_BAD_DESCRIPTOR);
        for (int i = threadIdx.x; i < t.rows * nf; i += 64 * C::NWAVE)
            i8_store<OUT>(a.C, (size_t)(t.r0 + i / nf) * a.N + n0 + i % nf, __builtin_nanf(""));
        return;
    }
    /* The block this workgroup begins with. Rows of 4 KB put the lines of one
     * block into a few memory channels, and experts that run through K side by
     * side into the same ones; begun at different places they spread (sums are
     * exact in any order). Workgroups that share weights, or in SHARED an expert's
     * weights and tokens, keep step. us, 24,576 rows of 256 experts: all from block
     * 0 525, by expert and feature tile 445, by expert 430; 1,536 rows in
     * smaller tiles 462 and 374. One matrix gains nothing. */
    const int rot = SHARED ? (t.e * 8 + t.e / 4) % nblk : GROUPED ? (n0 / F * 4 + t.e) % nblk : 0;
    /* load i of a wave's share of stage st; past the end zeros, no traffic */
    auto issue = [&](int st, int slot, int i) {
        constexpr int LB = C::LW + C::LX;
        const int in = st * KB + i / LB, k = i % LB;
        const uint32_t oob = in < nblk ? 0u : I8_OOB;
        int blk = min(in, nblk - 1);
        if (GROUPED) blk = blk + rot < nblk ? blk + rot : blk + rot - nblk;
        const int so = blk * 128;
        uint8_t *buf = lds + slot * C::STAGE + i / LB * C::SUB;
        if (k < C::LW) i8_dma16(rw, wo[min(k, C::LW - 1)] | oob, so, buf + 1024 * (C::LW * wave + k));
        else {
            const int j = max(0, min(k - C::LW, C::LX - 1));
            i8_dma16(rx, (blk < nblk - 1 ? xo[j] : xl[j]) | oob, so, buf + C::OFF_X + 1024 * (C::LX * wave + j));
        }
    };
#pragma unroll
    for (int s = 0; s < C::NST; s++)
#pragma unroll
        for (int i = 0; i < C::VM; i++) issue(s, s, i);

    struct Op { v4i w[WI], x[U]; };
    auto read_w = [&](Op &o, const uint8_t *buf, int i, int h) {
        const int r = 16 * (WI * wr + i) + rr;
        o.w[i] = *(const v4i *)(buf + r * 128 + 16 * swz(r, gq + 4 * h));
    };
    auto read_x = [&](Op &o, const uint8_t *buf, int u, int h) {
        const int r = 16 * (U * wt + u) + rr;
        o.x[u] = *(const v4i *)(buf + C::OFF_X + r * 128 + 16 * swz(r, gq + 4 * h));
    };
    v4i acc[WI][U];
#pragma unroll
    for (int i = 0; i < WI; i++)
#pragma unroll
        for (int u = 0; u < U; u++) acc[i][u] = v4i{0, 0, 0, 0};
    int slot = 0;
    /* the products of `cur`, the reads of `nxt` (half h of the block in buf)
     * and, with LOAD, block st's loads into slot `to`, spread among them */
    auto half = [&](const Op &cur, Op &nxt, const uint8_t *buf, int h, bool load, int st, int to) {
#pragma unroll
        for (int q = 0; q < WI * U; q++) {
            constexpr int N = WI * U, R = WI + U;
            acc[q % WI][q / WI] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur.w[q % WI], cur.x[q / WI], acc[q % WI][q / WI], 0, 0, 0);
            /* the wait for `cur` is not one for the reads below; with few products
             * to wait behind, the reads had better go first */
            if (WI * U >= 8 && q == 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < R; j++)
                if (j * N / (R + 1) == q) {
                    if (j < WI) read_w(nxt, buf, j, h);
                    else read_x(nxt, buf, j - WI, h);
                }
            if (load) {
#pragma unroll
                for (int l = 0; l < C::VM; l++)
                    if (l * N / C::VM == q) issue(st, to, l);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    i8_wait_vm<(C::NST - 1) * C::VM>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Op o0, o1;
    int st = 0;
    /* waves whose rows are all behind the bucket's last only load (24,576 rows,
     * Zipf, 492 -> 483 us) */
    if (GROUPED && C::WT > 1 && 16 * U * wt >= t.rows) {
        for (; st < nst; st++) {
            i8_wait_vm<(C::NST - 2) * C::VM>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int l = 0; l < C::VM; l++) issue(st + C::NST, slot, l);
            slot = slot + 1 == C::NST ? 0 : slot + 1;
        }
    } else {
#pragma unroll
        for (int i = 0; i < WI; i++) read_w(o0, lds, i, 0);
#pragma unroll
        for (int u = 0; u < U; u++) read_x(o0, lds, u, 0);
    }
    for (; st < nst; st++) {
        const uint8_t *buf = lds + slot * C::STAGE;
#pragma unroll
        for (int j = 0; j + 2 < 2 * KB; j += 2) {
            half(o0, o1, buf + j / 2 * C::SUB, 1, false, 0, 0);
            half(o1, o0, buf + (j / 2 + 1) * C::SUB, 0, false, 0, 0);
        }
        half(o0, o1, buf + (KB - 1) * C::SUB, 1, false, 0, 0);
        __builtin_amdgcn_s_waitcnt(0xC07F);        /* this stage's operands are in registers */
        i8_wait_vm<(C::NST - 2) * C::VM>();        /* the wave's loads of the next have landed */
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int free = slot;
        slot = slot + 1 == C::NST ? 0 : slot + 1;
        half(o1, o0, lds + slot * C::STAGE, 0, true, st + C::NST, free);
    }
    /* the loads past the end, then the ring becomes the output tile */
    __builtin_amdgcn_s_waitcnt(0xC07F);
    i8_wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    i8_leave<F, GROUPED, OUT, 64 * C::NWAVE>(a, t, n0, nf, lds, acc, 16 * WI * wr, 16 * U * wt, src_of);
}

/* more than 64 KB of LDS has to be asked for, once on each device */
static hipError_t allow_lds(const void *kernel, int bytes, uint64_t &done)
{
    int d = 0;
    hipError_t e = hipGetDevice(&d);
    if (e != hipSuccess || (d < 64 && (done >> d & 1))) return e;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && d < 64) done |= 1ull << d;
    return e;
}

template <int F, int T, int KB, int NST, bool GROUPED, int OUT>
static hipError_t i8_tile(const I8Args &a, I8Form form, hipStream_t st)
{
    using C = I8Tile<F, T, KB, NST>;
    constexpr int lds = C::lds(elem_bytes<OUT>());
    static uint64_t done = 0;
    const hipError_t e = allow_lds((const void *)k_i8_tile<F, T, KB, NST, GROUPED, OUT>, lds, done);
    if (e != hipSuccess) return e;
    const long groups = i8_waves(form, a.M, a.N, GROUPED ? a.n_experts : 0) / C::NWAVE;
    hipLaunchKernelGGL((k_i8_tile<F, T, KB, NST, GROUPED, OUT>), dim3((unsigned)groups), dim3(64 * C::NWAVE), lds, st, a);
    return hipGetLastError();
}

template <bool GROUPED, int OUT>
static hipError_t i8_launch(const I8Args &a, hipStream_t st)
{
    const I8Form form = GROUPED ? i8_grouped_form(a.M, a.N, a.K, a.n_experts) : i8_form(a.M, a.N, a.K);
    if (i8_waves(form, a.M, a.N, GROUPED ? a.n_experts : 0) > I8_MAX_WAVES) return hipErrorInvalidConfiguration;
    if constexpr (GROUPED) {
        if (form == I8_PAIR) return i8_pair<4, 2, 4, 2, GROUPED, OUT>(a, st);
    } else {
        if (form == I8_PAIR) return i8_pair<1, 1, 8, 4, GROUPED, OUT>(a, st);
        if (form == I8_64x2_DEEP) return i8_tile<64, 2, 2, 3, GROUPED, OUT>(a, form, st);
        if (form == I8_64x4) return i8_tile<64, 4, 1, 3, GROUPED, OUT>(a, form, st);
        if (form == I8_128x8) return i8_tile<128, 8, 1, 4, GROUPED, OUT>(a, form, st);
    }
    switch (form) {
    case I8_64x2: return i8_tile<64, 2, 1, 4, GROUPED, OUT>(a, form, st);
    case I8_128x4: return i8_tile<128, 4, 1, 3, GROUPED, OUT>(a, form, st);
    default: return i8_tile<256, 8, 1, 3, GROUPED, OUT>(a, form, st);
    }
}

hipError_t gemm_i8_launch(const I8Args &a, int out_type, hipStream_t st)
{
    if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.K % 16) return hipErrorInvalidValue;
    const bool grouped = a.table != nullptr;
    switch (out_type) {
    case DSV4_HIP_F32: return grouped ? i8_launch<true, DSV4_HIP_F32>(a, st) : i8_launch<false, DSV4_HIP_F32>(a, st);
    case DSV4_HIP_BF16: return grouped ? i8_launch<true, DSV4_HIP_BF16>(a, st) : i8_launch<false, DSV4_HIP_BF16>(a, st);
    case DSV4_HIP_F16: return grouped ? i8_launch<true, DSV4_HIP_F16>(a, st) : i8_launch<false, DSV4_HIP_F16>(a, st);
    default: return hipErrorInvalidValue;
    }
}

} // namespace dsv4
