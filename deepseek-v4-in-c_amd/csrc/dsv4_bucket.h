/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_bucket.h - what the products of quantized rows share (int8, 4-bit):
 * range-checked loads to registers and to LDS, and the tile of an expert's
 * bucket that a workgroup takes. */
#ifndef DSV4_BUCKET_H
#define DSV4_BUCKET_H

#include "dsv4_internal.h"

namespace dsv4 {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr uint32_t BUF_OOB = 0x80000000u;           /* beyond every buffer: reads zeros */

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buf_rsrc(const void *p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)bytes, 0x00020000);
}
/* The whole offset goes into the per-lane part: the range check subtracts the
 * scalar part from the buffer's size, which wraps for a buffer shorter than
 * that (a single row). */
template <int CPOL>
__device__ __forceinline__ v4i buf_ld16(__amdgpu_buffer_rsrc_t r, uint32_t voff)
{
    return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, 0, CPOL));
}

/* what one workgroup multiplies: rows r0 .. r0 + rows of the product against
 * matrix w (scales s) */
template <class S>
struct Bucket {
    const uint8_t *w;
    const S *s;
    int r0, rows;
    int e;                                         /* its expert */
    bool bad;                                      /* the table's entry is not a matrix of the product */
};

/* Row tile `t` of the buckets ex_off[0 .. E], each cut into tiles of TR rows;
 * rows == 0 past the last one. Every wave finds it by itself: a lane counts the
 * tiles of E / 64 experts, a scan over the lanes finds the one that holds t, a
 * scan of its experts' tiles the expert. Offsets are clamped to [0, M], so no
 * table makes a row out of range. `matrix_ok` judges the table's entry.
 *
 * With nt, `t` is the workgroup of a launch over nt feature tiles, *f the one it
 * takes: workgroups go round the eight XCDs, and each XCD gets a contiguous
 * eighth of the (row, feature) tiles, an expert's in groups of eight row tiles by
 * its feature tiles. So an XCD's L2 fetches an expert's tokens once for all
 * features and a popular expert's weights once for eight row tiles. us in int8's
 * 256 x 128 tiles, against feature tiles dealt out to the XCDs: 24,576 rows of 256
 * experts 2048 x 4096 453 -> 429, with Zipf 520 -> 484, 6,144 rows of 64 of them
 * 116 -> 106; groups of all row tiles by one feature tile after the other 485 and
 * no groups 345 rather than 327 at 24,576 rows of 64 experts 4096 x 2048, Zipf. */
template <int TR, class S, class ARGS, class OK>
__device__ __forceinline__ Bucket<S> bucket_tile(const ARGS &a, int t, int lane, OK matrix_ok, int nt = 0,
                                                 int *f = nullptr)
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
    Bucket<S> o;
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
    o.s = (const S *)m.s;
    o.bad = !matrix_ok(m);
    return o;
}

typedef __attribute__((address_space(3))) void lds_mem;

/* CPOL 2: past the caches, for what is read once */
template <int CPOL = 0>
__device__ __forceinline__ void buf_dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, int soff, uint8_t *dst)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_mem *)dst, 16, (int)voff, soff, 0, CPOL);
}
template <int N>
__device__ __forceinline__ void wait_vm()
{
    __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

/* more than 64 KB of LDS has to be asked for, once on each device */
inline hipError_t allow_lds(const void *kernel, int bytes, uint64_t &done)
{
    int d = 0;
    hipError_t e = hipGetDevice(&d);
    if (e != hipSuccess || (d < 64 && (done >> d & 1))) return e;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && d < 64) done |= 1ull << d;
    return e;
}

} // namespace

} // namespace dsv4

#endif /* DSV4_BUCKET_H */
