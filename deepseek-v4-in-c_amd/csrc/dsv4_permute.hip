/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_permute.hip - tokens to expert order and back, with gradients.
 *
 *   permute        stable counting sort of the (token, k) pairs by expert, and
 *                  rows[pos[t][k]] = x[t]
 *   permute_bwd    dx[t] = sum_k drows[pos[t][k]]
 *   unpermute      out[t] = sum_k w[t][k] * rows[pos[t][k]] (+ shared[t])
 *   unpermute_bwd  drows[pos[t][k]] = w[t][k] * dout[t]
 *                  dw[t][k] = sum_j dout[t][j] * rows[pos[t][k]][j]
 *
 * Sums run in fp32 in k order (dw: over a thread's elements, then over
 * threads in a fixed tree) and are rounded once to the element type, so the
 * same call gives the same bits. A pair without a row (pos outside [0, n *
 * topk)) adds nothing, receives nothing and has dw 0. All of them stream
 * memory and are bound by it; none uses a workspace.
 */
#include <initializer_list>

#include "dsv4_elem.h"
#include "dsv4_internal.h"

namespace dsv4 {

namespace {

constexpr int MAX_E = 1024, MAX_TOPK = 16;
constexpr size_t MAX_THREADS = 0xFFFFFF00u;        /* of one launch               */

/* Lanes of the wave that hold the same expert id; ids outside [0, E) share
 * one of their own. One ballot a bit of id + 1. */
__device__ __forceinline__ uint64_t lanes_of_id(int e, int E, int bits)
{
    const unsigned key = (unsigned)e < (unsigned)E ? (unsigned)e + 1u : 0u;
    uint64_t peers = ~0ull;
    for (int b = 0; b < bits; b++) {
        const bool bit = (key >> b) & 1u;
        const uint64_t m = __ballot(bit);
        peers &= bit ? m : ~m;
    }
    return peers;
}
__device__ __forceinline__ uint64_t lanes_below(int lane) { return lane ? ~0ull >> (64 - lane) : 0ull; }
__device__ __forceinline__ int id_bits(int E) { return 32 - __clz(E); }   /* of E, the largest key */

/* Exclusive scan of cnt[0 .. E) into off[0 .. E) by one wave, the total
 * returned to every lane: a lane sums E / 64 neighbours, a shuffle scan adds
 * the lanes below. */
__device__ __forceinline__ int scan_wave(int *off, const int *cnt, int E, int lane)
{
    const int per = (E + 63) / 64;
    int s = 0;
    for (int i = 0; i < per; i++) {
        const int e = lane * per + i;
        s += e < E ? cnt[e] : 0;
    }
    int incl = s;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    int run = incl - s;
    for (int i = 0; i < per; i++) {
        const int e = lane * per + i;
        if (e < E) {
            off[e] = run;
            run += cnt[e];
        }
    }
    return __shfl(incl, 63, 64);
}

/* pairs of each expert among [lo, hi) to cnt and, of those below `own`, to
 * bef: a wave takes 64 pairs, one LDS add an expert and wave. Returns whether
 * this thread met an id that is neither an expert nor -1. */
__device__ __forceinline__ bool count_pairs(int *cnt, int *bef, const int *idx, int lo, int hi, int own, int E)
{
    const int lane = threadIdx.x & 63, bits = id_bits(E);
    bool bad = false;
    for (int p0 = lo + (threadIdx.x & ~63); p0 < hi; p0 += blockDim.x) {
        const int p = p0 + lane;
        const int e = p < hi ? idx[p] : -1;
        bad |= e != -1 && (unsigned)e >= (unsigned)E;
        const uint64_t peers = lanes_of_id(e, E, bits);
        if ((unsigned)e < (unsigned)E && (peers & lanes_below(lane)) == 0) {
            atomicAdd(&cnt[e], __popcll(peers));
            if (bef && p0 < own) {
                const int n = __popcll(own - p0 >= 64 ? peers : peers & lanes_below(own - p0));
                if (n) atomicAdd(&bef[e], n);
            }
        }
    }
    return bad;
}

} // namespace

/* ---------------------------------------------------------------- sort --- */

/* Sort and copy in one launch: workgroup b owns `tpb` tokens (at most 128
 * pairs), counts every pair by itself (at most 32,768: 128 KB of ids from L2),
 * places its own and copies their rows. No workgroup waits for another. */
template <int TYPE, int V>
__global__ __launch_bounds__(512) void k_permute_one(PermuteArgs a, int tpb)
{
    __shared__ int cnt[MAX_E], bef[MAX_E], off[MAX_E];
    __shared__ int own_id[128], own_row[128];
    const int tid = threadIdx.x, lane = tid & 63, E = a.n_experts;
    const int npairs = a.n * a.topk;
    const int t0 = blockIdx.x * tpb, nt = min(tpb, a.n - t0);
    const int p0 = t0 * a.topk, np = nt * a.topk;  /* nt may be 0 in a call without tokens */
    for (int e = tid; e < E; e += 512) {
        cnt[e] = 0;
        bef[e] = 0;
    }
    if (tid < np) own_id[tid] = a.idx[p0 + tid];
    __syncthreads();
    const bool bad = count_pairs(cnt, bef, a.idx, 0, npairs, p0, E);
    if (bad && blockIdx.x == 0) atomicOr(a.status, ST_BAD_EXPERT_ID);
    __syncthreads();
    if (tid < 64) {
        const int total = scan_wave(off, cnt, E, lane);
        if (blockIdx.x == 0 && lane == 0) a.ex_off[E] = total;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = tid; e < E; e += 512) a.ex_off[e] = off[e];
    if (tid < np) {
        const int e = own_id[tid];
        int r = -1;
        if ((unsigned)e < (unsigned)E) {
            r = off[e] + bef[e];
            for (int i = 0; i < tid; i++) r += own_id[i] == e;
            a.row_tok[r] = t0 + tid / a.topk;
        }
        a.pos[p0 + tid] = r;
        own_row[tid] = r;
    }
    __syncthreads();
    constexpr int EB = elem_bytes<TYPE>();
    const int nv = a.hidden / V;
    const size_t rowb = (size_t)a.hidden * EB;
    for (int t = 0; t < nt; t++) {
        const uint8_t *src = (const uint8_t *)a.x + (size_t)(t0 + t) * rowb;
        for (int i = tid; i < nv; i += 512) {
            Elem<TYPE, V> v;
            v.load(src + (size_t)i * V * EB);
            for (int k = 0; k < a.topk; k++) {
                const int r = own_row[t * a.topk + k];
                if (r >= 0) v.store((uint8_t *)a.rows + (size_t)r * rowb + (size_t)i * V * EB);
            }
        }
    }
}

/* More pairs: counts, offsets, places and copies as four launches. Chunk c
 * holds pairs [1024 c, 1024 (c + 1)), the last one up to 2,047; its counts,
 * then the number of earlier pairs of each expert, wait in its own stretch of
 * pos (E <= 1024 words) until the launch that writes pos has read them. */
__device__ __forceinline__ int chunk_end(int c, int nch, int npairs) { return c + 1 == nch ? npairs : (c + 1) * 1024; }

__global__ __launch_bounds__(1024) void k_permute_count(PermuteArgs a, int nch)
{
    __shared__ int cnt[MAX_E];
    const int tid = threadIdx.x, c = blockIdx.x;
    cnt[tid] = 0;
    __syncthreads();
    const bool bad = count_pairs(cnt, nullptr, a.idx, c * 1024, chunk_end(c, nch, a.n * a.topk), 0, a.n_experts);
    if (bad) atomicOr(a.status, ST_BAD_EXPERT_ID);
    __syncthreads();
    if (tid < a.n_experts) a.pos[c * 1024 + tid] = cnt[tid];
}

__global__ __launch_bounds__(1024) void k_permute_scan(PermuteArgs a, int nch)
{
    __shared__ int cnt[MAX_E], off[MAX_E];
    const int tid = threadIdx.x, E = a.n_experts;
    int run = 0;
    if (tid < E)
        for (int c0 = 0; c0 < nch; c0 += 16) {     /* sixteen loads in flight */
            int v[16];
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = c0 + i < nch ? a.pos[(c0 + i) * 1024 + tid] : 0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (c0 + i < nch) a.pos[(c0 + i) * 1024 + tid] = run;
                run += v[i];
            }
        }
    cnt[tid] = run;
    __syncthreads();
    if (tid < 64) {
        const int total = scan_wave(off, cnt, E, tid);
        if (tid == 0) a.ex_off[E] = total;
    }
    __syncthreads();
    if (tid < E) a.ex_off[tid] = off[tid];
}

__global__ __launch_bounds__(1024) void k_permute_place(PermuteArgs a, int nch)
{
    __shared__ int cur[MAX_E];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, c = blockIdx.x, E = a.n_experts;
    const int hi = chunk_end(c, nch, a.n * a.topk), bits = id_bits(E);
    if (tid < E) cur[tid] = a.ex_off[tid] + a.pos[c * 1024 + tid];
    __syncthreads();
    for (int p0 = c * 1024; p0 < hi; p0 += 1024) {
        const int p = p0 + tid;
        const int e = p < hi ? a.idx[p] : -1;
        const uint64_t peers = lanes_of_id(e, E, bits);
        const int rank = __popcll(peers & lanes_below(lane));
        const bool ok = (unsigned)e < (unsigned)E;
        int r = -1;
        for (int w = 0; w < 16; w++) {             /* waves in order: rows of a bucket in pair order */
            if (w == wv && ok) r = cur[e] + rank;
            __syncthreads();
            if (w == wv && ok && rank == 0) cur[e] += __popcll(peers);
            __syncthreads();
        }
        if (p < hi) {
            a.pos[p] = r;
            if (ok) a.row_tok[r] = p / a.topk;
        }
    }
}

/* a thread copies one vector of a token to its topk rows */
template <int TYPE, int V>
__global__ __launch_bounds__(256) void k_permute_copy(PermuteArgs a)
{
    constexpr int EB = elem_bytes<TYPE>();
    const int nv = a.hidden / V;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)a.n * nv) return;
    const int t = (int)(i / nv), j = (int)(i - (size_t)t * nv);
    const size_t rowb = (size_t)a.hidden * EB, o = (size_t)j * V * EB;
    Elem<TYPE, V> v;
    v.load((const uint8_t *)a.x + t * rowb + o);
    for (int k = 0; k < a.topk; k++) {
        const int r = a.pos[(size_t)t * a.topk + k];
        if (r >= 0) v.store((uint8_t *)a.rows + r * rowb + o);
    }
}

/* ------------------------------------------------------------ way back --- */

/* A thread sums one vector over the token's topk rows, every row's load
 * issued before the first is used. W: weights (else 1). */
template <int TYPE, int V, int KMAX, bool W>
__global__ __launch_bounds__(256) void k_unpermute(UnpermuteArgs a)
{
    constexpr int EB = elem_bytes<TYPE>();
    const int nv = a.hidden / V;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)a.n * nv) return;
    const int t = (int)(i / nv), j = (int)(i - (size_t)t * nv);
    const size_t rowb = (size_t)a.hidden * EB, o = (size_t)j * V * EB;
    const int nrows = a.n * a.topk;
    int p[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; k++) p[k] = k < a.topk ? a.pos[(size_t)t * a.topk + k] : -1;
    Elem<TYPE, V> v[KMAX], s;
#pragma unroll
    for (int k = 0; k < KMAX; k++)
        if ((unsigned)p[k] < (unsigned)nrows) v[k].load((const uint8_t *)a.rows + p[k] * rowb + o);
    if (a.shared) s.load((const uint8_t *)a.shared + t * rowb + o);
    float acc[V], f[V];
#pragma unroll
    for (int q = 0; q < V; q++) acc[q] = 0.0f;
#pragma unroll
    for (int k = 0; k < KMAX; k++)
        if ((unsigned)p[k] < (unsigned)nrows) {
            const float w = W ? a.w[(size_t)t * a.topk + k] : 1.0f;
            v[k].get(f);
#pragma unroll
            for (int q = 0; q < V; q++) acc[q] = W ? fmaf(w, f[q], acc[q]) : acc[q] + f[q];
        }
    if (a.shared) {
        s.get(f);
#pragma unroll
        for (int q = 0; q < V; q++) acc[q] += f[q];
    }
    s.set(acc);
    s.store((uint8_t *)a.out + t * rowb + o);
}

/* A workgroup takes a token: dout once, its rows once, drows written and the
 * topk dot products kept in registers until the end. */
template <int TYPE, int V, int KMAX>
__global__ __launch_bounds__(256) void k_unpermute_bwd(UnpermuteBwdArgs a)
{
    constexpr int EB = elem_bytes<TYPE>();
    __shared__ float part[4][KMAX];
    const int tid = threadIdx.x, t = blockIdx.x, nv = a.hidden / V;
    const size_t rowb = (size_t)a.hidden * EB;
    const int nrows = a.n * a.topk;
    int p[KMAX];
    float w[KMAX], dot[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; k++) {
        p[k] = k < a.topk ? a.pos[(size_t)t * a.topk + k] : -1;
        if ((unsigned)p[k] >= (unsigned)nrows) p[k] = -1;
        w[k] = p[k] >= 0 ? a.w[(size_t)t * a.topk + k] : 0.0f;
        dot[k] = 0.0f;
    }
    for (int i = tid; i < nv; i += 256) {
        const size_t o = (size_t)i * V * EB;
        Elem<TYPE, V> d, y[KMAX];
        d.load((const uint8_t *)a.dout + t * rowb + o);
#pragma unroll
        for (int k = 0; k < KMAX; k++)
            if (p[k] >= 0) y[k].load((const uint8_t *)a.rows + p[k] * rowb + o);
        float fd[V], f[V];
        d.get(fd);
#pragma unroll
        for (int k = 0; k < KMAX; k++)
            if (p[k] >= 0) {
                y[k].get(f);
#pragma unroll
                for (int q = 0; q < V; q++) dot[k] = fmaf(fd[q], f[q], dot[k]);
#pragma unroll
                for (int q = 0; q < V; q++) f[q] = w[k] * fd[q];
                y[k].set(f);
                y[k].store((uint8_t *)a.drows + p[k] * rowb + o);
            }
    }
#pragma unroll
    for (int k = 0; k < KMAX; k++) {
        const float v = wave_sum(dot[k]);
        if ((tid & 63) == 0) part[tid >> 6][k] = v;
    }
    __syncthreads();
    if (tid < a.topk) a.dw[(size_t)t * a.topk + tid] = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
}

/* ----------------------------------------------------------- launchers --- */

namespace {

template <int TYPE, int V>
hipError_t permute_t(const PermuteArgs &a, hipStream_t st)
{
    const long pairs = (long)a.n * a.topk;
    if (pairs <= PERMUTE_ONE_MAX) {
        int tpb = 8;                               /* 128 pairs at the largest topk */
        const int blocks = a.n > 0 ? (a.n + tpb - 1) / tpb : 1;
        hipLaunchKernelGGL((k_permute_one<TYPE, V>), dim3(blocks), dim3(512), 0, st, a, tpb);
        return hipGetLastError();
    }
    const int nch = (int)(pairs / 1024);
    const size_t vecs = (size_t)a.n * (a.hidden / V);
    if (vecs > MAX_THREADS) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(k_permute_count, dim3(nch), dim3(1024), 0, st, a, nch);
    hipLaunchKernelGGL(k_permute_scan, dim3(1), dim3(1024), 0, st, a, nch);
    hipLaunchKernelGGL(k_permute_place, dim3(nch), dim3(1024), 0, st, a, nch);
    hipLaunchKernelGGL((k_permute_copy<TYPE, V>), dim3((unsigned)((vecs + 255) / 256)), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int TYPE, int V, bool W>
hipError_t unpermute_t(const UnpermuteArgs &a, hipStream_t st)
{
    const size_t vecs = (size_t)a.n * (a.hidden / V);
    if (vecs > MAX_THREADS) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)((vecs + 255) / 256)), block(256);
    if (a.topk <= 8) hipLaunchKernelGGL((k_unpermute<TYPE, V, 8, W>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_unpermute<TYPE, V, MAX_TOPK, W>), grid, block, 0, st, a);
    return hipGetLastError();
}

template <int TYPE, int V>
hipError_t unpermute_bwd_t(const UnpermuteBwdArgs &a, hipStream_t st)
{
    if ((size_t)a.n * 256 > MAX_THREADS) return hipErrorInvalidConfiguration;
    if (a.topk <= 8) hipLaunchKernelGGL((k_unpermute_bwd<TYPE, V, 8>), dim3(a.n), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_unpermute_bwd<TYPE, V, MAX_TOPK>), dim3(a.n), dim3(256), 0, st, a);
    return hipGetLastError();
}

/* rows of whole vectors at 16-byte addresses; single elements otherwise */
bool whole_vectors(int type, int hidden, std::initializer_list<const void *> ps)
{
    if ((size_t)hidden * elem_bytes_of(type) % 16) return false;
    for (const void *p : ps)
        if ((uintptr_t)p & 15u) return false;
    return true;
}

} // namespace

#define BY_TYPE(type, vec, CALL)                                                              \
    switch (type) {                                                                           \
    case DSV4_HIP_F32: return (vec) ? CALL(DSV4_HIP_F32, 4) : CALL(DSV4_HIP_F32, 1);          \
    case DSV4_HIP_BF16: return (vec) ? CALL(DSV4_HIP_BF16, 8) : CALL(DSV4_HIP_BF16, 1);       \
    case DSV4_HIP_F16: return (vec) ? CALL(DSV4_HIP_F16, 8) : CALL(DSV4_HIP_F16, 1);          \
    default: return hipErrorInvalidValue;                                                     \
    }

hipError_t permute_launch(const PermuteArgs &a, int type, hipStream_t st)
{
    if (a.n_experts < 1 || a.n_experts > MAX_E || a.topk < 1 || a.topk > MAX_TOPK) return hipErrorInvalidValue;
    const bool vec = whole_vectors(type, a.hidden, {a.x, a.rows});
#define CALL(T, V) permute_t<T, V>(a, st)
    BY_TYPE(type, vec, CALL)
#undef CALL
}

hipError_t unpermute_launch(const UnpermuteArgs &a, int type, hipStream_t st)
{
    if (a.topk < 1 || a.topk > MAX_TOPK || a.n < 1) return hipErrorInvalidValue;
    const bool vec = whole_vectors(type, a.hidden, {a.rows, a.out, a.shared});
#define CALL(T, V) (a.w ? unpermute_t<T, V, true>(a, st) : unpermute_t<T, V, false>(a, st))
    BY_TYPE(type, vec, CALL)
#undef CALL
}

hipError_t unpermute_bwd_launch(const UnpermuteBwdArgs &a, int type, hipStream_t st)
{
    if (a.topk < 1 || a.topk > MAX_TOPK || a.n < 1) return hipErrorInvalidValue;
    const bool vec = whole_vectors(type, a.hidden, {a.dout, a.rows, a.drows});
#define CALL(T, V) unpermute_bwd_t<T, V>(a, st)
    BY_TYPE(type, vec, CALL)
#undef CALL
}

} // namespace dsv4
