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
 * topk)) adds nothing, receives nothing and has dw 0. None uses a workspace.
 *
 * Bound: memory. us at 4,096 tokens of 4,096 bf16, six rows each (235 MB, 46 at
 * the rate of a plain copy): sort and copy 48.5, the gradient 43; 2,803 tokens of
 * which half the pairs are here: way back 18.2 (5.1 TB/s), both gradients 29.9
 * (5.4 TB/s). 64 tokens 5.2, the sort's chain of loads, counts and barriers. */
#include <algorithm>
#include <initializer_list>

#include "dsv4_elem.h"
#include "dsv4_internal.h"

namespace dsv4 {

namespace {

constexpr int MAX_E = 1024, MAX_TOPK = 16;
constexpr long MAX_WAVES = (1L << 26) - 4;         /* of one launch: 2^32 threads */

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

/* Pairs of each expert among [lo, hi) to cnt: a wave takes 64 pairs, one LDS
 * add an expert and wave. Returns whether this thread met an id that is neither
 * an expert nor -1. */
__device__ __forceinline__ bool count_pairs(int *cnt, const int *idx, int lo, int hi, int E)
{
    const int lane = threadIdx.x & 63, bits = id_bits(E);
    bool bad = false;
    for (int p0 = lo + (threadIdx.x & ~63); p0 < hi; p0 += blockDim.x) {
        const int p = p0 + lane;
        const int e = p < hi ? idx[p] : -1;
        bad |= e != -1 && (unsigned)e >= (unsigned)E;
        const uint64_t peers = lanes_of_id(e, E, bits);
        if ((unsigned)e < (unsigned)E && (peers & lanes_below(lane)) == 0) atomicAdd(&cnt[e], __popcll(peers));
    }
    return bad;
}

} // namespace

/* ---------------------------------------------------------------- sort --- */

/* Sort and copy in one launch: workgroup b owns `tpb` tokens (at most 256
 * pairs), counts every pair by itself (at most 32,768: 128 KB of ids from L2),
 * places its own and copies their rows. No workgroup waits for another. Its
 * tokens' first PF vectors a thread are in flight while it counts. A counter
 * word holds the expert's pairs in the low half and those before the
 * workgroup's own in the high half. Lanes that share the first lane's id add
 * once for all of them, so an expert that takes most pairs does not serialise
 * the adds. Eight ids a thread are asked for together. */
template <int TYPE, int V>
__global__ __launch_bounds__(1024) void k_permute_one(PermuteArgs a, int tpb)
{
    constexpr int NT = 1024, PF = 8, IDS = 8, EB = elem_bytes<TYPE>();
    static_assert(PERMUTE_ONE_MAX < 65536, "two counts in a word");
    static_assert(PERMUTE_ONE_MAX / 256 + MAX_TOPK <= 256, "own pairs");
    __shared__ uint32_t cnt[MAX_E];
    __shared__ int off[MAX_E];
    __shared__ int own_row[256];
    const int tid = threadIdx.x, lane = tid & 63, E = a.n_experts;
    const int npairs = a.n * a.topk;
    const int t0 = blockIdx.x * tpb, nt = min(tpb, a.n - t0);
    const int p0 = t0 * a.topk, np = nt * a.topk;  /* nt is 0 in a call without tokens */
    const int nv = a.hidden / V;
    const size_t rowb = (size_t)a.hidden * EB;
    const long items = (long)nt * nv;              /* vectors of the workgroup's tokens, one after another */
    const uint8_t *src = (const uint8_t *)a.x + (size_t)t0 * rowb;
    Elem<TYPE, V> v[PF];
    auto fetch = [&](long base) {
#pragma unroll
        for (int j = 0; j < PF; j++) {
            const long it = base + j * NT + tid;
            if (it < items) v[j].load(src + (size_t)it * V * EB);
        }
    };
    if (tid < E) cnt[tid] = 0;
    fetch(0);
    __syncthreads();
    bool bad = false;
    for (int b0 = 0; b0 < npairs; b0 += IDS * NT) {
        int id[IDS];
#pragma unroll
        for (int i = 0; i < IDS; i++) {
            const int q = b0 + i * NT + tid;
            id[i] = q < npairs ? a.idx[q] : -1;
        }
#pragma unroll
        for (int i = 0; i < IDS; i++) {
            const int q0 = b0 + i * NT + (tid & ~63), e = id[i];
            if (q0 >= npairs) break;               /* the wave's */
            const bool ok = (unsigned)e < (unsigned)E;
            bad |= !ok && e != -1;
            const int e0 = __builtin_amdgcn_readfirstlane(e);
            const uint64_t same = __ballot(e == e0);
            if (e != e0) {
                if (ok) atomicAdd(&cnt[e], q0 + lane < p0 ? 0x10001u : 1u);
            } else if (ok && lane == 0) {
                const int before = min(max(p0 - q0, 0), 64);
                const uint64_t m = before == 64 ? same : same & lanes_below(before);
                atomicAdd(&cnt[e], (uint32_t)__popcll(same) + ((uint32_t)__popcll(m) << 16));
            }
        }
    }
    if (bad && blockIdx.x == 0) atomicOr(a.status, ST_BAD_EXPERT_ID);
    __syncthreads();
    if (tid < 64) {                                /* first rows: exclusive scan of the counts */
        const int per = (E + 63) / 64;
        int sum = 0;
        for (int i = 0; i < per; i++) {
            const int e = lane * per + i;
            sum += e < E ? (int)(cnt[e] & 0xFFFFu) : 0;
        }
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(incl, d, 64);
            if (lane >= d) incl += u;
        }
        int run = incl - sum;
        for (int i = 0; i < per; i++) {
            const int e = lane * per + i;
            if (e < E) {
                off[e] = run;
                run += (int)(cnt[e] & 0xFFFFu);
            }
        }
        if (blockIdx.x == 0 && lane == 63) a.ex_off[E] = incl;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid < E) a.ex_off[tid] = off[tid];
    /* own pairs, a wave of them after the other: the high halves run on */
    const int bits = id_bits(E);
    for (int w = 0; w < (np + 63) / 64; w++) {
        if ((tid >> 6) == w) {
            const int e = tid < np ? a.idx[p0 + tid] : -1;
            const bool ok = (unsigned)e < (unsigned)E;
            const uint64_t peers = lanes_of_id(e, E, bits);
            const int rank = __popcll(peers & lanes_below(lane));
            int r = -1;
            if (ok) {
                r = off[e] + (int)(cnt[e] >> 16) + rank;
                a.row_tok[r] = t0 + tid / a.topk;
            }
            if (ok && rank == 0) cnt[e] += (uint32_t)__popcll(peers) << 16;
            if (tid < np) {
                a.pos[p0 + tid] = r;
                own_row[tid] = r;
            }
        }
        __syncthreads();
    }
    for (long base = 0; base < items; base += PF * NT) {
        if (base) fetch(base);
#pragma unroll
        for (int j = 0; j < PF; j++) {
            const long it = base + j * NT + tid;
            if (it >= items) break;
            const int t = (int)((uint32_t)it / (uint32_t)nv), i = (int)it - t * nv;
            uint8_t *dst = (uint8_t *)a.rows + (size_t)i * V * EB;
            for (int k = 0; k < a.topk; k++) {
                const int r = own_row[t * a.topk + k];
                if (r >= 0) v[j].store(dst + (size_t)r * rowb);
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
    const bool bad = count_pairs(cnt, a.idx, c * 1024, chunk_end(c, nch, a.n * a.topk), a.n_experts);
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

/* Wave w of a launch takes 128 vectors of a token, so that the token's rows
 * and weights are scalar loads and the branches on them uniform. */
constexpr int WAVE_VECS = 128;
struct WaveItem {
    int t, j;                                      /* token, the lane's first vector (the second is 64 on) */
};
__device__ __forceinline__ WaveItem wave_item(int nv)
{
    const int cpt = (nv + WAVE_VECS - 1) / WAVE_VECS, w = wave_id();
    const int t = __builtin_amdgcn_readfirstlane((int)((uint32_t)w / (uint32_t)cpt));
    return WaveItem{t, (w - t * cpt) * WAVE_VECS + (int)(threadIdx.x & 63)};
}

/* a token's vectors to its topk rows */
template <int TYPE, int V>
__global__ __launch_bounds__(256) void k_permute_copy(PermuteArgs a)
{
    constexpr int EB = elem_bytes<TYPE>();
    const int nv = a.hidden / V;
    const WaveItem it = wave_item(nv);
    if (it.t >= a.n) return;
    const size_t rowb = (size_t)a.hidden * EB;
    Elem<TYPE, V> v[2];
#pragma unroll
    for (int h = 0; h < 2; h++)
        if (it.j + 64 * h < nv) v[h].load((const uint8_t *)a.x + it.t * rowb + (size_t)(it.j + 64 * h) * V * EB);
    for (int k = 0; k < a.topk; k++) {
        const int r = ld_uniform(a.pos, it.t * a.topk + k);
        if (r < 0) continue;
#pragma unroll
        for (int h = 0; h < 2; h++)
            if (it.j + 64 * h < nv) v[h].store((uint8_t *)a.rows + r * rowb + (size_t)(it.j + 64 * h) * V * EB);
    }
}

/* ------------------------------------------------------------ way back --- */

/* A lane sums two vectors over the token's topk rows, every row's load issued
 * before the first is used. W: weights (else 1). */
template <int TYPE, int V, int KMAX, bool W, bool ONCE>
__global__ __launch_bounds__(256) void k_unpermute(UnpermuteArgs a)
{
    constexpr int EB = elem_bytes<TYPE>();
    const int nv = a.hidden / V;
    const WaveItem it = wave_item(nv);
    if (it.t >= a.n) return;
    const size_t rowb = (size_t)a.hidden * EB;
    const int nrows = a.n * a.topk;
    int p[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; k++) p[k] = k < a.topk ? ld_uniform(a.pos, it.t * a.topk + k) : -1;
    const bool two = it.j + 64 < nv;
    if (it.j >= nv) return;
    const size_t o0 = (size_t)it.j * V * EB, o1 = two ? o0 + (size_t)64 * V * EB : o0;
    Elem<TYPE, V> v[KMAX][2], s[2];
#pragma unroll
    for (int k = 0; k < KMAX; k++)
        if ((unsigned)p[k] < (unsigned)nrows) {
            v[k][0].template load<ONCE>((const uint8_t *)a.rows + p[k] * rowb + o0);
            v[k][1].template load<ONCE>((const uint8_t *)a.rows + p[k] * rowb + o1);
        }
    if (a.shared) {
        s[0].load((const uint8_t *)a.shared + it.t * rowb + o0);
        s[1].load((const uint8_t *)a.shared + it.t * rowb + o1);
    }
    float acc[2][V], f[V];
#pragma unroll
    for (int q = 0; q < V; q++) acc[0][q] = acc[1][q] = 0.0f;
#pragma unroll
    for (int k = 0; k < KMAX; k++)
        if ((unsigned)p[k] < (unsigned)nrows) {
            const float w = W ? ld_uniform(a.w, it.t * a.topk + k) : 1.0f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                v[k][h].get(f);
#pragma unroll
                for (int q = 0; q < V; q++) acc[h][q] = W ? fmaf(w, f[q], acc[h][q]) : acc[h][q] + f[q];
            }
        }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (a.shared) {
            s[h].get(f);
#pragma unroll
            for (int q = 0; q < V; q++) acc[h][q] += f[q];
        }
        if (h == 0 || two) {
            s[h].set(acc[h]);
            s[h].store((uint8_t *)a.out + it.t * rowb + (h ? o1 : o0));
        }
    }
}

/* A workgroup takes a token: dout once, its rows once, drows written and the
 * topk dot products kept in registers until the end. */
template <int TYPE, int V, int KMAX, bool ONCE, int NT>
__global__ __launch_bounds__(NT) void k_unpermute_bwd(UnpermuteBwdArgs a)
{
    constexpr int EB = elem_bytes<TYPE>();
    __shared__ float part[NT / 64][KMAX];
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
    for (int i = tid; i < nv; i += NT) {
        const size_t o = (size_t)i * V * EB;
        Elem<TYPE, V> d, y[KMAX];
        d.template load<ONCE>((const uint8_t *)a.dout + t * rowb + o);
#pragma unroll
        for (int k = 0; k < KMAX; k++)
            if (p[k] >= 0) y[k].template load<ONCE>((const uint8_t *)a.rows + p[k] * rowb + o);
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
    if (tid < a.topk) {
        float v = part[0][tid];
#pragma unroll
        for (int w = 1; w < NT / 64; w++) v += part[w][tid];
        a.dw[(size_t)t * a.topk + tid] = v;
    }
}

/* ----------------------------------------------------------- launchers --- */

namespace {

/* Rows beyond what the caches keep are read past them: 24,576 rows of 8 KB 66
 * -> 43 us, and their gradients' 16,818 of which half are there 29 -> 30 after a
 * forward pass that left 18 rather than 24. A batch's rows, just written by the
 * products, are better found there (384 rows of 16 KB 3.9 -> 3.3). */
template <int TYPE>
bool reads_once(long n, long topk, long hidden) { return n * topk * hidden * elem_bytes<TYPE>() > 64L << 20; }

long wave_items(long n, long nv) { return n * ((nv + WAVE_VECS - 1) / WAVE_VECS); }

template <int TYPE, int V>
hipError_t permute_t(const PermuteArgs &a, hipStream_t st)
{
    const long pairs = (long)a.n * a.topk;
    /* One launch with a workgroup a CU, since each counts every pair (us, at most
     * 16 tokens a workgroup / this / four launches: 32,000 x 1 of 128 bf16 69.4 /
     * 16.0 / 19.4, 16,000 x 2 of 256 39.7 / 17.5 / 19.5, 8,000 x 2 of 1024 18.0 /
     * 15.4 / 20.6). Four launches for more pairs (39,456 of 1024 36.2 in one, 28.5
     * in four) and where the copy of long rows outweighs the launches (32,000 x 1
     * of 2048 86.7 / 59.3 / 51.8, 16,000 x 2 of 4096 93.9 / 97.0 / 90.7; 4,096 x 6
     * of 4096 45.0 / 45.0 / 46.4, 8,000 x 1 of 2048 15.6 / 14.7 / 23.5). */
    const int tpb = a.n ? (int)(((long)a.n + 255) / 256) : 1;
    const bool long_copy = tpb > 16 && (long)a.n * a.hidden * elem_bytes<TYPE>() > 64L << 20;
    if (pairs <= PERMUTE_ONE_MAX && !long_copy) {
        const int blocks = a.n > 0 ? (a.n + tpb - 1) / tpb : 1;
        hipLaunchKernelGGL((k_permute_one<TYPE, V>), dim3(blocks), dim3(1024), 0, st, a, tpb);
        return hipGetLastError();
    }
    const int nch = (int)(pairs / 1024);
    const long waves = wave_items(a.n, a.hidden / V);
    if (waves > MAX_WAVES) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(k_permute_count, dim3(nch), dim3(1024), 0, st, a, nch);
    hipLaunchKernelGGL(k_permute_scan, dim3(1), dim3(1024), 0, st, a, nch);
    hipLaunchKernelGGL(k_permute_place, dim3(nch), dim3(1024), 0, st, a, nch);
    hipLaunchKernelGGL((k_permute_copy<TYPE, V>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int TYPE, int V, bool W>
hipError_t unpermute_t(const UnpermuteArgs &a, hipStream_t st)
{
    const long waves = wave_items(a.n, a.hidden / V);
    if (waves > MAX_WAVES) return hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
    const bool once = reads_once<TYPE>(a.n, a.topk, a.hidden);
#define GO(KMAX)                                                                                           \
    if (once) hipLaunchKernelGGL((k_unpermute<TYPE, V, KMAX, W, true>), grid, block, 0, st, a);            \
    else hipLaunchKernelGGL((k_unpermute<TYPE, V, KMAX, W, false>), grid, block, 0, st, a)
    if (a.topk <= 8) { GO(8); } else { GO(MAX_TOPK); }
#undef GO
    return hipGetLastError();
}

template <int TYPE, int V>
hipError_t unpermute_bwd_t(const UnpermuteBwdArgs &a, hipStream_t st)
{
    if ((long)a.n * 4 > MAX_WAVES) return hipErrorInvalidConfiguration;
    const bool once = reads_once<TYPE>(a.n, a.topk, a.hidden);
    /* fewer tokens than CUs: more threads each (7 tokens of 7,216 bf16, the
     * forward pass included, 13.9 -> 10.2 us) */
    const bool few = a.n <= 256 && a.hidden / V > 256;
#define GO(KMAX, ONCE, NT) hipLaunchKernelGGL((k_unpermute_bwd<TYPE, V, KMAX, ONCE, NT>), dim3(a.n), dim3(NT), 0, st, a)
#define GO_K(KMAX)                                                                                         \
    if (few) GO(KMAX, false, 1024);                                                                        \
    else if (once) GO(KMAX, true, 256);                                                                    \
    else GO(KMAX, false, 256)
    if (a.topk <= 8) { GO_K(8); } else { GO_K(MAX_TOPK); }
#undef GO_K
#undef GO
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
