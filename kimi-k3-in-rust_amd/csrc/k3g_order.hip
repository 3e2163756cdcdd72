/* k3g_order.hip - tokens in expert order and back: the sort of the (token, slot) pairs by
 * expert, token rows gathered into that order, expert rows brought back with the router's
 * weights, and the gradients of both. Device pointers and a stream, no context and no
 * allocation: for callers with experts of their own.
 *
 * With pairs p = t * topk + j, e(p) = idx[p] and pos[p] the place of pair p among the kept
 * pairs in (expert, pair) order:
 *   permute          sorted[pos[p]] = x[p / topk]
 *   its gradient     dx[t] = sum_j dsorted[pos[t, j]]
 *   unpermute        out[t] = sum_j wt[t, j] sorted[pos[t, j]] (+ add[t])
 *   its gradients    dsorted[pos[t, j]] = wt[t, j] dout[t],
 *                    dwt[t, j] = sum_i sorted[pos[t, j]][i] dout[t][i]
 * All four are walked by token: a token's row is read or written once, whatever its topk, and
 * the slots are summed in their order in one thread, so nothing is atomic and the results do
 * not depend on the launch. Memory bounds them where the rows are many (one MI355X, on which a large
 * copy moves 4.7 TB/s: 2,000 x 16 fp32 rows of 3584 back in 83 us, 5.6 TB/s; gradients of 4,096 x 8
 * bf16 rows of 7168 in 188 us, 5.3 TB/s), the launch where they are few (16 rows of 3584 back: 3.5 us
 * of GPU time, 7 with a call's host time). */
#include <stdio.h>

#include "k3g_dev.h"
#include "k3g_host.h"
#include "k3g_kernels.h"

#define OD_MAX_EXPERTS 1024
#define OD_MAX_PAIRS (1 << 23)         /* a block of 256 threads each makes fewer than 2^32 */
#define OD_MAX_WIDTH (1 << 24)
#define OD_THREADS 1024                /* threads of a sort block */
#define OD_WAVES (OD_THREADS / 64)
#define OD_CHUNKS 128                  /* chunks of a sort at most */

/* ------------------------------------------------------------------------ sort ---- */

/* The lanes of the wave with the same key (ballots over its bits; lanes without a key form a
 * group of their own). */
__device__ __forceinline__ uint64_t od_peers(int key, int nb)
{
    uint64_t peers = __ballot(key >= 0);
    if (key < 0) peers = ~peers;
    for (int b = 0; b < nb; ++b) {
        const bool one = key >= 0 && ((key >> b) & 1);
        const uint64_t m = __ballot(one);
        peers &= one ? m : ~m;
    }
    return peers;
}

/* An expert number, -1 for a dropped pair's and, reported, for one past the experts. */
__device__ __forceinline__ int od_valid(int k, int E, int *err)
{
    if (k < E) return k < 0 ? -1 : k;
    k3d_raise(err, K3G_ERR_EXPERT_RANGE);
    return -1;
}

/* The pairs of each expert in each chunk of m * OD_THREADS pairs. */
__global__ void __launch_bounds__(OD_THREADS)
k_order_count(const int32_t *__restrict__ idx, int P, int E, int m, int32_t *__restrict__ cnt)
{
    __shared__ int h[OD_MAX_EXPERTS];
    const int first = blockIdx.x * m * OD_THREADS, end = min(P, first + m * OD_THREADS);
    for (int e = threadIdx.x; e < E; e += OD_THREADS) h[e] = 0;
    __syncthreads();
    for (int p = first + threadIdx.x; p < end; p += 4 * OD_THREADS) {
        int k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = p + i * OD_THREADS < end ? idx[p + i * OD_THREADS] : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k[i] >= 0 && k[i] < E) atomicAdd(&h[k[i]], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += OD_THREADS) cnt[(size_t)blockIdx.x * E + e] = h[e];
}

/* A chunk's pairs into their places: wave w takes m * 64 consecutive pairs, 64 at a time; a
 * pair's rank is the wave's earlier pairs of its expert (a count in LDS) plus those in lanes
 * before it. Then, a thread an expert, the waves' counts become running sums, the chunks before
 * give where the chunk's first pair of it goes (counts of k_order_count; one chunk needs none),
 * and a block scan of the totals gives where the expert begins.
 * M > 0: m = M, and a thread's experts and ranks stay in registers, every load asked for before
 * the first is used (3,702 pairs in one block 11.4 -> 6.0 us, half of it by 16 waves for 8). M = 0:
 * any m; a pair's rank waits in its own entry of pos between the two walks. */
template <int M>
__global__ void __launch_bounds__(OD_THREADS)
k_order_place(const int32_t *__restrict__ idx, int P, int E, int any_m,
              const int32_t *__restrict__ cnt, int nch, int32_t *__restrict__ perm,
              int32_t *__restrict__ off, int32_t *pos, int *err)
{
    __shared__ int wc[OD_WAVES][OD_MAX_EXPERTS];
    __shared__ int first[OD_MAX_EXPERTS];
    __shared__ int red[(OD_WAVES + 1) * 2];
    const int c = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int m = M ? M : any_m;
    const int p0 = (c * OD_WAVES + w) * m * 64, end = min(P, p0 + m * 64);
    int key[M ? M : 1], rank[M ? M : 1];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int p = p0 + 64 * i + lane;
        key[i] = p < end ? idx[p] : -1;
    }
    constexpr int EPT = OD_MAX_EXPERTS / OD_THREADS;
    int tot[EPT], prev[EPT];
#pragma unroll
    for (int u = 0; u < EPT; ++u) {
        const int e = tid + OD_THREADS * u;
        tot[u] = prev[u] = 0;
        if (e >= E) continue;
#pragma unroll
        for (int q = 0; q < OD_WAVES; ++q) wc[q][e] = 0;
        if (nch == 1) continue;
#pragma unroll 16
        for (int q = 0; q < nch; ++q) {
            const int v = cnt[(size_t)q * E + e];
            if (q < c) prev[u] += v;
            tot[u] += v;
        }
    }
    __syncthreads();
    const int nb = 32 - __clz(E > 1 ? E - 1 : 1);
    const uint64_t lt = (1ull << lane) - 1;
    /* rank among the wave's pairs so far; atomics: lanes read what others wrote a step before */
    auto place = [&](int k) {
        const uint64_t peers = od_peers(k, nb);
        const int r = __popcll(peers & lt);
        const int before = k >= 0 ? __hip_atomic_load(&wc[w][k], __ATOMIC_RELAXED,
                                                      __HIP_MEMORY_SCOPE_WAVEFRONT) : 0;
        __builtin_amdgcn_wave_barrier();
        if (k >= 0 && r == 0)
            __hip_atomic_store(&wc[w][k], before + __popcll(peers), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WAVEFRONT);
        __builtin_amdgcn_wave_barrier();
        return before + r;
    };
    if constexpr (M > 0) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            key[i] = od_valid(key[i], E, err);
            rank[i] = place(key[i]);
        }
    } else {
        for (int p = p0 + lane; p - lane < end; p += 64) {
            const int k = od_valid(p < end ? idx[p] : -1, E, err), r = place(k);
            if (p < end) pos[p] = k >= 0 ? r : -1;
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < EPT; ++u) {
        const int e = tid + OD_THREADS * u;
        if (e >= E) continue;
        int s = 0;
#pragma unroll
        for (int q = 0; q < OD_WAVES; ++q) {
            const int v = wc[q][e];
            wc[q][e] = s;
            s += v;
        }
        if (nch == 1) tot[u] = s;
    }
    int v[EPT], all[EPT], at = 0;
#pragma unroll
    for (int u = 0; u < EPT; ++u) v[u] = tot[u];
    k3d_block_exscan_n<EPT, OD_WAVES>(v, all, red);
#pragma unroll
    for (int u = 0; u < EPT; ++u) {
        const int e = tid + OD_THREADS * u;
        if (e < E) {
            first[e] = at + v[u] + prev[u];
            if (c == 0) off[e] = at + v[u];
        }
        at += all[u];
    }
    if (c == 0 && tid == 0) off[E] = at;
    __syncthreads();
    if constexpr (M > 0) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int p = p0 + 64 * i + lane;
            if (p >= end) continue;
            const int at = key[i] >= 0 ? first[key[i]] + wc[w][key[i]] + rank[i] : -1;
            if (at >= 0) perm[at] = p;
            pos[p] = at;
        }
    } else {
        for (int p = p0 + lane; p < end; p += 64) {
            const int r = pos[p];
            if (r < 0) continue;
            const int e = idx[p], at = first[e] + wc[w][e] + r;
            perm[at] = p;
            pos[p] = at;
        }
    }
}

/* ------------------------------------------------------------------ row vectors ---- */

/* 16 bytes of a row, whatever the row's alignment (rows of an odd width begin at any element;
 * global loads of 16 bytes take any address). */
typedef uint32_t od_v4u __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <typename T> struct OdRow;
template <> struct OdRow<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ void get(const od_v4u &u, float *f)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(u[i]);
    }
    static __device__ __forceinline__ od_v4u put(const float *f)
    {
        return od_v4u{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3])};
    }
};
template <> struct OdRow<uint16_t> {
    static constexpr int V = 8;
    static __device__ __forceinline__ void get(const od_v4u &u, float *f)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = k3d_bf16lo(u[i]);
            f[2 * i + 1] = k3d_bf16hi(u[i]);
        }
    }
    static __device__ __forceinline__ od_v4u put(const float *f)
    {
        od_v4u u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = k3d_bf16x2(f[2 * i], f[2 * i + 1]);
        return u;
    }
};

/* Vector v of the n-element row at p: whole ones in one load or store, the last one's elements
 * one by one when n ends inside it. STREAM: marked as not to be kept in the caches. The sorted rows
 * are read or written once in a call; where they are more than the 256 MB of the last-level cache
 * (OD_STREAM), keeping them only drives other rows out and their write-back meets the next reads
 * (4,096 x 8 bf16 rows of 7168 there and back 238 -> 217 us, 2,000 x 16 fp32 rows of 3584 back 94
 * -> 83); fewer may still be there for the caller's next kernel. */
#define OD_STREAM ((size_t)256 << 20)

template <bool STREAM = false, typename T>
__device__ __forceinline__ od_v4u od_load(const T *p, int v, int n)
{
    constexpr int V = OdRow<T>::V;
    if (V * (v + 1) <= n) {
        const od_v4u *a = (const od_v4u *)(p + V * v);
        return STREAM ? __builtin_nontemporal_load(a) : *a;
    }
    T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = V * v + i < n ? p[V * v + i] : (T)0;
    od_v4u u;
    __builtin_memcpy(&u, e, 16);
    return u;
}

template <bool STREAM = false, typename T>
__device__ __forceinline__ void od_store(T *p, int v, int n, const od_v4u &u)
{
    constexpr int V = OdRow<T>::V;
    if (V * (v + 1) <= n) {
        od_v4u *a = (od_v4u *)(p + V * v);
        if (STREAM) __builtin_nontemporal_store(u, a);
        else *a = u;
        return;
    }
    T e[V];
    __builtin_memcpy(e, &u, 16);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (V * v + i < n) p[V * v + i] = e[i];
}

/* --------------------------------------------------------------------- kernels ---- */

/* A block of 256 threads is 256 >> tx_log tokens of 1 << tx_log vectors each; the grid is
 * (tokens, vectors). */
struct OdGrid {
    int T, k, n, P, tx_log;
};

/* This thread's token and vector; false past the last. WIDE: a wave has one token, which is then
 * known to be the same in every lane (its places and weights come by scalar loads). */
template <typename T, bool WIDE>
__device__ __forceinline__ bool od_mine(const OdGrid &g, int &t, int &v)
{
    t = blockIdx.x * (256 >> g.tx_log) + (threadIdx.x >> g.tx_log);
    if (WIDE) t = __builtin_amdgcn_readfirstlane(t);
    v = (blockIdx.y << g.tx_log) + (threadIdx.x & ((1 << g.tx_log) - 1));
    return t < g.T && OdRow<T>::V * v < g.n;
}

template <typename T, bool WIDE, bool STREAM>
__global__ void __launch_bounds__(256)
k_permute(const OdGrid g, const T *__restrict__ x, const int32_t *__restrict__ pos,
          T *__restrict__ sorted)
{
    int t, v;
    if (!od_mine<T, WIDE>(g, t, v)) return;
    const od_v4u u = od_load(x + (size_t)t * g.n, v, g.n);
    const int32_t *pt = pos + (size_t)t * g.k;
#pragma unroll 4
    for (int j = 0; j < g.k; ++j) {
        const int p = pt[j];
        if ((unsigned)p < (unsigned)g.P) od_store<STREAM>(sorted + (size_t)p * g.n, v, g.n, u);
    }
}

/* out[t] = sum_j w_j row_j, products and sums rounded separately in slot order as the layer's
 * combine does, then + add[t]; without weights the gradient of k_permute. Eight rows are asked
 * for before the first is added (one after the other the 16 rows of a decoding token took 6.2 us). */
template <typename T, bool WIDE, bool STREAM>
__global__ void __launch_bounds__(256)
k_unpermute(const OdGrid g, const T *__restrict__ sorted, const int32_t *__restrict__ pos,
            const float *__restrict__ wt, const T *__restrict__ add, T *__restrict__ out)
{
    constexpr int V = OdRow<T>::V, AHEAD = 8;
    int t, v;
    if (!od_mine<T, WIDE>(g, t, v)) return;
    const int32_t *pt = pos + (size_t)t * g.k;
    const float *wrow = wt ? wt + (size_t)t * g.k : nullptr;
    float acc[V], f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    od_v4u extra = {0, 0, 0, 0};
    if (add) extra = od_load(add + (size_t)t * g.n, v, g.n);
    for (int j0 = 0; j0 < g.k; j0 += AHEAD) {
        int p[AHEAD];
        float w[AHEAD];
        od_v4u u[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            p[i] = j0 + i < g.k ? pt[j0 + i] : -1;
            w[i] = wt && j0 + i < g.k ? wrow[j0 + i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if ((unsigned)p[i] < (unsigned)g.P) u[i] = od_load<STREAM>(sorted + (size_t)p[i] * g.n, v, g.n);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if ((unsigned)p[i] >= (unsigned)g.P) continue;
            OdRow<T>::get(u[i], f);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += wt ? w[i] * f[e] : f[e];
        }
    }
    if (add) {
        OdRow<T>::get(extra, f);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += f[i];
    }
    od_store(out + (size_t)t * g.n, v, g.n, OdRow<T>::put(acc));
}

/* WV waves (a block of four) per JB slots of a token: their rows of dsorted and entries of dwt from
 * one read of dout; a token's slots on one XCD (block b runs on XCD b % 8), whose L2 then serves
 * dout to the next ones. */
template <typename T, int WV, int JB, bool STREAM>
__global__ void __launch_bounds__(256)
k_unpermute_grad(const OdGrid g, const T *__restrict__ dout, const T *__restrict__ sorted,
                 const int32_t *__restrict__ pos, const float *__restrict__ wt,
                 T *__restrict__ dsorted, float *__restrict__ dwt)
{
    constexpr int V = OdRow<T>::V, PER = 4 / WV;
    __shared__ float part[JB][4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & (64 * WV - 1);
    const int xcd = blockIdx.x & 7, s = (blockIdx.x >> 3) * PER + wave / WV, ng = (g.k + JB - 1) / JB;
    const int t = 8 * (s / ng) + xcd, j0 = s % ng * JB;
    if (t >= g.T) return;
    const size_t pair = (size_t)t * g.k + j0;
    int p[JB];
    float w[JB], sum[JB];
#pragma unroll
    for (int i = 0; i < JB; ++i) {
        p[i] = j0 + i < g.k ? pos[pair + i] : -1;
        if ((unsigned)p[i] >= (unsigned)g.P) p[i] = -1;
        w[i] = dsorted && p[i] >= 0 ? wt[pair + i] : 0.0f;
        sum[i] = 0.0f;
    }
    for (int v = lane; V * v < g.n; v += 64 * WV) {
        float go[V], f[V];
        od_v4u u[JB];
        const od_v4u d = od_load(dout + (size_t)t * g.n, v, g.n);
        if (dwt) {
#pragma unroll
            for (int i = 0; i < JB; ++i)
                if (p[i] >= 0) u[i] = od_load<STREAM>(sorted + (size_t)p[i] * g.n, v, g.n);
        }
        OdRow<T>::get(d, go);
#pragma unroll
        for (int i = 0; i < JB; ++i) {
            if (p[i] < 0) continue;
            if (dwt) {
                OdRow<T>::get(u[i], f);
#pragma unroll
                for (int e = 0; e < V; ++e) sum[i] += f[e] * go[e];
            }
            if (dsorted) {
#pragma unroll
                for (int e = 0; e < V; ++e) f[e] = w[i] * go[e];
                od_store<STREAM>(dsorted + (size_t)p[i] * g.n, v, g.n, OdRow<T>::put(f));
            }
        }
    }
    if (!dwt) return;
#pragma unroll
    for (int i = 0; i < JB; ++i) sum[i] = k3d_wave_sum(sum[i]);
    if (WV == 1) {
#pragma unroll
        for (int i = 0; i < JB; ++i)
            if (lane == 0 && j0 + i < g.k) dwt[pair + i] = sum[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < JB; ++i)
        if ((threadIdx.x & 63) == 0) part[i][wave] = sum[i];
    __syncthreads();
    if (threadIdx.x < JB && j0 + (int)threadIdx.x < g.k) {
        const float *q = part[threadIdx.x];
        dwt[pair + threadIdx.x] = q[0] + q[1] + q[2] + q[3];
    }
}

/* ------------------------------------------------------------------ entry points ---- */

/* Chunks of the sort and the multiple m of OD_THREADS pairs that each has. Up to 4096 pairs one
 * block does all (5,600 in one block 11.0 us, in chunks 7.8); past that a chunk is 2048, 4096 or
 * 8192 pairs, or what makes 128 chunks: every chunk reads the counts of all, so there are few.
 * us, on 384 experts: 8 pairs 3.4, 1024 3.8, 4096 7.4, 32,768 8.1, 524,288 18.6. */
static int sort_chunks(int P, int *m)
{
    int per = P <= OD_THREADS ? 1 : P <= 2 * OD_THREADS ? 2 : 4;
    if (P > 4 * OD_THREADS) {
        if (P <= 32 * 2 * OD_THREADS) per = 2;
        else if (P > 32 * 4 * OD_THREADS) per = 8;
        if (P > OD_CHUNKS * 8 * OD_THREADS)
            per = (P + OD_CHUNKS * OD_THREADS - 1) / (OD_CHUNKS * OD_THREADS);
    }
    *m = per;
    return P ? (P + per * OD_THREADS - 1) / (per * OD_THREADS) : 1;
}

/* sizes every call here shares: 0 when they are ones the kernels take */
static int bad_sizes(const char *who, int T, int topk)
{
    if (T < 0 || topk < 1 || topk > K3G_MAX_TOPK || (int64_t)T * topk > OD_MAX_PAIRS) {
        fprintf(stderr, "%s: needs 0 <= tokens, 1 <= topk <= %d and at most %d pairs (%d x %d)\n", who,
                K3G_MAX_TOPK, OD_MAX_PAIRS, T, topk);
        return 1;
    }
    return 0;
}

extern "C" size_t k3g_sort_bytes(int T, int topk, int n_experts)
{
    if (T < 0 || topk < 1 || topk > K3G_MAX_TOPK || (int64_t)T * topk > OD_MAX_PAIRS ||
        n_experts < 1 || n_experts > OD_MAX_EXPERTS)
        return 0;
    int m;
    const int nch = sort_chunks(T * topk, &m);
    return nch > 1 ? (size_t)nch * n_experts * sizeof(int32_t) : 0;
}

extern "C" int k3g_sort_tokens(const int32_t *idx, int T, int topk, int n_experts, int32_t *perm,
                               int32_t *off, int32_t *pos, int *err, void *work,
                               size_t work_bytes, void *stream)
{
    const char *who = "k3g_sort_tokens";
    if (bad_sizes(who, T, topk)) return -1;
    if (n_experts < 1 || n_experts > OD_MAX_EXPERTS) {
        fprintf(stderr, "%s: needs 1 to %d experts (%d)\n", who, OD_MAX_EXPERTS, n_experts);
        return -1;
    }
    const int P = T * topk;
    if (!off || (P && (!idx || !perm || !pos)) || k3h_misaligned(idx, 4) || k3h_misaligned(perm, 4) ||
        k3h_misaligned(off, 4) || k3h_misaligned(pos, 4) || k3h_misaligned(err, 4) ||
        k3h_misaligned(work, 4)) {
        fprintf(stderr, "%s: a pointer is missing or not aligned to 4 bytes\n", who);
        return -1;
    }
    const size_t need = k3g_sort_bytes(T, topk, n_experts);
    if (need && (!work || work_bytes < need)) {
        fprintf(stderr, "%s: needs %zu bytes of workspace (%zu given)\n", who, need,
                work ? work_bytes : (size_t)0);
        return -1;
    }
    K3hOn on(stream);
    if (!on.ok) return -1;
    int m;
    const int nch = sort_chunks(P, &m);
    int32_t *cnt = (int32_t *)work;
    if (nch > 1 && k3h_launch(who, k_order_count, dim3(nch), dim3(OD_THREADS), on.st, idx, P, n_experts, m,
                              cnt))
        return -1;
    auto *place = m == 1 ? k_order_place<1> : m == 2 ? k_order_place<2> : m == 4 ? k_order_place<4>
                : m == 8 ? k_order_place<8> : k_order_place<0>;
    return k3h_launch(who, place, dim3(nch), dim3(OD_THREADS), on.st, idx, P, n_experts, m,
                      (const int32_t *)cnt, nch, perm, off, pos, err);
}

namespace {

/* The instance for these rows: WIDE when a wave has one token, STREAM when the sorted rows are more
 * than the last-level cache holds. */
#define OD_PICK(K, T, g)                                                                       \
    ((size_t)(g).P * (g).n * sizeof(T) > OD_STREAM                                             \
         ? ((g).tx_log >= 6 ? K<T, true, true> : K<T, false, true>)                            \
         : ((g).tx_log >= 6 ? K<T, true, false> : K<T, false, false>))

/* The checks the row calls share; rows and tokens as an OdGrid with its launch. */
int row_sizes(const char *who, int dt, int T, int topk, int n)
{
    if (bad_sizes(who, T, topk)) return -1;
    if (dt != K3_WF32 && dt != K3_WBF16) {
        fprintf(stderr, "%s: rows are fp32 (%d) or bf16 (%d), not %d\n", who, K3_WF32, K3_WBF16, dt);
        return -1;
    }
    if (n < 1 || n > OD_MAX_WIDTH) {
        fprintf(stderr, "%s: needs a width of 1 to %d (%d)\n", who, OD_MAX_WIDTH, n);
        return -1;
    }
    return 0;
}

int row_pointer(const char *who, const char *name, const void *p, int size, bool needed)
{
    if (needed && !p) {
        fprintf(stderr, "%s: %s is missing\n", who, name);
        return -1;
    }
    if (k3h_misaligned(p, size)) {
        fprintf(stderr, "%s: %s is not aligned to its elements (%d bytes)\n", who, name, size);
        return -1;
    }
    return 0;
}

dim3 row_grid(OdGrid &g, int V)
{
    const int nv = (g.n + V - 1) / V;
    g.tx_log = 0;
    while (g.tx_log < 8 && (1 << g.tx_log) < nv) ++g.tx_log;
    const int ty = 256 >> g.tx_log;
    return dim3((g.T + ty - 1) / ty, (nv + (1 << g.tx_log) - 1) >> g.tx_log);
}

}  // namespace

extern "C" int k3g_permute(const void *x, int dt, int T, int topk, int n, const int32_t *pos,
                           void *sorted, void *stream)
{
    const char *who = "k3g_permute";
    if (row_sizes(who, dt, T, topk, n)) return -1;
    const int size = dt == K3_WBF16 ? 2 : 4;
    if (row_pointer(who, "x", x, size, T > 0) || row_pointer(who, "pos", pos, 4, T > 0) ||
        row_pointer(who, "sorted", sorted, size, T > 0))
        return -1;
    if (!T) return 0;
    K3hOn on(stream);
    if (!on.ok) return -1;
    OdGrid g = {T, topk, n, T * topk, 0};
    const dim3 grid = row_grid(g, 16 / size);
    if (dt == K3_WBF16)
        return k3h_launch(who, OD_PICK(k_permute, uint16_t, g), grid, dim3(256), on.st, (const OdGrid)g,
                          (const uint16_t *)x, pos, (uint16_t *)sorted);
    return k3h_launch(who, OD_PICK(k_permute, float, g), grid, dim3(256), on.st, (const OdGrid)g, (const float *)x,
                      pos, (float *)sorted);
}

static int unpermute(const char *who, const void *sorted, int dt, int T, int topk, int n,
                     const int32_t *pos, const float *wt, const void *add, void *out, void *stream)
{
    if (row_sizes(who, dt, T, topk, n)) return -1;
    const int size = dt == K3_WBF16 ? 2 : 4;
    if (row_pointer(who, "the sorted rows", sorted, size, T > 0) ||
        row_pointer(who, "pos", pos, 4, T > 0) || row_pointer(who, "wt", wt, 4, false) ||
        row_pointer(who, "add", add, size, false) || row_pointer(who, "the output", out, size, T > 0))
        return -1;
    if (!T) return 0;
    K3hOn on(stream);
    if (!on.ok) return -1;
    OdGrid g = {T, topk, n, T * topk, 0};
    const dim3 grid = row_grid(g, 16 / size);
    if (dt == K3_WBF16)
        return k3h_launch(who, OD_PICK(k_unpermute, uint16_t, g), grid, dim3(256), on.st, (const OdGrid)g,
                          (const uint16_t *)sorted, pos, wt, (const uint16_t *)add, (uint16_t *)out);
    return k3h_launch(who, OD_PICK(k_unpermute, float, g), grid, dim3(256), on.st, (const OdGrid)g,
                      (const float *)sorted, pos, wt, (const float *)add, (float *)out);
}

extern "C" int k3g_permute_grad(const void *dsorted, int dt, int T, int topk, int n,
                                const int32_t *pos, void *dx, void *stream)
{
    return unpermute("k3g_permute_grad", dsorted, dt, T, topk, n, pos, nullptr, nullptr, dx, stream);
}

extern "C" int k3g_unpermute(const void *sorted, int dt, int T, int topk, int n, const int32_t *pos,
                             const float *wt, const void *add, void *out, void *stream)
{
    if (T > 0 && !wt) {
        fprintf(stderr, "k3g_unpermute: wt is missing\n");
        return -1;
    }
    return unpermute("k3g_unpermute", sorted, dt, T, topk, n, pos, wt, add, out, stream);
}

extern "C" int k3g_unpermute_grad(const void *dout, const void *sorted, int dt, int T, int topk,
                                  int n, const int32_t *pos, const float *wt, void *dsorted,
                                  float *dwt, void *stream)
{
    const char *who = "k3g_unpermute_grad";
    if (row_sizes(who, dt, T, topk, n)) return -1;
    const int size = dt == K3_WBF16 ? 2 : 4;
    if (row_pointer(who, "dout", dout, size, T > 0) || row_pointer(who, "pos", pos, 4, T > 0) ||
        row_pointer(who, "sorted", sorted, size, T > 0 && dwt) ||
        row_pointer(who, "wt", wt, 4, T > 0 && dsorted) ||
        row_pointer(who, "dsorted", dsorted, size, false) || row_pointer(who, "dwt", dwt, 4, false))
        return -1;
    if (!dsorted && !dwt) {
        fprintf(stderr, "%s: neither gradient is asked for\n", who);
        return -1;
    }
    if (!T) return 0;
    K3hOn on(stream);
    if (!on.ok) return -1;
    const OdGrid g = {T, topk, n, T * topk, 0};
    /* Short rows: a wave each. Four slots together where the rows are bf16 and make enough blocks all
     * the same: us, 3,978 x 15 rows of 535 41.8 -> 35.5, 4,096 x 8 of 2048 57 -> 45, of 64 9.9 -> 7.3,
     * of 7168 190 -> 189; fp32 rows, whose loads are twice as many, lose (4,096 x 8 of 256 14.0 ->
     * 17.4, 2,000 x 16 of 3584 185 -> 238). */
    const bool wave = n <= 128 * (16 / size), four = size == 2 && g.P >= 4096 && topk >= 3;
    const int64_t slots = (int64_t)((T + 7) / 8) * (four ? (topk + 3) / 4 : topk);
    const dim3 grid((unsigned)(8 * (wave ? (slots + 3) / 4 : slots)));
    const bool big = (size_t)g.P * n * size > OD_STREAM;
#define OD_GRAD(T, JB)                                                                                   \
    (big ? (wave ? k_unpermute_grad<T, 1, JB, true> : k_unpermute_grad<T, 4, JB, true>)                  \
         : (wave ? k_unpermute_grad<T, 1, JB, false> : k_unpermute_grad<T, 4, JB, false>))
    if (dt == K3_WBF16)
        return k3h_launch(who, four ? OD_GRAD(uint16_t, 4) : OD_GRAD(uint16_t, 1), grid, dim3(256), on.st, g,
                          (const uint16_t *)dout, (const uint16_t *)sorted, pos, wt, (uint16_t *)dsorted, dwt);
    return k3h_launch(who, OD_GRAD(float, 1), grid, dim3(256), on.st, g, (const float *)dout,
                      (const float *)sorted, pos, wt, (float *)dsorted, dwt);
}
