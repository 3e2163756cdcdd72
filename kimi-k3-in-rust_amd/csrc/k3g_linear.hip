/* k3g_linear.hip - products by matrices in plain rows, fp32 or bf16, one matrix or an expert's each
 * over the sorted rows, with what follows them in the epilogue, and their gradients.
 *
 *   forward    z[r][n] = sum_c x[row(r)][c] W[n][c] + bias[n],  y = act(z (, z3)) + residual
 *   grad_x     g[r][c] = sum_n dy[r][n] W[n][c] (+ dy3, W3) + add,  dx = g or g act'(z)
 *   grad_w     dW[n][c] = sum_r dy[r][n] x[row(r)][c],  dbias[n] = sum_r dy[r][n]
 *
 * All three are one tile O[b][a] = sum_k A[a][k] B[k][b], a the index that is contiguous in the
 * output: A is the matrix operand of the first two (rows a and contiguous k forward; contiguous a
 * in rows k backward) and the rows x of the third (contiguous a), B the rows x or dy (contiguous k)
 * and, of the third, dy with contiguous b. The matrix instruction's accumulator then holds four
 * consecutive a of one b a lane.
 */
#include <stdio.h>

#include "k3g_act.h"
#include "k3g_dev.h"
#include "k3g_gemm.h"
#include "k3g_groups.h"
#include "k3g_host.h"
#include "k3g_kernels.h"

#define LN_MAX_ROWS (1 << 23)
#define LN_MAX_WIDTH (1 << 20)

enum { LN_FWD, LN_GRAD_X, LN_GRAD_W };

struct LnArgs {
    const uint8_t *a, *a3;           /* the matrices (off NULL) or the first expert's pointers; grad_w: x */
    const uint8_t *b, *b3;           /* the rows: x, dy and dy3, dy */
    const int32_t *perm;             /* place -> pair, or NULL: place r is row r */
    uint32_t magic;                  /* ceil(2^32 / topk), 0 for a topk of 1 */
    int pairs;
    const int32_t *off;              /* [E + 1] places of each expert, or NULL: one, all places */
    int E, P;                        /* P places at most */
    int64_t step, dstep;             /* bytes from one expert's pointer to the next, of a and of y (grad_w) */
    int NA, NB, K;                   /* extents of a, of b (grad_w), of k (not grad_w) */
    uint8_t *y;                      /* the output; grad_w with off: the first expert's pointer to it */
    int act;
    float b1, b2, i1, i2;            /* caps and their reciprocals */
    const float *bias, *bias3;
    const uint8_t *add;              /* the residual, or what grad_x adds */
    uint8_t *z, *z3, *dz3;
    int accumulate;
    float *dbias;
};

/* ------------------------------------------------------------ values in memory ---- */

/* 16 bytes at any address that two have */
typedef gm_v4u ln_any16 __attribute__((aligned(2)));
typedef gm_v2u ln_any8 __attribute__((aligned(2)));
#ifdef __HIP_DEVICE_COMPILE__
#define LN_G(T) __attribute__((address_space(1))) T
#else
#define LN_G(T) T
#endif

__device__ __forceinline__ k3v4f ln_get4(const float *p, int n)
{
    const LN_G(float) *g = (const LN_G(float) *)p;
    if (n >= 4) {
        const gm_v4u v = *(const LN_G(ln_any16) *)g;
        return __builtin_bit_cast(k3v4f, v);
    }
    return k3v4f{g[0], n > 1 ? g[1] : 0.0f, n > 2 ? g[2] : 0.0f, 0.0f};
}

__device__ __forceinline__ k3v4f ln_get4(const uint16_t *p, int n)
{
    const LN_G(uint16_t) *g = (const LN_G(uint16_t) *)p;
    gm_v2u v;
    if (n >= 4) v = *(const LN_G(ln_any8) *)g;
    else v = gm_v2u{g[0] | (n > 1 ? (uint32_t)g[1] << 16 : 0u), n > 2 ? g[2] : 0u};
    return k3v4f{k3d_bf16lo(v.x), k3d_bf16hi(v.x), k3d_bf16lo(v.y), k3d_bf16hi(v.y)};
}

__device__ __forceinline__ void ln_put4(float *p, int n, const k3v4f &v)
{
    LN_G(float) *g = (LN_G(float) *)p;
    if (n >= 4) {
        *(LN_G(ln_any16) *)g = __builtin_bit_cast(gm_v4u, v);
        return;
    }
    g[0] = v[0];
    if (n > 1) g[1] = v[1];
    if (n > 2) g[2] = v[2];
}

__device__ __forceinline__ void ln_put4(uint16_t *p, int n, const k3v4f &v)
{
    LN_G(uint16_t) *g = (LN_G(uint16_t) *)p;
    const gm_v2u u = {k3d_bf16x2(v[0], v[1]), k3d_bf16x2(v[2], v[3])};
    if (n >= 4) {
        *(LN_G(ln_any8) *)g = u;
        return;
    }
    g[0] = (uint16_t)u.x;
    if (n > 1) g[1] = (uint16_t)(u.x >> 16);
    if (n > 2) g[2] = (uint16_t)u.y;
}

/* A unit: 8 consecutive values as they lie */
template <typename T>
struct LnUnit {
    gm_v4u v[sizeof(T) / 2];
};

/* n of them, zeros behind and for n <= 0 */
template <typename T>
__device__ __forceinline__ LnUnit<T> ln_unit(const T *p, int n)
{
    LnUnit<T> u;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.v[i] = gm_v4u{0, 0, 0, 0};
    if (n >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.v[i] = ((const LN_G(ln_any16) *)p)[i];
    } else if (n > 0) {
        const LN_G(T) *g = (const LN_G(T) *)p;
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            if (i >= n) continue;
            if constexpr (sizeof(T) == 4) u.v[i >> 2][i & 3] = __float_as_uint(g[i]);
            else u.v[0][i >> 1] |= (uint32_t)g[i] << (16 * (i & 1));
        }
    }
    return u;
}

/* Its bf16 pieces: one of bf16 values; of fp32 values three, 8 bits each, their sum exact as long as
 * the last is a normal number. The first is truncated, so none of a finite value is infinite, the
 * second rounded to nearest, so the last has either sign and the pairs of pieces that a product of
 * two fp32 values leaves out have no bias. An infinity is its first piece alone. */
template <typename T> constexpr int ln_pieces = sizeof(T) == 4 ? 3 : 1;

__device__ __forceinline__ void ln_split(const LnUnit<uint16_t> &u, gm_v4u (&p)[1]) { p[0] = u.v[0]; }

__device__ __forceinline__ void ln_split(const LnUnit<float> &u, gm_v4u (&p)[3])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[2];
        float r[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int e = 2 * i + j;
            h[j] = u.v[e >> 2][e & 3];
            const float x = __uint_as_float(h[j]);
            r[j] = fabsf(x) == __builtin_inff() ? 0.0f : x - __uint_as_float(h[j] & 0xFFFF0000u);
        }
        p[0][i] = __builtin_amdgcn_perm(h[1], h[0], 0x07060302u);
        p[1][i] = k3d_bf16x2(r[0], r[1]);
        p[2][i] = __builtin_amdgcn_perm(__float_as_uint(r[1] - k3d_bf16hi(p[1][i])),
                                        __float_as_uint(r[0] - k3d_bf16lo(p[1][i])), 0x07060302u);
    }
}

/* acc += A B: every pair of pieces but, of two fp32 operands, the three below 2^-23 of the product */
template <int PA, int PB>
__device__ __forceinline__ void ln_mma(const k3v8bf (&a)[PA], const k3v8bf (&b)[PB], k3v4f &acc)
{
#pragma unroll
    for (int i = PA - 1; i >= 0; --i)
#pragma unroll
        for (int j = PB - 1; j >= 0; --j)
            if (i + j <= 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc, 0, 0, 0);
}

/* ------------------------------------------------------------- rows and experts ---- */

/* the row of x that a place takes; -1 (zeros) for no pair of these tokens */
__device__ __forceinline__ int ln_row(const LnArgs &g, int place)
{
    if (!g.perm) return place;
    const uint32_t pair = (uint32_t)g.perm[place];
    if (pair >= (uint32_t)g.pairs) return -1;
    return (int)(g.magic ? __umulhi(pair, g.magic) : pair);
}

__device__ __forceinline__ const uint8_t *ln_matrix(const LnArgs &g, const uint8_t *w, int e)
{
    if (!g.off) return w;
    return gm_uniform_ptr(*(const uint8_t *const *)(w + (size_t)e * g.step));
}

/* ------------------------------------------------------------------- epilogue ---- */

/* What follows four consecutive sums v (and u, of the second matrix) of output row `row`, from
 * column a on: n of them are stored. */
template <int MODE, bool GATED, typename Y>
__device__ __forceinline__ void ln_finish(const LnArgs &g, Y *out, int e, size_t row, int a, k3v4f v, k3v4f u)
{
    const int n = min(4, g.NA - a);
    const size_t at = row * g.NA + a;
    if constexpr (MODE == LN_FWD) {
        if (g.bias) v += ln_get4(g.bias + (size_t)e * g.NA + a, n);
        if (GATED && g.bias3) u += ln_get4(g.bias3 + (size_t)e * g.NA + a, n);
        if (g.z) ln_put4((Y *)g.z + at, n, v);
        if (GATED && g.z3) ln_put4((Y *)g.z3 + at, n, u);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = GATED ? ka_situ(v[i], u[i], g.b1, g.b2, g.i1, g.i2) : ka_act(g.act, v[i]);
        if (g.add) v += ln_get4((const Y *)g.add + at, n);
    } else if constexpr (MODE == LN_GRAD_X) {
        if (g.add) v += ln_get4((const Y *)g.add + at, n);
        if (g.z) {
            const k3v4f z = ln_get4((const Y *)g.z + at, n);
            if (g.dz3) {
                const k3v4f z3 = ln_get4((const Y *)g.z3 + at, n);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float dg, du;
                    ka_situ_slopes(z[i], z3[i], g.b1, g.b2, g.i1, g.i2, dg, du);
                    u[i] = v[i] * du;
                    v[i] *= dg;
                }
                ln_put4((Y *)g.dz3 + at, n, u);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] *= ka_slope(g.act, z[i]);
            }
        }
    } else {
        if (g.accumulate) v += ln_get4(out + at, n);
    }
    ln_put4(out + at, n, v);
}

/* A wave's sums (MA x MB blocks of 16 a x 16 b) out by way of LDS (16 x (16 MA + 4) floats of its
 * own), so that it reads and writes whole pieces of rows: rows row0 + 0 .. rows - 1, columns col0 on.
 * GATED: the blocks are the two matrices' in turn. */
template <int MODE, bool GATED, typename Y, int MA, int MB>
__device__ __forceinline__ void ln_out(const LnArgs &g, float *lds, const k3v4f (&acc)[MA][MB], Y *out, int e,
                                       size_t row0, int rows, int col0)
{
    constexpr int PITCH = 16 * MA + 4, LANES = (GATED ? 2 : 4) * MA, STEP = 64 / LANES;
    const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const int f = 4 * (lane % LANES), from = GATED ? 32 * (f >> 4) + (f & 15) : f;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        gm_wave_sync();
#pragma unroll
        for (int i = 0; i < MA; ++i) *(k3v4f *)(lds + c * PITCH + 16 * i + 4 * q) = acc[i][j];
        gm_wave_sync();
#pragma unroll 2
        for (int r = lane / LANES; r < 16; r += STEP) {
            if (16 * j + r >= rows || col0 + f >= g.NA) continue;
            const float *o = lds + r * PITCH + from;
            const k3v4f v = *(const k3v4f *)o, u = GATED ? *(const k3v4f *)(o + 16) : k3v4f{0.f, 0.f, 0.f, 0.f};
            ln_finish<MODE, GATED, Y>(g, out, e, row0 + 16 * j + r, col0 + f, v, u);
        }
    }
}

/* rows x n zeros of an output (an expert without a matrix) */
template <int MODE, bool GATED, typename Y, int THREADS>
__device__ __forceinline__ void ln_zeros(const LnArgs &g, Y *out, size_t row0, int rows, int col0, int n)
{
    n = min(n, g.NA - col0);
    for (int i = threadIdx.x; i < rows * n; i += THREADS) {
        const size_t at = (row0 + i / n) * g.NA + col0 + i % n;
        out[at] = (Y)0;
        if (MODE == LN_FWD && g.z) ((Y *)g.z)[at] = (Y)0;
        if (MODE == LN_FWD && GATED && g.z3) ((Y *)g.z3)[at] = (Y)0;
        if (MODE == LN_GRAD_X && g.dz3) ((Y *)g.dz3)[at] = (Y)0;
    }
}

/* ---- which tile a workgroup takes: rows p0 .. p0 + np of expert e, a from a0, b from b0 (grad_w) ---- */
struct LnTile {
    int e, p0, np, a0, b0;
};

/* grad_w: every expert's tiles are shared out among the XCDs, an eighth in a row each, the first
 * eighth to another XCD for every expert; so a popular expert's do not lie on one, and an XCD's
 * neighbours read the same rows. */
template <int MODE, int TA, int TB>
__device__ __forceinline__ bool ln_tile(const LnArgs &g, LnTile &t)
{
    if constexpr (MODE == LN_GRAD_W) {
        const int na = (g.NA + TA - 1) / TA, nb = (g.NB + TB - 1) / TB, tiles = na * nb, per = (tiles + 7) / 8;
        const int s = blockIdx.x >> 3;
        t.e = s / per;
        const int i = ((blockIdx.x + t.e) & 7) * per + s - t.e * per;
        if (i >= tiles) return false;
        t.b0 = i / na * TB;
        t.a0 = i % na * TA;
        t.p0 = 0;
        t.np = g.P;
        if (g.off) {
            t.p0 = min(max(g.off[t.e], 0), g.P);
            t.np = min(max(g.off[t.e + 1], t.p0), g.P) - t.p0;
        }
        return true;
    } else {
        int ft;
        if (!gm_row_item<TB>(g.off, g.E, g.P, (g.NA + TA - 1) / TA, ft, t.e, t.p0, t.np)) return false;
        t.a0 = ft * TA;
        t.b0 = 0;
        return true;
    }
}

/* ------------------------------------------------------------------- LDS tiles ----
 *
 * An operand's tile of 32 k, bf16: contiguous k: rows of 64 bytes, 16-byte unit u of row r at slot
 * u ^ (r / 2 % 4); contiguous a (or b): 32 rows k of 128 values, 256 bytes, the 32-byte piece c at
 * slot c ^ (k % 4 + 4 (k / 8 % 2)), which the transposing read takes four rows k of at once. */
__device__ __forceinline__ int ln_krow(int row, int u) { return 64 * row + 16 * (u ^ ((row >> 1) & 3)); }
__device__ __forceinline__ int ln_swap(int k) { return (k & 3) | ((k >> 1) & 4); }

typedef short ln_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ln_v4s *ln_l4s;

__device__ __forceinline__ gm_v2u ln_read_tr(const uint8_t *p)
{
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_bit_cast(gm_v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ln_l4s)p));
#else
    return gm_v2u{};
#endif
}

/* block i's operand from a tile whose rows are k: lane (c, q) gets k = 8 q .. 8 q + 7 of index 16 i + c */
__device__ __forceinline__ k3v8bf ln_frag_t(const uint8_t *tile, int i)
{
    const int lane = threadIdx.x & 63, k = 8 * (lane >> 4) + ((lane & 15) >> 2), at = 32 * i + 8 * (lane & 3);
    const gm_v2u lo = ln_read_tr(tile + 256 * k + (at ^ (32 * ln_swap(k))));
    const gm_v2u hi = ln_read_tr(tile + 256 * (k + 4) + (at ^ (32 * ln_swap(k + 4))));
    return __builtin_bit_cast(k3v8bf, gm_v4u{lo.x, lo.y, hi.x, hi.y});
}

__device__ __forceinline__ k3v8bf ln_frag_k(const uint8_t *tile, int i)
{
    const int lane = threadIdx.x & 63;
    return __builtin_bit_cast(k3v8bf, *(const gm_v4u *)(tile + ln_krow(16 * i + (lane & 15), lane >> 4)));
}

/* ---- any types, widths and addresses: 128 x 128 outputs a workgroup, 32 k at a time. Units come to
 * registers a step ahead, and are split into their pieces on the way to LDS, once a workgroup. ---- */
#define LN_PLANE 8192                  /* 128 x 32 bf16 */

template <int MODE, bool GATED, typename TA, typename TB, typename Y>
__global__ void __launch_bounds__(256, 2)
k_ln_any(const LnArgs g)
{
    constexpr int PA = ln_pieces<TA>, PB = ln_pieces<TB>;
    constexpr int STAGE = (PA + PB) * LN_PLANE, OUT = 4 * 16 * 68 * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[STAGE > OUT ? STAGE : OUT];
    constexpr int FA = GATED ? 64 : 128;               /* outputs a of a tile */
    LnTile t;
    if (!ln_tile<MODE, FA, 128>(g, t)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = gm_uniform(tid >> 6), wa = wave & 1, wb = wave >> 1;
    const TA *a1 = (const TA *)g.a, *a3 = (const TA *)g.a3;
    Y *out = (Y *)g.y;
    if constexpr (MODE == LN_GRAD_W) {
        if (g.off) out = (Y *)gm_uniform_ptr(*(uint8_t *const *)(g.y + (size_t)t.e * g.dstep));
        if (!out || (g.accumulate && !t.np)) return;
    } else {
        a1 = (const TA *)ln_matrix(g, g.a, t.e);
        if (g.a3) a3 = (const TA *)ln_matrix(g, g.a3, t.e);
        if (!a1 || (g.a3 && !a3)) {
            ln_zeros<MODE, GATED, Y, 256>(g, out, t.p0, t.np, t.a0, FA);
            return;
        }
    }
    const int K = MODE == LN_GRAD_W ? t.np : g.K, nk = (K + 31) / 32;
    const int steps = MODE == LN_GRAD_X && g.a3 ? 2 * nk : nk;
    /* unit j of this thread: row and 16-byte slot of the tile, as it lies in memory */
    int ra[2], ua[2], rb[2], ub[2], xrow[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int id = tid + 256 * j;
        ra[j] = MODE == LN_FWD ? id >> 2 : id >> 4;
        ua[j] = MODE == LN_FWD ? id & 3 : id & 15;
        rb[j] = MODE == LN_GRAD_W ? id >> 4 : id >> 2;
        ub[j] = MODE == LN_GRAD_W ? id & 15 : id & 3;
        xrow[j] = -1;
        if (MODE == LN_FWD && rb[j] < t.np) xrow[j] = ln_row(g, t.p0 + rb[j]);
        if (MODE == LN_GRAD_X && rb[j] < t.np) xrow[j] = t.p0 + rb[j];
    }
    LnUnit<TA> va[2];
    LnUnit<TB> vb[2];
    auto fetch = [&](int s) {
        const bool second = MODE == LN_GRAD_X && s >= nk;
        const int k0 = 32 * (second ? s - nk : s);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const TA *p = a1;
            int n = 0;
            if constexpr (MODE == LN_FWD) {
                const int blk = ra[j] >> 4, f = t.a0 + (GATED ? 16 * (blk >> 1) + (ra[j] & 15) : ra[j]);
                const int k = k0 + 8 * ua[j];
                if (f < g.NA && k < K) {
                    p = (GATED && (blk & 1) ? a3 : a1) + (size_t)f * K + k;
                    n = K - k;
                }
            } else {
                const int k = k0 + ra[j], col = t.a0 + 8 * ua[j];
                const int row = k >= K ? -1 : MODE == LN_GRAD_W ? ln_row(g, t.p0 + k) : k;
                if (row >= 0 && col < g.NA) {
                    p = (second ? a3 : a1) + (size_t)row * g.NA + col;
                    n = g.NA - col;
                }
            }
            va[j] = ln_unit(p, n);
            const TB *b = (const TB *)(second ? g.b3 : g.b);
            n = 0;
            if constexpr (MODE == LN_GRAD_W) {
                const int k = k0 + rb[j], col = t.b0 + 8 * ub[j];
                if (k < K && col < g.NB) {
                    b += (size_t)(t.p0 + k) * g.NB + col;
                    n = g.NB - col;
                }
            } else {
                const int k = k0 + 8 * ub[j];
                if (xrow[j] >= 0 && k < K) {
                    b += (size_t)xrow[j] * K + k;
                    n = K - k;
                }
            }
            vb[j] = ln_unit(b, n);
        }
    };
    k3v4f acc[4][4], sums[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sums[i] = k3v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = k3v4f{0.f, 0.f, 0.f, 0.f};
    }
    const bool bias = MODE == LN_GRAD_W && g.dbias && t.a0 == 0 && wa == 0;
    if (steps) fetch(0);
    for (int s = 0; s < steps; ++s) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            gm_v4u pa[PA], pb[PB];
            ln_split(va[j], pa);
            ln_split(vb[j], pb);
            const int oa = MODE == LN_FWD ? ln_krow(ra[j], ua[j]) : 256 * ra[j] + ((16 * ua[j]) ^ (32 * ln_swap(ra[j])));
            const int ob = MODE == LN_GRAD_W ? 256 * rb[j] + ((16 * ub[j]) ^ (32 * ln_swap(rb[j]))) : ln_krow(rb[j], ub[j]);
#pragma unroll
            for (int i = 0; i < PA; ++i) *(gm_v4u *)(lds + i * LN_PLANE + oa) = pa[i];
#pragma unroll
            for (int i = 0; i < PB; ++i) *(gm_v4u *)(lds + (PA + i) * LN_PLANE + ob) = pb[i];
        }
        __syncthreads();
        if (s + 1 < steps) fetch(s + 1);
        k3v8bf fb[4][PB];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < PB; ++i) {
                const uint8_t *tile = lds + (PA + i) * LN_PLANE;
                fb[j][i] = MODE == LN_GRAD_W ? ln_frag_t(tile, 4 * wb + j) : ln_frag_k(tile, 4 * wb + j);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k3v8bf fa[PA];
#pragma unroll
            for (int p = 0; p < PA; ++p)
                fa[p] = MODE == LN_FWD ? ln_frag_k(lds + p * LN_PLANE, 4 * wa + i) : ln_frag_t(lds + p * LN_PLANE, 4 * wa + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) ln_mma<PA, PB>(fa, fb[j], acc[i][j]);
        }
        if (bias) {
            k3v8bf one[1];
            one[0] = __builtin_bit_cast(k3v8bf, gm_v4u{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
#pragma unroll
            for (int j = 0; j < 4; ++j) ln_mma<1, PB>(one, fb[j], sums[j]);
        }
    }
    __syncthreads();
    if (bias && lane < 16) {
        /* every row of the product with ones is the sums; lane c holds those of index c */
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = t.b0 + 64 * wb + 16 * j + lane;
            if (b >= g.NB) continue;
            float *o = g.dbias + (size_t)t.e * g.NB + b;
            *o = g.accumulate ? *o + sums[j][0] : sums[j][0];
        }
    }
    const int valid = MODE == LN_GRAD_W ? g.NB - t.b0 : t.np;
    ln_out<MODE, GATED, Y, 4, 4>(g, (float *)lds + wave * 16 * 68, acc, out, t.e,
                                 (size_t)(MODE == LN_GRAD_W ? t.b0 : t.p0) + 64 * wb, valid - 64 * wb,
                                 t.a0 + FA / 2 * wa);
}

/* ---------------------------------------------------- through the activation alone ---- */

template <typename T>
__global__ void __launch_bounds__(256)
k_ln_act_grad(const T *dh, const T *z, const T *z3, T *dz, T *dz3, size_t n, int act, float b1, float b2, float i1,
              float i2)
{
    for (size_t i = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x); i < n; i += 4 * (size_t)gridDim.x * 256) {
        const int m = (int)min(n - i, (size_t)4);
        k3v4f d = ln_get4(dh + i, m);
        const k3v4f v = ln_get4(z + i, m);
        if (z3) {
            const k3v4f u = ln_get4(z3 + i, m);
            k3v4f d3;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float dg, du;
                ka_situ_slopes(v[j], u[j], b1, b2, i1, i2, dg, du);
                d3[j] = d[j] * du;
                d[j] *= dg;
            }
            ln_put4(dz3 + i, m, d3);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] *= ka_slope(act, v[j]);
        }
        ln_put4(dz + i, m, d);
    }
}

/* ------------------------------------------------------------- entry points ---- */

static int ln_type(const char *who, const char *name, int dt)
{
    if (dt == K3_WF32 || dt == K3_WBF16) return 0;
    fprintf(stderr, "%s: %s is fp32 (%d) or bf16 (%d), not %d\n", who, name, K3_WF32, K3_WBF16, dt);
    return -1;
}

static int ln_pointer(const char *who, const char *name, const void *p, int to, bool needed)
{
    if ((p || !needed) && !k3h_misaligned(p, to)) return 0;
    fprintf(stderr, "%s: %s is missing or not aligned to %d bytes\n", who, name, to);
    return -1;
}

static int ln_size(int dt) { return dt == K3_WBF16 ? 2 : 4; }

static int ln_shape(const char *who, int rows, int cols, int n)
{
    if (rows >= 0 && rows <= LN_MAX_ROWS && cols >= 1 && cols <= LN_MAX_WIDTH && n >= 1 && n <= LN_MAX_WIDTH) return 0;
    fprintf(stderr, "%s: needs 0 to %d rows and widths from 1 to %d (%d rows, %d columns, %d features)\n", who,
            LN_MAX_ROWS, LN_MAX_WIDTH, rows, cols, n);
    return -1;
}

/* the activation of one product, or of two (pair) */
static int ln_activation(const char *who, int act, float b1, float b2, bool pair)
{
    if (act < K3G_ACT_NONE || act > K3G_ACT_SITU) {
        fprintf(stderr, "%s: no activation %d\n", who, act);
        return -1;
    }
    if ((act == K3G_ACT_SITU) != pair) {
        fprintf(stderr, "%s: the gated activation (%d) takes two products, the others one (%d)\n", who, K3G_ACT_SITU, act);
        return -1;
    }
    /* below, a cap's reciprocal may be infinite */
    if (pair && !(b1 >= 0x1p-100f && b2 >= 0x1p-100f)) {
        fprintf(stderr, "%s: the activation's caps are 2^-100 or more (%g, %g)\n", who, b1, b2);
        return -1;
    }
    return 0;
}

static void ln_caps(LnArgs &g, int act, float b1, float b2)
{
    g.act = act;
    g.b1 = b1;
    g.b2 = b2;
    g.i1 = 1.0f / b1;
    g.i2 = 1.0f / b2;
}

/* the sorted rows of experts: how many there may be, and where each one's row of x is */
static int ln_groups(const char *who, LnArgs &g, int rows, const int32_t *perm, int topk, const int32_t *off, int E,
                     int step, const char *table)
{
    if (E < 1 || E > GM_MAX_EXPERTS || topk < 1 || topk > K3G_MAX_TOPK || (!perm && topk != 1) ||
        (int64_t)rows * topk > LN_MAX_ROWS) {
        fprintf(stderr, "%s: needs 1 to %d experts, 1 <= topk <= %d (1 without perm) and at most %d pairs (%d "
                        "experts, %d x %d)\n", who, GM_MAX_EXPERTS, K3G_MAX_TOPK, LN_MAX_ROWS, E, rows, topk);
        return -1;
    }
    if (step < 8 || step % 8) {
        fprintf(stderr, "%s: %s is a multiple of 8 bytes (%d)\n", who, table, step);
        return -1;
    }
    /* pair / topk is the upper half of pair * ceil(2^32 / topk) for pairs below 2^32 / topk */
    g.perm = perm;
    g.magic = topk > 1 ? (uint32_t)((((uint64_t)1 << 32) + topk - 1) / topk) : 0;
    g.pairs = g.P = rows * topk;
    g.off = off;
    g.E = E;
    return 0;
}

template <int MODE, bool GATED, typename TA, typename TB, typename Y>
static int ln_run(const char *who, const LnArgs &g, hipStream_t st)
{
    const int64_t na = (g.NA + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
    const int64_t blocks = MODE == LN_GRAD_W ? 8 * (int64_t)g.E * ((na * ((g.NB + 127) / 128) + 7) / 8)
                                             : gm_row_items(g.off != nullptr, g.E, g.P, 128, na);
    if (blocks * 256 > UINT32_MAX) {
        fprintf(stderr, "%s: %d rows by %d columns (%d experts) are more than a launch takes\n", who,
                MODE == LN_GRAD_W ? g.NB : g.P, g.NA, g.E);
        return -1;
    }
    return k3h_launch(who, k_ln_any<MODE, GATED, TA, TB, Y>, dim3((unsigned)blocks), dim3(256), st, (LnArgs)g);
}

template <int MODE, bool GATED, typename TA, typename TB>
static int ln_run_y(const char *who, const LnArgs &g, int ydt, hipStream_t st)
{
    return ydt == K3_WBF16 ? ln_run<MODE, GATED, TA, TB, uint16_t>(who, g, st)
                           : ln_run<MODE, GATED, TA, TB, float>(who, g, st);
}

template <int MODE, bool GATED>
static int ln_product(const char *who, const LnArgs &g, int adt, int bdt, int ydt, void *stream)
{
    K3hOn on(stream);
    if (!on.ok) return -1;
    if (adt == K3_WBF16)
        return bdt == K3_WBF16 ? ln_run_y<MODE, GATED, uint16_t, uint16_t>(who, g, ydt, on.st)
                               : ln_run_y<MODE, GATED, uint16_t, float>(who, g, ydt, on.st);
    return bdt == K3_WBF16 ? ln_run_y<MODE, GATED, float, uint16_t>(who, g, ydt, on.st)
                           : ln_run_y<MODE, GATED, float, float>(who, g, ydt, on.st);
}

/* forward: x, the matrix operand and what follows are checked, g has the groups */
static int ln_forward(const char *who, LnArgs &g, const void *x, int xdt, int rows, int cols, const void *w,
                      const void *w3, int wdt, int to, int n, const K3gEpilogue *ep, void *y, int ydt, void *stream)
{
    static const K3gEpilogue none = {};
    if (!ep) ep = &none;
    const bool pair = w3 != nullptr, some = rows > 0;
    if (ln_type(who, "x", xdt) || ln_type(who, "w", wdt) || ln_type(who, "y", ydt) || ln_shape(who, rows, cols, n) ||
        ln_activation(who, ep->act, ep->b1, ep->b2, pair) || ln_pointer(who, "x", x, ln_size(xdt), some) ||
        ln_pointer(who, "w", w, to, some) || ln_pointer(who, "w3", w3, to, false) ||
        ln_pointer(who, "y", y, ln_size(ydt), some) || ln_pointer(who, "bias", ep->bias, 4, false) ||
        ln_pointer(who, "bias3", ep->bias3, 4, false) || ln_pointer(who, "residual", ep->residual, ln_size(ydt), false) ||
        ln_pointer(who, "z", ep->z, ln_size(ydt), false) || ln_pointer(who, "z3", ep->z3, ln_size(ydt), false))
        return -1;
    if (!pair && (ep->bias3 || ep->z3)) {
        fprintf(stderr, "%s: bias3 and z3 belong to a second matrix\n", who);
        return -1;
    }
    if (!rows) return 0;
    g.a = (const uint8_t *)w;
    g.a3 = (const uint8_t *)w3;
    g.b = (const uint8_t *)x;
    g.NA = n;
    g.K = cols;
    g.y = (uint8_t *)y;
    ln_caps(g, ep->act, ep->b1, ep->b2);
    g.bias = ep->bias;
    g.bias3 = ep->bias3;
    g.add = (const uint8_t *)ep->residual;
    g.z = (uint8_t *)ep->z;
    g.z3 = (uint8_t *)ep->z3;
    return pair ? ln_product<LN_FWD, true>(who, g, wdt, xdt, ydt, stream)
                : ln_product<LN_FWD, false>(who, g, wdt, xdt, ydt, stream);
}

extern "C" int k3g_matmul(const void *x, int xdt, int rows, int cols, const void *w, const void *w3, int wdt, int n,
                          const K3gEpilogue *ep, void *y, int ydt, void *stream)
{
    LnArgs g = {};
    g.pairs = g.P = rows;
    g.E = 1;
    return ln_forward("k3g_matmul", g, x, xdt, rows, cols, w, w3, wdt, ln_size(wdt), n, ep, y, ydt, stream);
}

extern "C" int k3g_grouped(const void *x, int xdt, int rows, int cols, const int32_t *perm, int topk,
                           const int32_t *off, int n_experts, const void *const *w, const void *const *w3, int w_step,
                           int wdt, int n, const K3gEpilogue *ep, void *y, int ydt, void *stream)
{
    const char *who = "k3g_grouped";
    LnArgs g = {};
    if (ln_shape(who, rows, cols, n) || ln_pointer(who, "off", off, 4, rows > 0) ||
        ln_pointer(who, "perm", perm, 4, false) || ln_groups(who, g, rows, perm, topk, off, n_experts, w_step, "w_step"))
        return -1;
    g.step = w_step;
    return ln_forward(who, g, x, xdt, rows, cols, w, w3, wdt, 8, n, ep, y, ydt, stream);
}

static int ln_back_x(const char *who, LnArgs &g, const void *dy, const void *dy3, int dydt, int rows, int n,
                     const void *w, const void *w3, int wdt, int to, int cols, const K3gBack *back, void *dx, int dxdt,
                     void *stream)
{
    static const K3gBack none = {};
    if (!back) back = &none;
    const bool some = rows > 0;
    if (ln_type(who, "dy", dydt) || ln_type(who, "w", wdt) || ln_type(who, "dx", dxdt) ||
        ln_shape(who, rows, cols, n) || ln_pointer(who, "dy", dy, ln_size(dydt), some) ||
        ln_pointer(who, "dy3", dy3, ln_size(dydt), false) || ln_pointer(who, "w", w, to, some) ||
        ln_pointer(who, "w3", w3, to, false) || ln_pointer(who, "dx", dx, ln_size(dxdt), some) ||
        ln_pointer(who, "add", back->add, ln_size(dxdt), false) || ln_pointer(who, "z", back->z, ln_size(dxdt), false) ||
        ln_pointer(who, "z3", back->z3, ln_size(dxdt), false) || ln_pointer(who, "dz3", back->dz3, ln_size(dxdt), false))
        return -1;
    if (!dy3 != !w3) {
        fprintf(stderr, "%s: dy3 and w3 belong together\n", who);
        return -1;
    }
    if (!back->z3 != !back->dz3 || (back->z3 && !back->z)) {
        fprintf(stderr, "%s: z3 and dz3 belong together, and to z\n", who);
        return -1;
    }
    if (back->z ? ln_activation(who, back->act, back->b1, back->b2, back->z3 != nullptr) : back->act != K3G_ACT_NONE) {
        if (!back->z) fprintf(stderr, "%s: z is missing for activation %d\n", who, back->act);
        return -1;
    }
    if (!rows) return 0;
    g.a = (const uint8_t *)w;
    g.a3 = (const uint8_t *)w3;
    g.b = (const uint8_t *)dy;
    g.b3 = (const uint8_t *)dy3;
    g.NA = cols;
    g.K = n;
    g.y = (uint8_t *)dx;
    ln_caps(g, back->act, back->b1, back->b2);
    g.add = (const uint8_t *)back->add;
    g.z = (uint8_t *)back->z;
    g.z3 = (uint8_t *)back->z3;
    g.dz3 = (uint8_t *)back->dz3;
    return ln_product<LN_GRAD_X, false>(who, g, wdt, dydt, dxdt, stream);
}

extern "C" int k3g_matmul_grad_x(const void *dy, const void *dy3, int dydt, int rows, int n, const void *w,
                                 const void *w3, int wdt, int cols, const K3gBack *back, void *dx, int dxdt,
                                 void *stream)
{
    LnArgs g = {};
    g.P = rows;
    g.E = 1;
    return ln_back_x("k3g_matmul_grad_x", g, dy, dy3, dydt, rows, n, w, w3, wdt, ln_size(wdt), cols, back, dx, dxdt,
                     stream);
}

extern "C" int k3g_grouped_grad_x(const void *dy, const void *dy3, int dydt, int rows, int n, const int32_t *off,
                                  int n_experts, const void *const *w, const void *const *w3, int w_step, int wdt,
                                  int cols, const K3gBack *back, void *dx, int dxdt, void *stream)
{
    const char *who = "k3g_grouped_grad_x";
    LnArgs g = {};
    if (ln_shape(who, rows, cols, n) || ln_pointer(who, "off", off, 4, rows > 0) ||
        ln_groups(who, g, rows, nullptr, 1, off, n_experts, w_step, "w_step"))
        return -1;
    g.step = w_step;
    return ln_back_x(who, g, dy, dy3, dydt, rows, n, w, w3, wdt, 8, cols, back, dx, dxdt, stream);
}

static int ln_back_w(const char *who, LnArgs &g, const void *dy, int dydt, const void *x, int xdt, int rows, int n,
                     int cols, int accumulate, void *dw, int dwdt, int to, float *dbias, void *stream)
{
    if (ln_type(who, "dy", dydt) || ln_type(who, "x", xdt) || ln_type(who, "dw", dwdt) ||
        ln_shape(who, rows, cols, n) || ln_pointer(who, "dy", dy, ln_size(dydt), rows > 0) ||
        ln_pointer(who, "x", x, ln_size(xdt), rows > 0) || ln_pointer(who, "dw", dw, to, true) ||
        ln_pointer(who, "dbias", dbias, 4, false))
        return -1;
    if (!rows && accumulate) return 0;
    g.a = (const uint8_t *)x;
    g.b = (const uint8_t *)dy;
    g.NA = cols;
    g.NB = n;
    g.y = (uint8_t *)dw;
    g.accumulate = accumulate;
    g.dbias = dbias;
    return ln_product<LN_GRAD_W, false>(who, g, xdt, dydt, dwdt, stream);
}

extern "C" int k3g_matmul_grad_w(const void *dy, int dydt, const void *x, int xdt, int rows, int n, int cols,
                                 int accumulate, void *dw, int dwdt, float *dbias, void *stream)
{
    LnArgs g = {};
    g.pairs = g.P = rows;
    g.E = 1;
    return ln_back_w("k3g_matmul_grad_w", g, dy, dydt, x, xdt, rows, n, cols, accumulate, dw, dwdt, ln_size(dwdt),
                     dbias, stream);
}

extern "C" int k3g_grouped_grad_w(const void *dy, int dydt, const void *x, int xdt, int rows, int n, int cols,
                                  const int32_t *perm, int topk, const int32_t *off, int n_experts, int accumulate,
                                  void *const *dw, int dw_step, int dwdt, float *dbias, void *stream)
{
    const char *who = "k3g_grouped_grad_w";
    LnArgs g = {};
    if (ln_shape(who, rows, cols, n) || ln_pointer(who, "off", off, 4, true) ||
        ln_pointer(who, "perm", perm, 4, false) || ln_groups(who, g, rows, perm, topk, off, n_experts, dw_step, "dw_step"))
        return -1;
    g.dstep = dw_step;
    return ln_back_w(who, g, dy, dydt, x, xdt, rows, n, cols, accumulate, (void *)dw, dwdt, 8, dbias, stream);
}

extern "C" int k3g_act_grad(const void *dh, int dt, int rows, int n, int act, float b1, float b2, const void *z,
                            const void *z3, void *dz, void *dz3, void *stream)
{
    const char *who = "k3g_act_grad";
    if (ln_type(who, "dh", dt)) return -1;
    if (rows < 0 || rows > 1 << 26 || n < 1 || n > 1 << 24) {
        fprintf(stderr, "%s: needs 0 to %d rows of 1 to %d values (%d of %d)\n", who, 1 << 26, 1 << 24, rows, n);
        return -1;
    }
    const bool some = rows > 0;
    if (ln_activation(who, act, b1, b2, act == K3G_ACT_SITU) || ln_pointer(who, "dh", dh, ln_size(dt), some) ||
        ln_pointer(who, "z", z, ln_size(dt), some) || ln_pointer(who, "dz", dz, ln_size(dt), some) ||
        ln_pointer(who, "z3", z3, ln_size(dt), some && act == K3G_ACT_SITU) ||
        ln_pointer(who, "dz3", dz3, ln_size(dt), some && act == K3G_ACT_SITU))
        return -1;
    if (act != K3G_ACT_SITU && (z3 || dz3)) {
        fprintf(stderr, "%s: z3 and dz3 belong to the gated activation\n", who);
        return -1;
    }
    if (some && dz == dz3) {
        fprintf(stderr, "%s: dz and dz3 are the same\n", who);
        return -1;
    }
    if (!some) return 0;
    K3hOn on(stream);
    if (!on.ok) return -1;
    const size_t count = (size_t)rows * n;
    const dim3 grid((unsigned)min((count + 1023) / 1024, (size_t)1 << 16));
    const float i1 = 1.0f / b1, i2 = 1.0f / b2;
    if (dt == K3_WBF16)
        return k3h_launch(who, k_ln_act_grad<uint16_t>, grid, dim3(256), on.st, (const uint16_t *)dh,
                          (const uint16_t *)z, (const uint16_t *)z3, (uint16_t *)dz, (uint16_t *)dz3, count, act, b1, b2,
                          i1, i2);
    return k3h_launch(who, k_ln_act_grad<float>, grid, dim3(256), on.st, (const float *)dh, (const float *)z,
                      (const float *)z3, (float *)dz, (float *)dz3, count, act, b1, b2, i1, i2);
}
