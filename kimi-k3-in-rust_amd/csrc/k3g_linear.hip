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
#include <math.h>
#include <stdio.h>

#include <utility>

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
    int T, pairs;                    /* rows of x, and their pairs */
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
    bool stream;                     /* results are more than the last-level cache holds */
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

/* four values as they lie, n of them there */
template <typename T> struct LnRaw;
template <> struct LnRaw<float> { gm_v4u v; };
template <> struct LnRaw<uint16_t> { gm_v2u v; };

__device__ __forceinline__ LnRaw<float> ln_raw4(const float *p, int n)
{
    const LN_G(uint32_t) *g = (const LN_G(uint32_t) *)p;
    if (n >= 4) return {*(const LN_G(ln_any16) *)g};
    return {gm_v4u{g[0], n > 1 ? g[1] : 0u, n > 2 ? g[2] : 0u, 0u}};
}

__device__ __forceinline__ LnRaw<uint16_t> ln_raw4(const uint16_t *p, int n)
{
    const LN_G(uint16_t) *g = (const LN_G(uint16_t) *)p;
    if (n >= 4) return {*(const LN_G(ln_any8) *)g};
    return {gm_v2u{g[0] | (n > 1 ? (uint32_t)g[1] << 16 : 0u), n > 2 ? g[2] : 0u}};
}

__device__ __forceinline__ k3v4f ln_values(const LnRaw<float> &r) { return __builtin_bit_cast(k3v4f, r.v); }
__device__ __forceinline__ k3v4f ln_values(const LnRaw<uint16_t> &r)
{
    return k3v4f{k3d_bf16lo(r.v.x), k3d_bf16hi(r.v.x), k3d_bf16lo(r.v.y), k3d_bf16hi(r.v.y)};
}

template <typename T>
__device__ __forceinline__ k3v4f ln_get4(const T *p, int n) { return ln_values(ln_raw4(p, n)); }

/* n of four values. stream: past the caches, for results that are more than the last-level cache's
 * 256 MB (LN_STREAM; gradients of 64 matrices 1408 x 2048 in fp32, 738 MB: 365 -> 268 us). Smaller
 * ones stay for whoever reads them next: rows of 4096 x 7168 in bf16 are 138 us either way, and what
 * reads them then 20 us, or 33 where they went past. */
#define LN_STREAM ((size_t)256 << 20)

__device__ __forceinline__ void ln_put4(float *p, int n, const k3v4f &v, bool stream)
{
    LN_G(float) *g = (LN_G(float) *)p;
    if (n >= 4) {
        const gm_v4u u = __builtin_bit_cast(gm_v4u, v);
        if (stream) __builtin_nontemporal_store(u, (LN_G(ln_any16) *)g);
        else *(LN_G(ln_any16) *)g = u;
        return;
    }
    g[0] = v[0];
    if (n > 1) g[1] = v[1];
    if (n > 2) g[2] = v[2];
}

__device__ __forceinline__ void ln_put4(uint16_t *p, int n, const k3v4f &v, bool stream)
{
    LN_G(uint16_t) *g = (LN_G(uint16_t) *)p;
    const gm_v2u u = {k3d_bf16x2(v[0], v[1]), k3d_bf16x2(v[2], v[3])};
    if (n >= 4) {
        if (stream) __builtin_nontemporal_store(u, (LN_G(ln_any8) *)g);
        else *(LN_G(ln_any8) *)g = u;
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

/* What the epilogue reads of an output's four values: what is added to them, and the values before
 * the activation. */
template <int MODE, typename Y>
struct LnRead {
    LnRaw<Y> add, z[MODE == LN_GRAD_X ? 2 : 1];
};

template <int MODE, typename Y>
__device__ __forceinline__ void ln_ask(const LnArgs &g, const Y *out, size_t at, int n, LnRead<MODE, Y> &r)
{
    const Y *add = MODE == LN_GRAD_W ? (g.accumulate ? out : nullptr) : (const Y *)g.add;
    if (add) r.add = ln_raw4(add + at, n);
    if (MODE == LN_GRAD_X && g.z) r.z[0] = ln_raw4((const Y *)g.z + at, n);
    if (MODE == LN_GRAD_X && g.dz3) r.z[MODE == LN_GRAD_X] = ln_raw4((const Y *)g.z3 + at, n);
}

/* What follows four consecutive sums v (and u, of the second matrix; b and b3 their biases): n of
 * them are stored at `at`. */
template <int MODE, bool GATED, typename Y>
__device__ __forceinline__ void ln_finish(const LnArgs &g, Y *out, size_t at, int n, k3v4f v, k3v4f u, const k3v4f &b,
                                          const k3v4f &b3, const LnRead<MODE, Y> &r)
{
    if constexpr (MODE == LN_FWD) {
        v += b;
        if (g.z) ln_put4((Y *)g.z + at, n, v, g.stream);
        if (GATED) {
            u += b3;
            if (g.z3) ln_put4((Y *)g.z3 + at, n, u, g.stream);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = GATED ? ka_situ(v[i], u[i], g.b1, g.b2, g.i1, g.i2) : ka_act(g.act, v[i]);
        if (g.add) v += ln_values(r.add);
    } else if constexpr (MODE == LN_GRAD_X) {
        if (g.add) v += ln_values(r.add);
        if (g.dz3) {
            const k3v4f z = ln_values(r.z[0]), z3 = ln_values(r.z[1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float dg, du;
                ka_situ_slopes(z[i], z3[i], g.b1, g.b2, g.i1, g.i2, dg, du);
                u[i] = v[i] * du;
                v[i] *= dg;
            }
            ln_put4((Y *)g.dz3 + at, n, u, g.stream);
        } else if (g.z) {
            const k3v4f z = ln_values(r.z[0]);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] *= ka_slope(g.act, z[i]);
        }
    } else {
        if (g.accumulate) v += ln_values(r.add);
    }
    ln_put4(out + at, n, v, g.stream);
}

/* A wave's sums (MA x MB blocks of 16 a x 16 b) out by way of LDS (16 x (16 MA + 4) floats of its
 * own), so that it reads and writes whole pieces of rows: rows row0 + 0 .. rows - 1, columns col0 on.
 * GATED: the blocks are the two matrices' in turn. Everything that 16 rows read from memory is asked
 * for in one or two goes, the first before their sums go to LDS (one piece of a row at a time, a residual of 4096 x 7168
 * took 50 of 248 us). */
template <int MODE, bool GATED, typename Y, int MA, int MB>
__device__ __forceinline__ void ln_out(const LnArgs &g, float *lds, const k3v4f (&acc)[MA][MB], Y *out, int e,
                                       size_t row0, int rows, int col0)
{
    constexpr int PITCH = 16 * MA + 4, LANES = (GATED ? 2 : 4) * MA, STEP = 64 / LANES, PASSES = 16 / STEP;
    constexpr int CHUNK = MODE == LN_GRAD_X && PASSES > 4 ? 4 : PASSES;       /* as registers allow */
    const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const int f = 4 * (lane % LANES), from = GATED ? 32 * (f >> 4) + (f & 15) : f, a = col0 + f, n = min(4, g.NA - a);
    k3v4f b = {0.f, 0.f, 0.f, 0.f}, b3 = b;
    if (n <= 0) rows = 0;
    if (MODE == LN_FWD && g.bias && n > 0) b = ln_get4(g.bias + (size_t)e * g.NA + a, n);
    if (MODE == LN_FWD && GATED && g.bias3 && n > 0) b3 = ln_get4(g.bias3 + (size_t)e * g.NA + a, n);
#pragma unroll 1
    for (int j = 0; j < MB; ++j) {
        const int r0 = 16 * j + lane / LANES;
        const size_t at = (row0 + r0) * g.NA + a;
#pragma unroll
        for (int p0 = 0; p0 < PASSES; p0 += CHUNK) {
            LnRead<MODE, Y> read[CHUNK];
#pragma unroll
            for (int p = 0; p < CHUNK; ++p)
                if (r0 + STEP * (p0 + p) < rows)
                    ln_ask<MODE, Y>(g, out, at + (size_t)(STEP * (p0 + p)) * g.NA, n, read[p]);
            if (!p0) {
                gm_wave_sync();
#pragma unroll
                for (int k = 0; k < MB; ++k) {
                    if (k != j) continue;      /* what follows is in the code once, not MB times */
#pragma unroll
                    for (int i = 0; i < MA; ++i) *(k3v4f *)(lds + c * PITCH + 16 * i + 4 * q) = acc[i][k];
                }
                gm_wave_sync();
            }
#pragma unroll
            for (int p = 0; p < CHUNK; ++p) {
                if (r0 + STEP * (p0 + p) >= rows) continue;
                const float *o = lds + (lane / LANES + STEP * (p0 + p)) * PITCH + from;
                const k3v4f v = *(const k3v4f *)o, u = GATED ? *(const k3v4f *)(o + 16) : k3v4f{0.f, 0.f, 0.f, 0.f};
                ln_finish<MODE, GATED, Y>(g, out, at + (size_t)(STEP * (p0 + p)) * g.NA, n, v, u, b, b3, read[p]);
            }
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

/* ---- bf16 rows and matrices whose widths are multiples of 8: BA x BB outputs by four waves, a
 * quarter each, 64 k at a time. The tiles come to LDS by DMA, two stages; an operand's fragments of
 * the next 32 k are read while the products of these 32 run, across the stages too, so a step has one
 * barrier, in its middle: before it every wave has read the last of this stage (into which the
 * copies for the step after the next then go) and its own copies of the next stage have arrived.
 *
 * Rows of contiguous k are 128 bytes of LDS, unit u of row r at slot u ^ (r % 8); rows k of
 * contiguous a or b as in the tiles of 32 k above, 64 of them. */
/* The 1 KB copies of an operand's stage by WV waves, WV i + wave the one of this wave: which row (TR: k) of the
 * tile this lane copies 16 bytes of, and which unit of it */
template <bool TR, int B, int WV>
__device__ __forceinline__ int ln_copy_row(int i, int lane, int wave)
{
    constexpr int UNITS = TR ? B / 8 : 8;
    return (64 / UNITS) * (WV * i + wave) + lane / UNITS;
}

template <bool TR, int B, int WV>
__device__ __forceinline__ int ln_copy_unit(int i, int lane, int wave)
{
    if (!TR) return (lane & 7) ^ (lane >> 3);
    return (lane % (B / 8)) ^ (2 * ln_swap(ln_copy_row<TR, B, WV>(i, lane, wave)));
}

/* block i's operand of k 32 kh .. 32 kh + 31 */
template <bool TR, int B>
__device__ __forceinline__ k3v8bf ln_frag(const uint8_t *tile, int kh, int i)
{
    const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    if constexpr (TR) {
        const int k = 32 * kh + 8 * q + (c >> 2), at = 32 * i + 8 * (c & 3);
        const gm_v2u lo = ln_read_tr(tile + 2 * B * k + (at ^ (32 * ln_swap(k))));
        const gm_v2u hi = ln_read_tr(tile + 2 * B * (k + 4) + (at ^ (32 * ln_swap(k + 4))));
        return __builtin_bit_cast(k3v8bf, gm_v4u{lo.x, lo.y, hi.x, hi.y});
    } else {
        return __builtin_bit_cast(k3v8bf, *(const gm_v4u *)(tile + 128 * (16 * i + c) + 16 * ((4 * kh + q) ^ (c & 7))));
    }
}

/* f(0) ... f(N - 1), each with its number as a constant */
template <typename F, int... I>
__device__ __forceinline__ void ln_each(F f, std::integer_sequence<int, I...>)
{
    (f(GmInt<I>{}), ...);
}

/* A copy in two instructions with whatever stands between them: where in LDS it goes, then the 64
 * lanes x 16 bytes from base + at. M0 is not put back: nothing else in these kernels uses it (the
 * compiler keeps no value in it, and of the instructions that read it none is here). */
template <int MORE>
__device__ __forceinline__ void ln_dma_at(uint32_t lds)
{
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0" : : "s"(lds), "i"(MORE) : "scc", "memory");
}
__device__ __forceinline__ void ln_dma(const uint8_t *base, uint32_t at)
{
    asm volatile("global_load_lds_dwordx4 %0, %1" : : "v"(at), "s"(base) : "memory");
}

/* acc += A B in place. BIG: sums of 128 accumulation registers a lane; the compiler, given the
 * builtin, moves a third of them about in every step, so the instruction stands here. Its operands
 * come from LDS as they are (a vector instruction that writes one needs two wait states before it: the
 * compiler puts none in front of assembly), and whoever reads the sums waits first: ln_settle. */
template <bool BIG>
__device__ __forceinline__ void ln_mfma(const k3v8bf &a, const k3v8bf &b, k3v4f &acc)
{
    if constexpr (BIG)
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
    else acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}

/* the same with sums in general registers and an operand that is made in registers */
template <bool BIG>
__device__ __forceinline__ void ln_mfma_v(const k3v8bf &a, const k3v8bf &b, k3v4f &acc)
{
    if constexpr (BIG)
        asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
    else acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}

/* every product under way has written its sums */
template <bool BIG, int N>
__device__ __forceinline__ void ln_settle(k3v4f (&acc)[N])
{
    if constexpr (BIG) {
        asm volatile("s_nop 15\n\ts_nop 15" : : : "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("" : "+a"(acc[i]));
    }
}

/* What is issued after which of the N = MA MB products of 32 k (in the order of A's blocks): reads
 * of the next fragments (a block i of A, in place, after its last product; MA + j: block j of B, to
 * the other half) and copies. An instruction of a wave takes four cycles to issue, a product sixteen:
 * one of these after a product at a time leaves the matrix cores busy, several in a row do not. */
template <int MA, int MB, int C>
struct LnPlan {
    static constexpr int N = MA * MB, BAR = MB * (MA / 4 > 1 ? MA / 4 : 1) - 1;
    static constexpr int ALL = (2 * N - 1 - BAR) / C, STRIDE = ALL < 4 ? ALL : 4;
    static constexpr int FIRST = (N - 2 - BAR) / STRIDE + 1 < C ? (N - 2 - BAR) / STRIDE + 1 : C;
    signed char read[N][2], copy[N];
    constexpr void put(int slot, int what)
    {
        while (slot < N - 1 && read[slot][0] >= 0) ++slot;
        read[slot][read[slot][0] >= 0] = (signed char)what;
    }
    /* bar: the second half, whose reads and copies come after product BAR */
    constexpr LnPlan(bool bar) : read(), copy()
    {
        for (int i = 0; i < N; ++i) read[i][0] = read[i][1] = copy[i] = -1;
        const int from = bar ? BAR + 1 : 0, room = N - from;
        for (int i = 0; i < MA; ++i) {
            const int done = MB * i + MB - 1;
            if (done >= from) put(done, i);
        }
        for (int j = 0; j < MB; ++j) put(from + j * room / (2 * MB), MA + j);
        for (int i = 0; i < MA; ++i)
            if (MB * i + MB - 1 < from) put(from + room / 2 + 2 * i, i);
        for (int c = 0; c < C; ++c)
            if ((c < FIRST) == bar) copy[bar ? from + c * STRIDE : (c - FIRST) * STRIDE + STRIDE / 2] = (signed char)c;
    }
};

template <int MODE, bool GATED, typename Y, int BA, int BB, int WV>
__global__ void __launch_bounds__(64 * WV, BA + BB > 256 && WV == 4 ? 1 : 2)
k_ln_tile(const LnArgs g)
{
    constexpr bool TA = MODE != LN_FWD, TB = MODE == LN_GRAD_W;
    constexpr int MA = BA / 32, MB = BB / (8 * WV), STAGE = 128 * (BA + BB), FA = GATED ? BA / 2 : BA;
    constexpr int CA = BA / (8 * WV), CB = BB / (8 * WV);           /* a wave's copies of a stage */
    constexpr bool BIG = MA * MB > 16;
    static_assert(WV * 16 * (16 * MA + 4) * 4 <= 2 * STAGE, "the sums' way out");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * STAGE];
    LnTile t;
    if (!ln_tile<MODE, FA, BB>(g, t)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = gm_uniform(tid >> 6), wa = wave & 1, wb = wave >> 1;
    const uint8_t *m1 = g.a, *m3 = g.a3;
    Y *out = (Y *)g.y;
    if constexpr (MODE == LN_GRAD_W) {
        if (g.off) out = (Y *)gm_uniform_ptr(*(uint8_t *const *)(g.y + (size_t)t.e * g.dstep));
        if (!out || (g.accumulate && !t.np)) return;
    } else {
        m1 = ln_matrix(g, g.a, t.e);
        if (g.a3) m3 = ln_matrix(g, g.a3, t.e);
        if (!m1 || (g.a3 && !m3)) {
            ln_zeros<MODE, GATED, Y, 64 * WV>(g, out, t.p0, t.np, t.a0, FA);
            return;
        }
    }
    const int K = MODE == LN_GRAD_W ? t.np : g.K, nk = (K + 63) / 64;
    const int steps = MODE == LN_GRAD_X && g.a3 ? 2 * nk : nk;
    /* a matrix comes by the caller's table, and the host has not seen its address: one that is not
     * aligned for DMA is copied by DMA from the 16 bytes around, and then (fix) by registers */
    const bool aligned = ((((uintptr_t)m1) | (uintptr_t)m3) & 15) == 0;
    const bool gather = MODE == LN_GRAD_W && g.perm;
    const uint32_t ldsp = (uint32_t)(uintptr_t)(k3lds)lds + 1024 * wave;

    /* What this lane copies: at oa, ob from bases that move on by a stage's k, and no further than the
     * end of the operand, so all reads are of memory that is there. Whatever of it is not of these
     * rows, columns or k gives outputs that are not stored, or is set to zero once it has arrived
     * (fix). Forward with two matrices, their blocks of 16 rows alternate in A, and all that a wave
     * copies is of one. */
    const size_t a0 = MODE == LN_FWD ? (size_t)t.a0 * K : (size_t)t.a0;
    const uint8_t *sa = MODE == LN_GRAD_W ? g.a : GATED && wave & 2 ? m3 : m1, *sb = g.b;
    const uint8_t *ea = sa + 2 * (size_t)g.NA * (MODE == LN_GRAD_W ? g.T : g.K);
    const uint8_t *eb = sb + 2 * (size_t)(MODE == LN_FWD ? g.T : g.P) * (MODE == LN_GRAD_W ? g.NB : g.K);
    sa += 2 * (MODE == LN_GRAD_W && !gather ? a0 + (size_t)t.p0 * g.NA : a0);
    if (MODE == LN_GRAD_W) sb += 2 * ((size_t)t.p0 * g.NB + t.b0);
    else if (MODE != LN_FWD || !g.perm) sb += 2 * (size_t)t.p0 * K;
    uint32_t oa[CA], ob[CB], bad = 0;          /* bit i of bad: row i of B is of no pair */
#pragma unroll
    for (int i = 0; i < CA; ++i) {
        const uint32_t r = ln_copy_row<TA, BA, WV>(i, lane, wave), u = ln_copy_unit<TA, BA, WV>(i, lane, wave);
        if (MODE == LN_FWD) oa[i] = 2 * (GATED ? 16 * (r >> 5) + (r & 15) : r) * K + 16 * u;
        else oa[i] = 2 * (gather ? 0 : r) * g.NA + 16 * u;
    }
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const uint32_t r = ln_copy_row<TB, BB, WV>(i, lane, wave), u = ln_copy_unit<TB, BB, WV>(i, lane, wave);
        ob[i] = 2 * r * (MODE == LN_GRAD_W ? g.NB : K) + 16 * u;
        if (MODE == LN_FWD && g.perm) {
            const int row = ln_row(g, t.p0 + min((int)r, t.np - 1));
            if (row < 0) bad |= 1u << i;
            ob[i] = 2 * (uint32_t)max(row, 0) * K + 16 * u;
        }
    }
    const bool any_bad = MODE == LN_FWD && __any(bad != 0);
    /* the gathered rows of step s, asked for a step ahead of their copies; which of them are none, and
     * which of the copies under way are */
    int rows[MODE == LN_GRAD_W ? CA : 1];
    uint32_t none = 0, flying = 0;
    auto look = [&](int s) {
        if constexpr (MODE == LN_GRAD_W) {
            none = 0;
#pragma unroll
            for (int i = 0; i < CA; ++i) {
                const int k = 64 * s + ln_copy_row<TA, BA, WV>(i, lane, wave);
                rows[i] = k < K ? ln_row(g, t.p0 + k) : -1;
                if (rows[i] < 0) none |= 1u << i;
            }
        }
    };
    auto left = [&](int s) { return K - 64 * (MODE == LN_GRAD_X && s >= nk ? s - nk : s); };
    uint32_t la = 0, lb = 0, lodd = 0;
    const uint8_t *odd = sa;                   /* a matrix that is not aligned: its base and limit of the last copies */
    /* before the copies of step s */
    auto turn = [&](int s) {
        if (MODE == LN_GRAD_X && s == nk && s < steps) {
            sa = m3 + 2 * a0;
            ea = m3 + 2 * (size_t)g.NA * g.K;
            sb = g.b3 + 2 * (size_t)t.p0 * K;
            eb = g.b3 + 2 * (size_t)g.P * g.K;
        }
        /* a step past the last is copied all the same, one unit over and over, and not read */
        if (s >= steps) {
            sa = ea - 16;
            sb = eb - 16;
        }
        la = (uint32_t)min((size_t)(ea - sa) - 16, (size_t)0xFFFFFFF0u);
        lb = (uint32_t)min((size_t)(eb - sb) - 16, (size_t)0xFFFFFFF0u);
    };
    auto at_a = [&](int i) {
        if (MODE == LN_GRAD_W && gather) return (uint32_t)max(rows[MODE == LN_GRAD_W ? i : 0], 0) * (2u * g.NA) + oa[i];
        return oa[i];
    };
    auto copy_a = [&](int i) { ln_dma(MODE == LN_GRAD_W ? sa : (const uint8_t *)((uintptr_t)sa & ~(uintptr_t)15), min(at_a(i), la)); };
    auto copy_b = [&](int i) { ln_dma(sb, min(ob[i], lb)); };
    auto moved = [&]() {
        odd = sa;
        lodd = la;
        if (!gather) sa += TA ? (size_t)128 * g.NA : (size_t)128;
        sb += TB ? (size_t)128 * g.NB : (size_t)128;
        flying = none;
    };
    auto copy_to = [&](auto c_, uint32_t to) {
        constexpr int C = decltype(c_)::value;
        ln_dma_at<(C < CA ? 0 : 128 * BA) + 1024 * WV * (C < CA ? C : C - CA)>(to);
        if constexpr (C < CA) copy_a(C);
        else copy_b(C - CA);
    };
    auto copies = [&](int s) {
        const uint32_t to = ldsp + (s & 1) * STAGE;
        turn(s);
        ln_each([&](auto c_) { copy_to(c_, to); }, std::make_integer_sequence<int, CA + CB>{});
        moved();
    };
    /* what this wave's copies of step s brought that does not count, and what DMA could not bring */
    auto fix = [&](int s) {
        const int k = left(s);
        if (s >= steps || (k >= 64 && aligned && !any_bad && !(gather && __any(flying != 0)))) return;
        uint8_t *to = lds + (s & 1) * STAGE + 1024 * wave + 16 * lane;
#pragma unroll
        for (int i = 0; i < CA; ++i) {
            const int r = ln_copy_row<TA, BA, WV>(i, lane, wave), u = ln_copy_unit<TA, BA, WV>(i, lane, wave);
            gm_v4u *o = (gm_v4u *)(to + 1024 * WV * i);
            if (gather ? flying >> i & 1 : (TA ? r : 8 * u) >= k) *o = gm_v4u{0, 0, 0, 0};
            else if (!aligned) *o = *(const LN_G(ln_any16) *)(odd + min(oa[i], lodd));
        }
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const int r = ln_copy_row<TB, BB, WV>(i, lane, wave), u = ln_copy_unit<TB, BB, WV>(i, lane, wave);
            if ((TB ? r : 8 * u) >= k || (bad >> i & 1)) *(gm_v4u *)(to + 128 * BA + 1024 * WV * i) = gm_v4u{0, 0, 0, 0};
        }
        /* no load is pending behind this: the compiler would wait for it, and so for all copies, below */
        gm_wait_vm<0>();
    };

    k3v4f acc[MA][MB], sums[MB];
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        sums[j] = k3v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < MA; ++i) acc[i][j] = k3v4f{0.f, 0.f, 0.f, 0.f};
    }
    const bool bias = MODE == LN_GRAD_W && g.dbias && t.a0 == 0 && wa == 0;
    const k3v8bf one = __builtin_bit_cast(k3v8bf, gm_v4u{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
    k3v8bf fa[MA], fb[2][MB];
    auto read_a = [&](int s, int kh, int i) { fa[i] = ln_frag<TA, BA>(lds + (s & 1) * STAGE, kh, MA * wa + i); };
    auto read_b = [&](int s, int kh, int j) {
        fb[kh][j] = ln_frag<TB, BB>(lds + (s & 1) * STAGE + 128 * BA, kh, MB * wb + j);
    };
    constexpr int PLAN1 = LnPlan<MA, MB, CA + CB>::FIRST;
    /* the products of half kh of step s and what goes on meanwhile: reads of the next half (of the next
     * step after the barrier that the second half has), and copies: of step s + 2 after that barrier,
     * of step s + 1 the rest in the first half */
    auto half = [&](auto kh_, int s) {
        constexpr int KH = decltype(kh_)::value;
        static constexpr LnPlan<MA, MB, CA + CB> plan(KH == 1);
        const uint32_t to = ldsp + ((s + 1 + KH) & 1) * STAGE;
        if (KH == 1) turn(s + 2);
        ln_each([&](auto m_) {
            constexpr int M = decltype(m_)::value, I = M / MB, J = M % MB, C = plan.copy[M];
            constexpr int R0 = plan.read[M][0], R1 = plan.read[M][1];
            ln_mfma<BIG>(fa[I], fb[KH][J], acc[I][J]);
            if constexpr (C >= 0) copy_to(GmInt<C>{}, to);
            if constexpr (KH == 1 && M == plan.BAR) {
                __builtin_amdgcn_s_waitcnt(0x0070);            /* vmcnt(0) lgkmcnt(0) */
                fix(s + 1);
                __syncthreads();
            }
            if constexpr (R0 >= MA) read_b(s + KH, 1 - KH, R0 - MA);
            else if constexpr (R0 >= 0) read_a(s + KH, 1 - KH, R0);
            if constexpr (R1 >= MA) read_b(s + KH, 1 - KH, R1 - MA);
            else if constexpr (R1 >= 0) read_a(s + KH, 1 - KH, R1);
            __builtin_amdgcn_sched_barrier(0);
        }, std::make_integer_sequence<int, MA * MB>{});
        if (bias) {
#pragma unroll
            for (int j = 0; j < MB; ++j) ln_mfma_v<BIG>(one, fb[KH][j], sums[j]);
        }
        if (KH == 0) moved();
    };
    if (steps) {
        if (gather) look(0);
        copies(0);
        gm_wait_vm<0>();
        fix(0);
        __syncthreads();
        if (gather) look(1);
        turn(1);
        ln_each([&](auto c_) { copy_to(c_, ldsp + STAGE); }, std::make_integer_sequence<int, PLAN1>{});
#pragma unroll
        for (int i = 0; i < MA; ++i) read_a(0, 0, i);
#pragma unroll
        for (int j = 0; j < MB; ++j) read_b(0, 0, j);
        if (BIG) asm volatile("s_nop 7" : : : "memory");       /* the sums' zeros */
        for (int s = 0; s < steps; ++s) {
            half(GmInt<0>{}, s);
            if (gather) look(s + 2);
            half(GmInt<1>{}, s);
        }
        gm_wait_vm<0>();
#pragma unroll
        for (int i = 0; i < MA; ++i) ln_settle<BIG>(acc[i]);
        if (MODE == LN_GRAD_W && BIG) {
#pragma unroll
            for (int j = 0; j < MB; ++j) asm volatile("" : "+v"(sums[j]));
        }
    }
    __syncthreads();
    if (bias && lane < 16) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const int b = t.b0 + 16 * MB * wb + 16 * j + lane;
            if (b >= g.NB) continue;
            float *o = g.dbias + (size_t)t.e * g.NB + b;
            *o = g.accumulate ? *o + sums[j][0] : sums[j][0];
        }
    }
    const int valid = MODE == LN_GRAD_W ? g.NB - t.b0 : t.np;
    ln_out<MODE, GATED, Y, MA, MB>(g, (float *)lds + wave * 16 * (16 * MA + 4), acc, out, t.e,
                                   (size_t)(MODE == LN_GRAD_W ? t.b0 : t.p0) + 16 * MB * wb, valid - 16 * MB * wb,
                                   t.a0 + FA / 2 * wa);
}

/* ---------------------------------------------------- through the activation alone ---- */

template <typename T>
__global__ void __launch_bounds__(256)
k_ln_act_grad(const T *dh, const T *z, const T *z3, T *dz, T *dz3, size_t n, int act, float b1, float b2, float i1,
              float i2, bool stream)
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
            ln_put4(dz3 + i, m, d3, stream);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] *= ka_slope(act, v[j]);
        }
        ln_put4(dz + i, m, d, stream);
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
    g.T = rows;
    g.pairs = g.P = rows * topk;
    g.off = off;
    g.E = E;
    return 0;
}

/* workgroups of tiles of fa outputs by fb */
template <int MODE>
static int64_t ln_grid(const LnArgs &g, int fa, int fb)
{
    const int64_t na = (g.NA + fa - 1) / fa;
    if (MODE != LN_GRAD_W) return gm_row_items(g.off != nullptr, g.E, g.P, fb, na);
    return 8 * (int64_t)g.E * ((na * ((g.NB + fb - 1) / fb) + 7) / 8);
}

template <int MODE>
static int ln_launch(const char *who, void (*kernel)(LnArgs), const LnArgs &g, int fa, int fb, int threads,
                     hipStream_t st)
{
    const int64_t blocks = ln_grid<MODE>(g, fa, fb);
    if (blocks * threads > UINT32_MAX) {
        fprintf(stderr, "%s: %d rows by %d columns (%d experts) are more than a launch takes\n", who,
                MODE == LN_GRAD_W ? g.NB : g.P, g.NA, g.E);
        return -1;
    }
    return k3h_launch(who, kernel, dim3((unsigned)blocks), dim3(threads), st, (LnArgs)g);
}

/* bf16 operands whose rows are whole units of 16 bytes */
template <int MODE>
static bool ln_tiles(const LnArgs &g)
{
    if (g.NA % 8 && MODE != LN_FWD) return false;
    if (MODE == LN_GRAD_W ? g.NB % 8 : g.K % 8) return false;
    return !k3h_misaligned(g.b, 16) && !k3h_misaligned(g.b3, 16) && !(MODE == LN_GRAD_W && k3h_misaligned(g.a, 16));
}

/* about how many tiles of fa outputs by fb there are: of an expert's rows, half a tile more than they fill */
template <int MODE>
static double ln_count(const LnArgs &g, int fa, int fb)
{
    const double na = (g.NA + fa - 1) / fa;
    if (MODE == LN_GRAD_W) return na * ((g.NB + fb - 1) / fb) * g.E;
    if (!g.off) return na * ((g.P + fb - 1) / fb);
    const int met = g.E < g.P ? g.E : g.P;
    const double mean = (double)g.P / met;
    return na * met * (mean < fb / 2 ? 1.0 : mean / fb + 0.5);
}

/* 256 x 256 tiles (one a CU) or 128 x 128 (two at a time)? */
template <int MODE>
static bool ln_wide(const LnArgs &g, bool gated)
{
    const double wide = 10.0 * ceil(ln_count<MODE>(g, gated ? 128 : 256, 256) / 256);
    const double small = fmax(3.0 * ceil(ln_count<MODE>(g, gated ? 64 : 128, 128) / 256), 4.2);
    return wide < small;
}

template <int MODE, bool GATED, typename TA, typename TB, typename Y>
static int ln_run(const char *who, const LnArgs &g, hipStream_t st)
{
    if constexpr (sizeof(TA) == 2 && sizeof(TB) == 2) {
        if (ln_tiles<MODE>(g)) {
            if (ln_wide<MODE>(g, GATED))
                return ln_launch<MODE>(who, k_ln_tile<MODE, GATED, Y, 256, 256, 8>, g, GATED ? 128 : 256, 256, 512, st);
            return ln_launch<MODE>(who, k_ln_tile<MODE, GATED, Y, 128, 128, 4>, g, GATED ? 64 : 128, 128, 256, st);
        }
    }
    return ln_launch<MODE>(who, k_ln_any<MODE, GATED, TA, TB, Y>, g, GATED ? 64 : 128, 128, 256, st);
}

template <int MODE, bool GATED, typename TA, typename TB>
static int ln_run_y(const char *who, const LnArgs &g, int ydt, hipStream_t st)
{
    return ydt == K3_WBF16 ? ln_run<MODE, GATED, TA, TB, uint16_t>(who, g, st)
                           : ln_run<MODE, GATED, TA, TB, float>(who, g, st);
}

template <int MODE, bool GATED>
static int ln_product(const char *who, LnArgs &g, int adt, int bdt, int ydt, void *stream)
{
    K3hOn on(stream);
    if (!on.ok) return -1;
    g.stream = (size_t)(MODE == LN_GRAD_W ? (size_t)g.E * g.NB : g.P) * g.NA * ln_size(ydt) > LN_STREAM;
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
    g.T = g.pairs = g.P = rows;
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
    g.T = g.pairs = g.P = rows;
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
    const bool big = count * ln_size(dt) > LN_STREAM;
    if (dt == K3_WBF16)
        return k3h_launch(who, k_ln_act_grad<uint16_t>, grid, dim3(256), on.st, (const uint16_t *)dh,
                          (const uint16_t *)z, (const uint16_t *)z3, (uint16_t *)dz, (uint16_t *)dz3, count, act, b1, b2,
                          i1, i2, big);
    return k3h_launch(who, k_ln_act_grad<float>, grid, dim3(256), on.st, (const float *)dh, (const float *)z,
                      (const float *)z3, (float *)dz, (float *)dz3, count, act, b1, b2, i1, i2,
                      big);
}
