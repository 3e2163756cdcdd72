/* k3g_mx.hip - MXFP4 beyond the layer's own weights: values quantised to it and read back, and
 * products of activations quantised to it with weights in it.
 *
 * Quantisation (OCP Microscaling Formats 1.0): a block is 32 consecutive values of a row; with
 * m their largest magnitude, E = max(floor(log2 m) - 2, -127), so m / 2^E lies in [4, 8) and
 * E2M1's largest value, 6, is reached; the scale byte is E + 127 and a code is x / 2^E in E2M1,
 * to nearest even, what exceeds 6 as 6. Only exponents are read, so nothing here is rounded but
 * the codes. A block with an infinity or NaN gets scale byte 255: it is NaN as a whole.
 *
 * Product: y[r][i] = sum_k q(x)[row(r)][k] W[i][k], both sides in MXFP4, on the scaled matrix
 * instructions with FP4 operands, fp32 accumulation: v_mfma_scale_f32_16x16x128_f8f6f4 for few rows
 * (k_mx_few), v_mfma_scale_f32_32x32x64_f8f6f4 for many (k_mx_gemm). Of the first, the A operand is
 * the tiled layout's 1 KB chunk as it lies (lane L: row L % 16, block L / 16 of the 128 columns, its
 * scale byte with it); the B operand is the same of 16 activation rows. A row of activations is
 * stored for that as quads of 512 columns, 272 bytes: 16 blocks of 16 bytes in column order,
 * then 16 scale bytes, block 4 j + q at 4 q + j, so lane (row, q) gets the scales of its four
 * chunks j in one dword; columns past the last are zero.
 *
 * What bounds them, and what they reach (one MI355X; a large copy moves 4.7 TB/s, read and written):
 * with few rows an expert the stream of the weights, 5.5 to 5.9 TB/s; with many the matrix cores, 3.0
 * to 3.5 PFLOP/s (8192 rows by 7168 x 7168 in 238 us: 50 % busy at about 2.1 GHz; on the same data the
 * matrix instructions alone would take 1.28 of the 1.93 us that a workgroup's 512 columns take, with
 * the operands' reads from LDS 1.47, with the weights' loads 1.69); there and back, memory, 6.5 TB/s
 * (32768 x 7168 bf16 values, 178 us). */
#include <stdio.h>

#include "k3g_act.h"
#include "k3g_dev.h"
#include "k3g_gemm.h"
#include "k3g_groups.h"
#include "k3g_host.h"
#include "k3g_kernels.h"

#define MX_QT 4352                   /* a tiled weight quad: 16 rows x 512 columns */
#define MX_XQ 272                    /* an activation quad: 1 row x 512 columns */
#define MX_MAX_ROWS (1 << 26)
#define MX_MAX_COLS (1 << 20)
#define MX_MAX_PAIRS (1 << 23)
#define MX_MAX_EXPERTS GM_MAX_EXPERTS
#define MX_MAX_QUADS (1 << 26)       /* activation quads of a call: 32 bits for 17 units of 16 bytes each */
#define MX_MAX_BLOCKS (1 << 23)      /* a launch has fewer than 2^32 threads: past 2^31 they loop */

typedef int mx_v8i __attribute__((ext_vector_type(8)));

/* ------------------------------------------------------------- quantisation ---- */

/* 16 bytes of values. STREAM: not to be kept in the caches, for values that are more than the
 * last-level cache's 256 MB (MX_STREAM; 32768 x 7168 bf16 values there and back 221 -> 178 us). */
#define MX_STREAM ((size_t)256 << 20)

template <bool STREAM>
__device__ __forceinline__ gm_v4u mx_get(const void *p)
{
    return STREAM ? __builtin_nontemporal_load((const gm_v4u *)p) : *(const gm_v4u *)p;
}

__device__ __forceinline__ void mx_values(const gm_v4u &u, float (&f)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(u[i]);
}

__device__ __forceinline__ void mx_values(const gm_v4u &u, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = k3d_bf16lo(u[i]);
        f[2 * i + 1] = k3d_bf16hi(u[i]);
    }
}

/* This lane's V values of a block that it shares with the 32 / V lanes around it: their codes,
 * element i in nibble i, and the block's scale byte. Magnitudes are compared as bits, so a NaN is
 * the largest of all. x / 2^E is a multiplication by 2^-E, exact down to 2^-126. */
template <int V>
__device__ __forceinline__ uint32_t mx_quant(const float (&x)[V], uint32_t &scale)
{
    static_assert(V == 4 || V == 8, "lanes of a block");
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    /* of the four lanes of a quad, then, where eight lanes share a block, of its other quad */
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));
    if (V == 4) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true));
    const bool finite = m < 0x7F800000u;
    const uint32_t byte = finite ? (uint32_t)max((int)(m >> 23) - 2, 0) : 127u;
    const float inv = __uint_as_float((254u - byte) << 23);
    uint32_t c = 0;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -6.0f, 6.0f);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.0f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.0f, 1);
    if constexpr (V == 8) {
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.0f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.0f, 3);
    }
    scale = finite ? byte : 255u;
    return finite ? c : 0u;
}

/* A lane takes 16 bytes of values, 8 of bf16 (four lanes a block) or 4 of fp32 (eight), so loads and
 * stores of a wave are whole lines (fp32 with 8 values a lane, every other 16 bytes at a time, 21127 x
 * 5248 values there and back 259 -> 154 us). */
template <typename T, bool STREAM>
__global__ void __launch_bounds__(256)
k_mx_quant(const T *__restrict__ x, size_t n, uint8_t *__restrict__ packed,
           uint8_t *__restrict__ scales)
{
    constexpr int V = 16 / sizeof(T), LANES = 32 / V;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        float f[V];
        mx_values(mx_get<STREAM>(x + V * i), f);
        uint32_t s;
        const uint32_t c = mx_quant(f, s);
        if (V == 8) *(uint32_t *)(packed + 4 * i) = c;
        else *(uint16_t *)(packed + 2 * i) = (uint16_t)c;
        if (i % LANES == 0) scales[i / LANES] = (uint8_t)s;
    }
}

template <typename T, bool STREAM>
__global__ void __launch_bounds__(256)
k_mx_dequant(const uint8_t *__restrict__ packed, const uint8_t *__restrict__ scales, size_t n,
             T *__restrict__ out)
{
    constexpr int V = 16 / sizeof(T), LANES = 32 / V;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const uint32_t b = scales[i / LANES];
        const uint32_t c = V == 8 ? *(const uint32_t *)(packed + 4 * i) : *(const uint16_t *)(packed + 2 * i);
        const float s = b == 255u ? __builtin_nanf("") : k3d_e8m0(b);
        float f[8];
        k3d_fp4x8(c, 1.0f, f);
        gm_v4u u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            u[j] = V == 8 ? k3d_bf16x2(f[2 * j] * s, f[2 * j + 1] * s) : __float_as_uint(f[j] * s);
        gm_v4u *o = (gm_v4u *)(out + V * i);
        if (STREAM) __builtin_nontemporal_store(u, o);
        else *o = u;
    }
}

/* 8 consecutive values */
struct Mx8 {
    float f[8];
};

__device__ __forceinline__ Mx8 mx_load8(const float *p)
{
    const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
    return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}

__device__ __forceinline__ Mx8 mx_load8(const uint16_t *p)
{
    Mx8 v;
    mx_values(*(const gm_v4u *)p, v.f);
    return v;
}

/* x as activation quads (see the top), a wave per quad, and a row of zeros behind them */
template <typename T>
__global__ void __launch_bounds__(256)
k_mx_x(const T *__restrict__ x, size_t nquads, int nQ, int cols, uint8_t *__restrict__ xq)
{
    const int lane = threadIdx.x & 63;
    for (size_t quad = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); quad < nquads + nQ;
         quad += (size_t)gridDim.x * 4) {
        const size_t row = quad / nQ;
        const int col = 512 * (int)(quad - row * nQ) + 8 * lane;
        Mx8 v = {{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
        if (col < cols && quad < nquads) v = mx_load8(x + row * cols + col);
        uint32_t s;
        uint8_t *o = xq + quad * MX_XQ;
        *(uint32_t *)(o + 4 * lane) = mx_quant(v.f, s);
        const int b = lane >> 2;
        if ((lane & 3) == 0) o[256 + 4 * (b & 3) + (b >> 2)] = (uint8_t)s;
    }
}

/* ------------------------------------------------------------------ product ---- */

struct MxProduct {
    const uint8_t *xq;               /* activation quads of T rows and a row of zeros */
    const void *x;                   /* the rows themselves */
    int T, cols, nQ, nK;             /* rows; columns, quads and 128-column chunks of a row */
    const int32_t *perm;             /* place -> pair, or NULL: place r is row r */
    int topk;
    const int32_t *off;              /* [E + 1] places of each expert, or NULL: one, all places */
    int E, P;                        /* P places at most */
    const uint8_t *w, *w3;           /* off NULL: the matrix; else the first expert's pointer */
    int64_t step;                    /* bytes from one expert's pointer to the next */
    int N;
    float b1, b2, i1, i2;            /* the activation's caps and their reciprocals */
    void *y;
    bool stream;                     /* y is more than the last-level cache holds */
};

/* What perm says of a place (the place itself without one), and the activation row that is: -1
 * (zeros) for no pair of these tokens. */
__device__ __forceinline__ int mx_pair(const MxProduct &g, int place) { return g.perm ? g.perm[place] : place; }

__device__ __forceinline__ int mx_row(const MxProduct &g, int pair)
{
    if (!g.perm) return pair;
    const int t = pair / g.topk;
    return pair >= 0 && t < g.T ? t : -1;
}

/* where a pair's activation quads begin, in units of 16 bytes */
__device__ __forceinline__ uint32_t mx_units(const MxProduct &g, int pair)
{
    const int row = mx_row(g, pair);
    return (uint32_t)(row < 0 ? g.T : row) * (uint32_t)(g.nQ * (MX_XQ / 16));
}

__device__ __forceinline__ const uint8_t *mx_matrix(const MxProduct &g, const uint8_t *w, int e)
{
    if (!g.off) return w;
    return gm_uniform_ptr(*(const uint8_t *const *)(w + (size_t)e * g.step));
}

__device__ __forceinline__ void mx_put(float *o, const k3v4f &v) { *(k3v4f *)o = v; }
__device__ __forceinline__ void mx_put(uint16_t *o, const k3v4f &v)
{
    *(uint2 *)o = make_uint2(k3d_bf16x2(v[0], v[1]), k3d_bf16x2(v[2], v[3]));
}

template <int J>
__device__ __forceinline__ k3v4f mx_mma4(const gm_v4u &a, uint32_t sa, const gm_v4u &b, uint32_t sb,
                                         const k3v4f &acc)
{
    const mx_v8i av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
    const mx_v8i bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, J, (int)sa, J, (int)sb);
}

/* v, worked out from here on: an address made of it is not kept in registers over a loop (64-bit
 * ones of every weight and activation pointer took 25 registers more than there are) */
__device__ __forceinline__ uint32_t mx_here(uint32_t v)
{
    asm volatile("" : "+v"(v));
    return v;
}

template <int TM>
__device__ __forceinline__ bool mx_item(const MxProduct &g, int nft, int &ft, int &e, int &p0, int &np)
{
    return gm_row_item<TM>(g.off, g.E, g.P, nft, ft, e, p0, np);
}

__device__ __forceinline__ float mx_act(const MxProduct &g, float gate, float up)
{
    return ka_situ(gate, up, g.b1, g.b2, g.i1, g.i2);
}

/* np rows of zeros from p0 on, features n0 .. n0 + n (an expert without a matrix) */
template <typename Y, int THREADS>
__device__ __forceinline__ void mx_zeros(const MxProduct &g, int p0, int np, int n0, int n)
{
    n = min(n, g.N - n0);
    for (int i = threadIdx.x; i < np * n; i += THREADS)
        ((Y *)g.y)[(size_t)(p0 + i / n) * g.N + n0 + i % n] = (Y)0;
}

/* ---- few rows: a workgroup of WV waves takes 16 NB places by U row blocks of 16 features (gated:
 * U / 2 of each matrix), and the waves share the columns: wave v sums quads v, v + WV, ..., so all
 * the weights of a row block are asked for at once however few row blocks there are. The partial
 * sums meet in LDS and are added in the order of the waves. Both operands come straight from
 * memory, a quad ahead.
 *
 * X: what x is: activation quads, or (a few tokens, NB 1) fp32 or bf16 values that every workgroup
 * quantises by itself, a quad of each row at a time by the wave that needs it: one launch less,
 * for 8 loads and about 40 operations a row and quad beside the 4 KB of each row block. */
struct MxQuads;

template <typename X, int U, int NB>
struct MxFew {
    const uint8_t *w[U];               /* the row blocks' first quads */
    uint32_t x[NB];                    /* this lane's row, in units of 16 bytes (X quads) */
    const X *row;                      /* x itself */
    uint8_t *lds;                      /* this wave's quads of 16 rows (X values) */
    int lane, np, p0;
};

template <typename X, int WV, int U, int NB>
__device__ __forceinline__ void mx_few_sums(const MxProduct &g, const MxFew<X, U, NB> &t, int wave,
                                            k3v4f (&acc)[U][NB])
{
    constexpr bool QUADS = __is_same(X, MxQuads);
    static_assert(QUADS || NB == 1, "values only with one block of rows");
    const int c = t.lane & 15, q = t.lane >> 4;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[u][n] = k3v4f{0.f, 0.f, 0.f, 0.f};
    gm_v4u a[4][U], b[4][NB];
    uint32_t sA[2][U], sB[2][NB];
    auto load = [&](int Q, auto jc) {
        constexpr int J = decltype(jc)::value;
        const uint32_t at = mx_here(16 * t.lane);
#pragma unroll
        for (int u = 0; u < U; ++u) a[J][u] = *(gm_g4)(t.w[u] + (size_t)Q * MX_QT + 1024 * J + at);
        if constexpr (QUADS) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
                b[J][n] = *(gm_g4)(g.xq + (size_t)Q * MX_XQ + (uint64_t)mx_here(t.x[n]) * 16 + 64 * J + 16 * q);
        }
    };
    auto load_scales = [&](int Q, uint32_t (&s)[U], uint32_t (&sb)[NB]) {
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = gm_ld4(t.w[u] + (size_t)Q * MX_QT + 4096 + mx_here(4 * t.lane));
        if constexpr (QUADS) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
                sb[n] = gm_ld4(g.xq + (size_t)Q * MX_XQ + (uint64_t)mx_here(t.x[n]) * 16 + 256 + 4 * q);
        }
    };
    /* this quad of every row into LDS, unit u of row r at slot u ^ r, the scales behind */
    auto values = [&](int Q) {
        if constexpr (!QUADS) {
            const int col = 512 * Q + 8 * t.lane, blk = t.lane >> 2, cols = g.cols;
            gm_wave_sync();
            for (int r = 0; r < t.np; ++r) {
                const int row = gm_uniform(mx_row(g, mx_pair(g, t.p0 + r)));
                Mx8 v = {{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
                if (col < cols && row >= 0) v = mx_load8(t.row + (size_t)row * cols + col);
                uint32_t s;
                const uint32_t code = mx_quant(v.f, s);
                *(uint32_t *)(t.lds + 256 * r + 16 * (blk ^ r) + 4 * (t.lane & 3)) = code;
                if ((t.lane & 3) == 0) t.lds[4096 + 16 * r + 4 * (blk & 3) + (blk >> 2)] = (uint8_t)s;
            }
            gm_wave_sync();
            sB[0][0] = *(const uint32_t *)(t.lds + 4096 + 16 * c + 4 * q);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j][0] = *(const gm_v4u *)(t.lds + 256 * c + 16 * ((4 * j + q) ^ c));
        }
    };
    auto chunk = [&](auto jc) {
        constexpr int J = decltype(jc)::value;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int u = 0; u < U; ++u) acc[u][n] = mx_mma4<J>(a[J][u], sA[0][u], b[J][n], sB[0][n], acc[u][n]);
    };
    if (wave >= g.nQ) return;
    load_scales(wave, sA[0], sB[0]);
    load(wave, GmInt<0>{});
    load(wave, GmInt<1>{});
    load(wave, GmInt<2>{});
    load(wave, GmInt<3>{});
    int Q = wave;
    for (; Q + WV < g.nQ; Q += WV) {
        load_scales(Q + WV, sA[1], sB[1]);
        values(Q);
        chunk(GmInt<0>{});
        load(Q + WV, GmInt<0>{});
        chunk(GmInt<1>{});
        load(Q + WV, GmInt<1>{});
        chunk(GmInt<2>{});
        load(Q + WV, GmInt<2>{});
        chunk(GmInt<3>{});
        load(Q + WV, GmInt<3>{});
#pragma unroll
        for (int u = 0; u < U; ++u) sA[0][u] = sA[1][u];
#pragma unroll
        for (int n = 0; n < NB; ++n) sB[0][n] = sB[1][n];
    }
    values(Q);
    const int left = g.nK - 4 * Q;
    chunk(GmInt<0>{});
    if (left > 1) chunk(GmInt<1>{});
    if (left > 2) chunk(GmInt<2>{});
    if (left > 3) chunk(GmInt<3>{});
}

template <typename X, typename Y, bool GATED, int WV, int U, int NB>
__global__ void __launch_bounds__(64 * WV)
k_mx_few(const MxProduct g)
{
    constexpr bool QUADS = __is_same(X, MxQuads);
    constexpr int RB = GATED ? U / 2 : U, SUMS = WV * U * NB * 1024, VALUES = QUADS ? 0 : WV * MX_QT;
    __shared__ __attribute__((aligned(16))) uint8_t lds[SUMS > VALUES ? SUMS : VALUES];
    const int nrb = g.N / 16, nft = (nrb + RB - 1) / RB;
    int ft, e, p0, np;
    if (!mx_item<16 * NB>(g, nft, ft, e, p0, np)) return;
    const uint8_t *w1 = mx_matrix(g, g.w, e), *w3 = GATED ? mx_matrix(g, g.w3, e) : w1;
    if (!w1 || !w3) {
        mx_zeros<Y, 64 * WV>(g, p0, np, 16 * RB * ft, 16 * RB);
        return;
    }
    const int wave = gm_uniform(threadIdx.x >> 6);
    MxFew<X, U, NB> t;
    t.lane = threadIdx.x & 63;
    const int c = t.lane & 15, q = t.lane >> 4;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int rb = RB * ft + u % RB;
        t.w[u] = gm_uniform_ptr((u >= RB ? w3 : w1) + (rb >= nrb ? 0 : (size_t)rb * g.nQ * MX_QT));
    }
    if constexpr (QUADS) {
#pragma unroll
        for (int n = 0; n < NB; ++n) t.x[n] = mx_units(g, mx_pair(g, p0 + min(16 * n + c, np - 1)));
    } else {
        t.row = (const X *)g.x;
        t.lds = lds + wave * MX_QT;
    }
    t.np = np;
    t.p0 = p0;
    k3v4f acc[U][NB];
    mx_few_sums<X, WV, U, NB>(g, t, wave, acc);
    /* the waves' sums: tile (u, n) of wave v at (v U NB + u NB + n) KB, 16 bytes a lane */
    if constexpr (!QUADS) __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NB; ++n)
            *(k3v4f *)(lds + 1024 * ((wave * U + u) * NB + n) + 16 * t.lane) = acc[u][n];
    __syncthreads();
    auto total = [&](int u, int n) {
        k3v4f s = *(const k3v4f *)(lds + 1024 * (u * NB + n) + 16 * t.lane);
#pragma unroll
        for (int v = 1; v < WV; ++v)
            if (v < g.nQ) s += *(const k3v4f *)(lds + 1024 * ((v * U + u) * NB + n) + 16 * t.lane);
        return s;
    };
#pragma unroll
    for (int i0 = 0; i0 < RB * NB; i0 += WV) {
        const int i = i0 + wave, r = i / NB, n = i - r * NB;
        if (i >= RB * NB || RB * ft + r >= nrb || 16 * n + c >= np) continue;
        k3v4f v = total(r, n);
        if (GATED) {
            const k3v4f up = total(RB + r, n);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = mx_act(g, v[j], up[j]);
        }
        mx_put((Y *)g.y + (size_t)(p0 + 16 * n + c) * g.N + 16 * (RB * ft + r) + 4 * q, v);
    }
}

/* ---- many rows: a workgroup of four waves takes up to TM places by 4 x 64 features (gated: 4 x
 * 32 of each matrix). The activation quads of its places go to LDS by DMA, two stages of one quad;
 * the 16-byte unit u of row r lies at slot u ^ (r % 16) of the row's 256 bytes, so 16 rows of an
 * operand read 16 different slots. Weights go straight from memory to registers, a quad ahead: no
 * two waves of a workgroup share them.
 *
 * The products are v_mfma_scale_f32_32x32x64_f8f6f4: an instruction with scales takes longer to
 * issue than the 16 cycles the 16x16x128 form keeps the matrix cores (from registers alone, one
 * or two waves a SIMD, 5.4 and 6.9 PFLOP/s against 8.2 and 9.3). Its A operand is half a chunk of
 * two row blocks: lane (d, hi) = (L % 32, L / 32) holds MX block 2 h + hi of the matrix row
 * that lies 16 (d / 4 % 2) + 4 (d / 8) + d % 4 from the first. In that order of rows a lane's 16
 * sums are 16 features in a row, 16 hi on, of place d. */
typedef float mx_v16f __attribute__((ext_vector_type(16)));

template <int J>
__device__ __forceinline__ mx_v16f mx_mma32(const gm_v4u &a, uint32_t sa, const gm_v4u &b, uint32_t sb,
                                            const mx_v16f &acc)
{
    const mx_v8i av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
    const mx_v8i bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc, 4, 4, J, (int)sa, J, (int)sb);
}

template <int TM, int WV>
struct MxWave {
    static constexpr int SCALES = TM * 256, STAGE = TM * MX_XQ;
    static constexpr int COPIES = (TM / 4 + WV - 1) / WV;      /* of 4 rows, by each wave */
    const uint8_t *w[2];               /* two pairs of row blocks: the first's first quad, */
    uint32_t at[2], sat[2];            /* this lane's codes and scales from there */
    const uint8_t *xq;                 /* the activations; in units of 16 bytes from there: */
    int row[COPIES], rows;             /* rows 4 (wave + WV i) .. + 3: the one this lane copies a unit of, */
    uint32_t unit[COPIES];             /* and which; the one whose scales it copies (waves below TM / 64) */
    uint32_t lds;
    const uint8_t *ldsp;
    int lane, wave, nQ, nK;
};

/* NB blocks of 32 places */
template <int TM, int WV, int NB>
__device__ __forceinline__ void mx_gemm_sums(const MxProduct &g, const MxWave<TM, WV> &t,
                                             mx_v16f (&acc)[2][NB])
{
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[r][n] = mx_v16f{};
    const int d = t.lane & 31, hi = t.lane >> 5;
    gm_v4u a[4][2][2];
    uint32_t sA[2][2], sN[2][2], x[MxWave<TM, WV>::COPIES], xs;
    auto load = [&](int Q, auto jc) {
        constexpr int J = decltype(jc)::value;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t at = mx_here(t.at[r]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                a[J][h][r] = *(gm_g4)(t.w[r] + (size_t)Q * MX_QT + 1024 * J + 512 * h + at);
        }
    };
    auto load_scales = [&](int Q, uint32_t (&s)[2][2]) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t at = mx_here(t.sat[r]);
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h][r] = gm_ld4(t.w[r] + (size_t)Q * MX_QT + 4096 + 128 * h + at);
        }
    };
    auto dma = [&](int Q) {
        const uint32_t st = t.lds + (Q & 1) * t.STAGE;
        const uint8_t *from = t.xq + (size_t)Q * MX_XQ;
#pragma unroll
        for (int i = 0; WV * i < 8 * NB; ++i) {
            const int at = WV * i + t.wave;
            if (WV * (i + 1) <= 8 * NB || at < 8 * NB)
                gm_dma16(from + (uint64_t)mx_here(x[i]) * 16, st + 1024 * at);
        }
        if (64 * t.wave < 32 * NB)
            gm_dma16(from + (uint64_t)mx_here(xs) * 16, st + t.SCALES + 1024 * t.wave);
    };
    /* operands are read one block ahead of their products, over the chunks of a quad (two and three
     * ahead are no faster: 8192 rows by 8192 x 8192 in 314, 316 and 319 us) */
    gm_v4u b[2];
    auto read = [&](const uint8_t *st, int jh, int n) {
        return *(const gm_v4u *)(st + 256 * d + 16 * ((2 * jh + hi) ^ (d & 15)) + 8192 * n);
    };
    auto chunk = [&](const uint8_t *st, const uint32_t (&sB)[2][NB], auto jc) {
        constexpr int J = decltype(jc)::value;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int i = (2 * J + h) * NB + n;
                if (i + 1 < 8 * NB) b[(i + 1) & 1] = read(st, (i + 1) / NB, (i + 1) % NB);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    acc[r][n] = mx_mma32<J>(a[J][h][r], sA[h][r], b[i & 1], sB[h][n], acc[r][n]);
            }
    };
    auto quad = [&](int Q, auto more) {
        constexpr bool MORE = decltype(more)::value;
        /* this quad's copies are older than the 20 weight loads issued since */
        gm_wait_vm<20>();
        __syncthreads();
        if (MORE) {
            dma(Q + 1);
            load_scales(Q + 1, sN);
        }
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *st = t.ldsp + (Q & 1) * t.STAGE;
        uint32_t sB[2][NB];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NB; ++n)
                sB[h][n] = *(const uint32_t *)(st + t.SCALES + 512 * n + 16 * d + 8 * h + 4 * hi);
        const int left = MORE ? 4 : t.nK - 4 * Q;
        b[0] = read(st, 0, 0);
        chunk(st, sB, GmInt<0>{});
        if (MORE) load(Q + 1, GmInt<0>{});
        if (left > 1) chunk(st, sB, GmInt<1>{});
        if (MORE) load(Q + 1, GmInt<1>{});
        if (left > 2) chunk(st, sB, GmInt<2>{});
        if (MORE) load(Q + 1, GmInt<2>{});
        if (left > 3) chunk(st, sB, GmInt<3>{});
        if (MORE) {
            load(Q + 1, GmInt<3>{});
#pragma unroll
            for (int i = 0; i < 4; ++i) sA[i >> 1][i & 1] = sN[i >> 1][i & 1];
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    /* the weights are asked for before the rows of the activations are known */
    load_scales(0, sA);
    load(0, GmInt<0>{});
    load(0, GmInt<1>{});
    load(0, GmInt<2>{});
    load(0, GmInt<3>{});
#pragma unroll
    for (int i = 0; i < t.COPIES; ++i) x[i] = mx_units(g, t.row[i]) + t.unit[i];
    xs = mx_units(g, t.rows) + 16;
    dma(0);
    gm_wait_vm<0>();
    for (int Q = 0; Q + 1 < t.nQ; ++Q) quad(Q, GmInt<1>{});
    quad(t.nQ - 1, GmInt<0>{});
}

/* 16 consecutive sums as units of 16 bytes at o, unit i at slot (u + i) ^ x */
__device__ __forceinline__ void mx_put16(uint8_t *o, int u, int x, const mx_v16f &v, float)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *(k3v4f *)(o + 16 * ((u + i) ^ x)) = k3v4f{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
}

__device__ __forceinline__ void mx_put16(uint8_t *o, int u, int x, const mx_v16f &v, uint16_t)
{
#pragma unroll
    for (int i = 0; i < 2; ++i)
        *(gm_v4u *)(o + 16 * ((u + i) ^ x)) =
            gm_v4u{k3d_bf16x2(v[8 * i], v[8 * i + 1]), k3d_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                   k3d_bf16x2(v[8 * i + 4], v[8 * i + 5]), k3d_bf16x2(v[8 * i + 6], v[8 * i + 7])};
}

/* The sums go out by way of LDS, a wave's own 16 KB (TM 128) at a time: a lane holds 32 or 64 bytes
 * of one place's row, and stored as they are they reach the L2 as quarters of lines (470 MB of bf16
 * rows cost 129 of 729 us); read back by rows, a wave stores 8 rows of 128 bytes at once. */
template <typename Y, bool GATED, int NB, int TM, int WV>
__device__ __forceinline__ void mx_gemm_tile(const MxProduct &g, const MxWave<TM, WV> &t, uint8_t *lds,
                                             int p0, int np, int rb0)
{
    mx_v16f acc[2][NB];
    mx_gemm_sums<TM, WV, NB>(g, t, acc);
    const int d = t.lane & 31, hi = t.lane >> 5;
    constexpr int F = GATED ? 32 : 64, UNITS = F * (int)sizeof(Y) / 16;      /* of a row */
    constexpr int FIT = TM * 128 / (32 * UNITS * 16), PER = FIT < NB ? FIT : NB;
    static_assert(WV * TM * 128 <= 2 * MxWave<TM, WV>::STAGE, "LDS");
    uint8_t *mine = lds + t.wave * TM * 128;
    __syncthreads();
#pragma unroll
    for (int n0 = 0; n0 < NB; n0 += PER) {
#pragma unroll
        for (int n = n0; n < n0 + PER && n < NB; ++n) {
            const int row = 32 * (n - n0) + d;
#pragma unroll
            for (int r = 0; r < (GATED ? 1 : 2); ++r) {
                mx_v16f v = acc[r][n];
                if (GATED) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = mx_act(g, v[i], acc[1][n][i]);
                }
                mx_put16(mine + 16 * UNITS * row, (32 * r + 16 * hi) * (int)sizeof(Y) / 16, row % UNITS, v, Y());
            }
        }
        gm_wave_sync();
        const int u = t.lane % UNITS, f = 16 * rb0 + u * (16 / (int)sizeof(Y));
        const int rows = min(np - 32 * n0, 32 * PER);
        Y *o = (Y *)g.y + (size_t)(p0 + 32 * n0) * g.N + f;
        for (int row = t.lane / UNITS; row < rows; row += 64 / UNITS)
            if (f < g.N) {
                const gm_v4u v = *(const gm_v4u *)(mine + 16 * (UNITS * row + (u ^ row % UNITS)));
                if (g.stream) __builtin_nontemporal_store(v, (gm_v4u *)(o + (size_t)row * g.N));
                else *(gm_v4u *)(o + (size_t)row * g.N) = v;
            }
        gm_wave_sync();
    }
}

template <typename Y, bool GATED, int TM, int WV>
__global__ void __launch_bounds__(64 * WV, 2)
k_mx_gemm(const MxProduct g)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * MxWave<TM, WV>::STAGE];
    constexpr int RB = GATED ? 2 : 4;           /* row blocks of a wave in a matrix */
    const int nrb = g.N / 16, nft = (nrb + WV * RB - 1) / (WV * RB);
    int ft, e, p0, np;
    if (!mx_item<TM>(g, nft, ft, e, p0, np)) return;
    MxWave<TM, WV> t;
    t.lane = threadIdx.x & 63;
    t.wave = gm_uniform(threadIdx.x >> 6);
    t.nQ = g.nQ;
    t.nK = g.nK;
    t.xq = g.xq;
    t.lds = (uint32_t)(uintptr_t)(k3lds)lds;
    t.ldsp = lds;
    const uint8_t *w1 = mx_matrix(g, g.w, e), *w3 = GATED ? mx_matrix(g, g.w3, e) : w1;
    const int rb0 = (WV * ft + t.wave) * RB;
    if (!w1 || !w3) {
        mx_zeros<Y, 64 * WV>(g, p0, np, 16 * WV * RB * ft, 16 * WV * RB);
        return;
    }
    const int d = t.lane & 31, hi = t.lane >> 5, row = 4 * (d >> 3) + (d & 3);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        /* row blocks past the last are read as the first one and never stored */
        const int rb = rb0 + (GATED ? 0 : 2 * r);
        t.w[r] = gm_uniform_ptr((GATED && r ? w3 : w1) + (rb >= nrb ? 0 : (size_t)rb * g.nQ * MX_QT));
        const uint32_t second = rb + 1 < nrb ? ((d >> 2) & 1) * (uint32_t)g.nQ * MX_QT : 0;
        t.at[r] = second + 16 * row + 256 * hi;
        t.sat[r] = second + 4 * row + 64 * hi;
    }
    const int nb = (np + 31) / 32;
#pragma unroll
    for (int i = 0; i < t.COPIES; ++i) {
        const int r = 4 * (WV * i + t.wave) + (t.lane >> 4);
        t.row[i] = mx_pair(g, p0 + min(r, np - 1));
        t.unit[i] = (t.lane & 15) ^ (r & 15);
    }
    t.rows = mx_pair(g, p0 + min(64 * t.wave + t.lane, np - 1));
    if constexpr (TM == 128) {
        if (nb == 4) return mx_gemm_tile<Y, GATED, 4>(g, t, lds, p0, np, rb0);
        if (nb == 3) return mx_gemm_tile<Y, GATED, 3>(g, t, lds, p0, np, rb0);
    }
    if (nb == 2) return mx_gemm_tile<Y, GATED, 2>(g, t, lds, p0, np, rb0);
    mx_gemm_tile<Y, GATED, 1>(g, t, lds, p0, np, rb0);
}

/* ------------------------------------------------------------- entry points ---- */

static int mx_type(const char *who, int dt)
{
    if (dt == K3_WF32 || dt == K3_WBF16) return 0;
    fprintf(stderr, "%s: values are fp32 (%d) or bf16 (%d), not %d\n", who, K3_WF32, K3_WBF16, dt);
    return -1;
}

static bool mx_shape_ok(int rows, int cols)
{
    return rows >= 0 && rows <= MX_MAX_ROWS && cols >= 32 && cols % 32 == 0 && cols <= MX_MAX_COLS;
}

static int mx_shape(const char *who, int rows, int cols)
{
    if (mx_shape_ok(rows, cols)) return 0;
    fprintf(stderr, "%s: needs 0 to %d rows and a multiple of 32 columns up to %d (%d x %d)\n", who,
            MX_MAX_ROWS, MX_MAX_COLS, rows, cols);
    return -1;
}

static int mx_pointer(const char *who, const char *name, const void *p, int to, bool needed)
{
    if ((p || !needed) && !k3h_misaligned(p, to)) return 0;
    fprintf(stderr, "%s: %s is missing or not aligned to %d bytes\n", who, name, to);
    return -1;
}

extern "C" int k3g_quant_mxfp4(const void *x, int dt, int rows, int cols, void *packed, void *scales,
                               void *stream)
{
    const char *who = "k3g_quant_mxfp4";
    if (mx_type(who, dt) || mx_shape(who, rows, cols) || mx_pointer(who, "x", x, 16, rows > 0) ||
        mx_pointer(who, "packed", packed, 16, rows > 0) || mx_pointer(who, "scales", scales, 1, rows > 0))
        return -1;
    if (!rows) return 0;
    K3hOn on(stream);
    if (!on.ok) return -1;
    const size_t n = (size_t)rows * cols / (dt == K3_WBF16 ? 8 : 4);
    const dim3 grid((unsigned)min((n + 255) / 256, (size_t)MX_MAX_BLOCKS));
    const bool big = 16 * n > MX_STREAM;
    if (dt == K3_WBF16)
        return k3h_launch(who, big ? k_mx_quant<uint16_t, true> : k_mx_quant<uint16_t, false>, grid,
                          dim3(256), on.st, (const uint16_t *)x, n, (uint8_t *)packed, (uint8_t *)scales);
    return k3h_launch(who, big ? k_mx_quant<float, true> : k_mx_quant<float, false>, grid, dim3(256),
                      on.st, (const float *)x, n, (uint8_t *)packed, (uint8_t *)scales);
}

extern "C" int k3g_dequant_mxfp4(const void *packed, const void *scales, int rows, int cols, void *out,
                                 int dt, void *stream)
{
    const char *who = "k3g_dequant_mxfp4";
    if (mx_type(who, dt) || mx_shape(who, rows, cols) || mx_pointer(who, "out", out, 16, rows > 0) ||
        mx_pointer(who, "packed", packed, 16, rows > 0) || mx_pointer(who, "scales", scales, 1, rows > 0))
        return -1;
    if (!rows) return 0;
    K3hOn on(stream);
    if (!on.ok) return -1;
    const size_t n = (size_t)rows * cols / (dt == K3_WBF16 ? 8 : 4);
    const dim3 grid((unsigned)min((n + 255) / 256, (size_t)MX_MAX_BLOCKS));
    const bool big = 16 * n > MX_STREAM;
    if (dt == K3_WBF16)
        return k3h_launch(who, big ? k_mx_dequant<uint16_t, true> : k_mx_dequant<uint16_t, false>, grid,
                          dim3(256), on.st, (const uint8_t *)packed, (const uint8_t *)scales, n,
                          (uint16_t *)out);
    return k3h_launch(who, big ? k_mx_dequant<float, true> : k_mx_dequant<float, false>, grid, dim3(256),
                      on.st, (const uint8_t *)packed, (const uint8_t *)scales, n, (float *)out);
}

extern "C" size_t k3g_mxfp4_work_bytes(int rows, int cols)
{
    if (!mx_shape_ok(rows, cols) || !rows) return 0;
    /* and a row of zeros behind them, for places without one */
    const size_t quads = ((size_t)rows + 1) * ((cols + 511) / 512);
    return quads < MX_MAX_QUADS ? quads * MX_XQ : 0;
}

/* Which kernel a product runs on: rows of a tile, its row blocks (of each matrix), the waves that
 * share its columns (0: k_mx_gemm, a wave per four row blocks, or two of each matrix), and whether x
 * is quantised inside it. */
struct MxPlan {
    int tm, rb, wv;
    bool values;
    unsigned blocks;
};

/* workgroups of tiles of tm rows by rb row blocks */
static int64_t mx_grid(const MxProduct &g, int tm, int rb)
{
    return gm_row_items(g.off != nullptr, g.E, g.P, tm, (g.N / 16 + rb - 1) / rb);
}

/* One matrix: a CU's workgroups take turns on what bounds them (its matrix cores, the data that
 * its L1 returns), so a call lasts as long as the CU with the most, ceil(workgroups / 256) times the
 * time of one. That time, in us at 7168 columns beside about 6 of quantisation and launch, is `us`:
 * the tile with the smallest product is taken. Only 7168 columns were measured; the rule does not look
 * at them. Whole calls, us, bf16, tiles in the table's order:
 *   16 rows by 3584            23.4  .     23.3  .     14.3  10.9  12.4  9.5   8.5
 *   64 rows                    28.9  .     28.6  .     20.2  14.4  11.7  12.9  16.6
 *   256 rows                   33.7  30.7  26.6  23.0  19.5  21.8  26.2  30.2  42.6
 *   512 rows by 6144           34.9  32.5  28.2  25.5  48.1  50.8  63.5  89.1  135
 *   1024 rows                  37.7  36.5  45.6  39.9  85.6
 *   2048 rows                  66.1  60.9  70.1  74.0  162
 *   4096 rows by 7168          130   139   153   166   365
 * Up to four rows are quantised inside (1 row 5.5 against 7.2, 4 rows 7.6 and 7.7, 8 rows 10.8 and
 * 7.5).
 *
 * Experts: a few tokens meet about one row an expert, and the weights are all there is to wait for.
 * From 17 rows of x on the rule counts workgroups before it looks at the rows an expert: many experts
 * of about one row then run by 64 places too, where the second line has the forms by 16 and 32 7 %
 * ahead. Nothing between 8 and 4096 tokens by 384 experts was measured.
 * us, bf16: quantised inside, before by 16 places, by 32, k_mx_gemm by 64, by 128:
 *   1 token x 8 by 384 of 7168 -> 2 x 2048     21.9  23.9  24.0  24.7  24.9
 *   8 tokens x 8                               133   131   131   141   141
 *   16 x 8 by 8 of 4096 -> 2 x 1408            27.7  14.4  14.9  15.9  16.0
 *   64 x 2                                     28.2  16.3  16.0  16.2  16.4
 *   256 x 2                                    58.1  25.8  24.1  22.2  30.7
 *   1024 x 2                                   202   62.9  52.8  33.4  35.1
 *   4096 x 8 by 384 of 2048 -> 7168            4021  1854  1452  750   680
 *   4096 x 8 by 384 of 7168 -> 2 x 2048        9186  2648  2224  1291  1221 */
static MxPlan mx_plan(const MxProduct &g, bool gated)
{
    static const struct { int tm, rb, wv; float us; } tiles[] = {
        {128, 16, 0, 28.f}, {128, 12, 0, 25.f}, {64, 16, 0, 20.f}, {64, 12, 0, 17.f}, {64, 4, 4, 13.5f},
        {32, 4, 4, 8.f},    {16, 4, 4, 5.5f},   {16, 2, 4, 3.4f},  {16, 1, 8, 2.6f},
    };
    const int RB = gated ? 2 : 4;
    if (!g.off) {
        if (g.P <= 4) return {16, 1, 8, true, 0};
        MxPlan best = {};
        float least = 0.0f;
        for (const auto &t : tiles) {
            const float us = (float)((mx_grid(g, t.tm, t.rb) + 255) / 256) * t.us;
            if (!best.tm || us < least) {
                best = {t.tm, t.rb, t.wv, false, 0};
                least = us;
            }
        }
        return best;
    }
    const int met = min(g.E, g.P), mean = (g.P + met - 1) / met;
    if (g.T <= 16 && mean <= 2) return {16, RB, 4, true, 0};
    /* row tiles there will be, about: one an expert or more */
    const int64_t nft = (g.N / 16 + 4 * RB - 1) / (4 * RB);
    if (mean > 48 && max(met, g.P / 128) * nft >= 256) return {128, 4 * RB, 0, false, 0};
    if (max(met, g.P / 64) * nft >= 256) return {64, 4 * RB, 0, false, 0};
    return {mean > 16 ? 32 : 16, RB, 4, false, 0};
}

template <typename X, typename Y, bool GATED, int WV, int U, int NB>
static int mx_run_few(const char *who, const MxProduct &g, const MxPlan &p, hipStream_t st)
{
    return k3h_launch(who, k_mx_few<X, Y, GATED, WV, U, NB>, dim3(p.blocks), dim3(64 * WV), st, (MxProduct)g);
}

template <typename Y, bool GATED, int TM, int WV>
static int mx_run_gemm(const char *who, const MxProduct &g, const MxPlan &p, hipStream_t st)
{
    return k3h_launch(who, k_mx_gemm<Y, GATED, TM, WV>, dim3(p.blocks), dim3(64 * WV), st, (MxProduct)g);
}

template <typename X>
static int mx_launch_values(const char *who, const MxProduct &g, const MxPlan &p, bool bf, bool gated,
                            hipStream_t st)
{
    if (gated) return bf ? mx_run_few<X, uint16_t, true, 4, 4, 1>(who, g, p, st)
                         : mx_run_few<X, float, true, 4, 4, 1>(who, g, p, st);
    if (p.wv == 8) return bf ? mx_run_few<X, uint16_t, false, 8, 1, 1>(who, g, p, st)
                             : mx_run_few<X, float, false, 8, 1, 1>(who, g, p, st);
    return bf ? mx_run_few<X, uint16_t, false, 4, 4, 1>(who, g, p, st)
              : mx_run_few<X, float, false, 4, 4, 1>(who, g, p, st);
}

template <typename Y>
static int mx_launch(const char *who, const MxProduct &g, const MxPlan &p, bool gated, hipStream_t st)
{
    if (!p.wv) {
        if (gated) return p.tm == 128 ? mx_run_gemm<Y, true, 128, 4>(who, g, p, st)
                                      : mx_run_gemm<Y, true, 64, 4>(who, g, p, st);
        if (p.rb == 12) return p.tm == 128 ? mx_run_gemm<Y, false, 128, 3>(who, g, p, st)
                                           : mx_run_gemm<Y, false, 64, 3>(who, g, p, st);
        return p.tm == 128 ? mx_run_gemm<Y, false, 128, 4>(who, g, p, st)
                           : mx_run_gemm<Y, false, 64, 4>(who, g, p, st);
    }
    if (gated) return p.tm == 32 ? mx_run_few<MxQuads, Y, true, 4, 4, 2>(who, g, p, st)
                                 : mx_run_few<MxQuads, Y, true, 4, 4, 1>(who, g, p, st);
    if (p.wv == 8) return mx_run_few<MxQuads, Y, false, 8, 1, 1>(who, g, p, st);
    if (p.rb == 2) return mx_run_few<MxQuads, Y, false, 4, 2, 1>(who, g, p, st);
    if (p.tm == 64) return mx_run_few<MxQuads, Y, false, 4, 4, 4>(who, g, p, st);
    return p.tm == 32 ? mx_run_few<MxQuads, Y, false, 4, 4, 2>(who, g, p, st)
                      : mx_run_few<MxQuads, Y, false, 4, 4, 1>(who, g, p, st);
}

/* the product of checked arguments */
static int mx_product(const char *who, MxProduct &g, const void *x, int xdt, int cols, int ydt,
                      void *work, size_t work_bytes, void *stream)
{
    const size_t need = k3g_mxfp4_work_bytes(g.T, cols);
    if (!need) {
        fprintf(stderr, "%s: %d x %d activations are more than %d blocks of 512\n", who, g.T, cols,
                MX_MAX_QUADS);
        return -1;
    }
    if (!work || k3h_misaligned(work, 16) || work_bytes < need) {
        fprintf(stderr, "%s: needs a workspace of %zu bytes, aligned to 16 (%zu given)\n", who, need,
                work ? work_bytes : (size_t)0);
        return -1;
    }
    K3hOn on(stream);
    if (!on.ok) return -1;
    g.nQ = (cols + 511) / 512;
    g.nK = (cols + 127) / 128;
    g.xq = (const uint8_t *)work;
    g.x = x;
    g.cols = cols;
    g.stream = (size_t)g.P * g.N * (ydt == K3_WBF16 ? 2 : 4) > MX_STREAM;
    const bool bf = ydt == K3_WBF16, gated = g.w3 != nullptr;
    MxPlan plan = mx_plan(g, gated);
    const int64_t blocks = mx_grid(g, plan.tm, plan.rb);
    if (blocks * 512 > UINT32_MAX) {
        fprintf(stderr, "%s: %d places by %d features are more than a launch takes\n", who, g.P, g.N);
        return -1;
    }
    plan.blocks = (unsigned)blocks;
    if (plan.values)
        return xdt == K3_WBF16 ? mx_launch_values<uint16_t>(who, g, plan, bf, gated, on.st)
                               : mx_launch_values<float>(who, g, plan, bf, gated, on.st);
    const size_t nquads = (size_t)g.T * g.nQ;
    const dim3 xgrid((unsigned)min((nquads + g.nQ + 3) / 4, (size_t)MX_MAX_BLOCKS));
    if (xdt == K3_WBF16 ? k3h_launch(who, k_mx_x<uint16_t>, xgrid, dim3(256), on.st, (const uint16_t *)x,
                                     nquads, g.nQ, cols, (uint8_t *)work)
                        : k3h_launch(who, k_mx_x<float>, xgrid, dim3(256), on.st, (const float *)x, nquads,
                                     g.nQ, cols, (uint8_t *)work))
        return -1;
    return bf ? mx_launch<uint16_t>(who, g, plan, gated, on.st) : mx_launch<float>(who, g, plan, gated, on.st);
}

static int mx_features(const char *who, int n)
{
    if (n >= 16 && n % 16 == 0 && n <= MX_MAX_COLS) return 0;
    fprintf(stderr, "%s: needs a multiple of 16 features up to %d (%d)\n", who, MX_MAX_COLS, n);
    return -1;
}

extern "C" int k3g_matmul_mxfp4(const void *x, int xdt, int rows, int cols, const void *w, int n, void *y,
                                int ydt, void *work, size_t work_bytes, void *stream)
{
    const char *who = "k3g_matmul_mxfp4";
    if (mx_type(who, xdt) || mx_type(who, ydt) || mx_shape(who, rows, cols) || mx_features(who, n) ||
        mx_pointer(who, "x", x, 16, rows > 0) || mx_pointer(who, "w", w, 16, rows > 0) ||
        mx_pointer(who, "y", y, 16, rows > 0))
        return -1;
    if (!rows) return 0;
    MxProduct g = {};
    g.T = g.P = rows;
    g.topk = g.E = 1;
    g.w = (const uint8_t *)w;
    g.N = n;
    g.y = y;
    return mx_product(who, g, x, xdt, cols, ydt, work, work_bytes, stream);
}

extern "C" int k3g_grouped_mxfp4(const void *x, int xdt, int rows, int cols, const int32_t *perm, int topk,
                                 const int32_t *off, int n_experts, const void *const *w,
                                 const void *const *w3, int w_step, int n, float b1, float b2, void *y,
                                 int ydt, void *work, size_t work_bytes, void *stream)
{
    const char *who = "k3g_grouped_mxfp4";
    if (mx_type(who, xdt) || mx_type(who, ydt) || mx_shape(who, rows, cols) || mx_features(who, n) ||
        mx_pointer(who, "x", x, 16, rows > 0) || mx_pointer(who, "y", y, 16, rows > 0) ||
        mx_pointer(who, "off", off, 4, rows > 0) || mx_pointer(who, "perm", perm, 4, false) ||
        mx_pointer(who, "w", w, 8, rows > 0) || mx_pointer(who, "w3", w3, 8, false))
        return -1;
    if (n_experts < 1 || n_experts > MX_MAX_EXPERTS || topk < 1 || topk > K3G_MAX_TOPK || (!perm && topk != 1) ||
        (int64_t)rows * topk > MX_MAX_PAIRS) {
        fprintf(stderr, "%s: needs 1 to %d experts, 1 <= topk <= %d (1 without perm) and at most %d "
                        "pairs (%d experts, %d x %d)\n", who, MX_MAX_EXPERTS, K3G_MAX_TOPK, MX_MAX_PAIRS, n_experts, rows,
                topk);
        return -1;
    }
    if (w_step < 8 || w_step % 8) {
        fprintf(stderr, "%s: w_step is a multiple of 8 bytes (%d)\n", who, w_step);
        return -1;
    }
    /* below, a cap's reciprocal may be infinite */
    if (w3 && !(b1 >= 0x1p-100f && b2 >= 0x1p-100f)) {
        fprintf(stderr, "%s: the activation's caps are 2^-100 or more (%g, %g)\n", who, b1, b2);
        return -1;
    }
    if (!rows) return 0;
    MxProduct g = {};
    g.T = rows;
    g.perm = perm;
    g.topk = topk;
    g.off = off;
    g.E = n_experts;
    g.P = rows * topk;
    g.w = (const uint8_t *)w;
    g.w3 = (const uint8_t *)w3;
    g.step = w_step;
    g.N = n;
    g.b1 = b1;
    g.b2 = b2;
    g.i1 = 1.0f / b1;
    g.i2 = 1.0f / b2;
    g.y = y;
    return mx_product(who, g, x, xdt, cols, ydt, work, work_bytes, stream);
}
