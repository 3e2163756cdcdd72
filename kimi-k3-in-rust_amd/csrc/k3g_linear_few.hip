/* k3g_linear_few.hip - products of a few rows, and of experts that have a few each (k3g_linear.hip
 * has the formulas), of any types and widths: the weights are read once and are all there is to wait
 * for.
 *
 * A workgroup of WV waves takes 16 NB places by U blocks of 16 rows of the matrix (of two: 8 features
 * of each in a block, gates in rows 0 to 7, ups in rows 8 to 15, so few features still make enough
 * blocks). The waves share the columns: wave v takes chunks v, v + WV, ... of 64, D of them under way
 * at a time, operands straight from memory to registers; a chunk is a line of every row (of bf16). The
 * partial sums meet in LDS and are added in the order of the waves.
 *
 * What bounds it is memory: one row by 2 x 2048 x 7168 in bf16, 58.8 MB, in 14.6 us, 4.0 TB/s, of which
 * a call that does nothing takes 2; 24 rows by 3584 x 7168, 52 MB, in 19.9 us, 2.6 TB/s: the rows are
 * read again for every block of features, from the caches. */
#include <type_traits>

#include "k3g_linear.h"

template <bool GATED, typename TA, typename TB, int U, int WV, int NB, int D>
__global__ void __launch_bounds__(64 * WV)
k_ln_few(const LnArgs g, int ydt)
{
    constexpr int PA = ln_pieces<TA>, PB = ln_pieces<TB>, FB = GATED ? 8 : 16, FW = U * FB;
    __shared__ __attribute__((aligned(16))) k3v4f lds[WV * U * NB * 64];
    int ft, e, p0, np;
    if (!gm_row_item<16 * NB>(g.off, g.E, g.P, (g.NA + FW - 1) / FW, ft, e, p0, np)) return;
    const uint8_t *m1 = ln_matrix(g, g.a, e), *m3 = GATED ? ln_matrix(g, g.a3, e) : m1;
    if (!m1 || !m3) {
        if (ydt == K3_WBF16) ln_zeros<LN_FWD, GATED, uint16_t, 64 * WV>(g, (uint16_t *)g.y, p0, np, ft * FW, FW);
        else ln_zeros<LN_FWD, GATED, float, 64 * WV>(g, (float *)g.y, p0, np, ft * FW, FW);
        return;
    }
    const int lane = threadIdx.x & 63, wave = gm_uniform(threadIdx.x >> 6), c = lane & 15, q = lane >> 4;
    const int K = g.K, full = K >> 6, mine = full > wave ? (full - wave - 1) / WV + 1 : 0;
    const TA *w[U];
    const TB *x[NB];
    bool none[NB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        /* features past the last are read as the last one and never stored */
        const int f = min(ft * FW + u * FB + (c & (FB - 1)), g.NA - 1);
        w[u] = (const TA *)(GATED && c >= 8 ? m3 : m1) + (size_t)f * K;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int row = ln_row(g, p0 + min(16 * n + c, np - 1));
        none[n] = row < 0;
        x[n] = (const TB *)g.b + (size_t)max(row, 0) * K;
    }
    k3v4f acc[U][NB];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[u][n] = k3v4f{0.f, 0.f, 0.f, 0.f};
    LnUnit<TA> a[D][2][U];
    LnUnit<TB> b[D][2][NB];
    auto load = [&](int i, int d) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 64 * (wave + WV * i) + 32 * h + 8 * q;
#pragma unroll
            for (int u = 0; u < U; ++u) a[d][h][u] = ln_unit(w[u] + k, 8);
#pragma unroll
            for (int n = 0; n < NB; ++n) b[d][h][n] = ln_unit(x[n] + k, 8);
        }
    };
    auto sum = [&](int d) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            k3v8bf pb[NB][PB];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                gm_v4u p[PB];
                ln_split(b[d][h][n], p);
#pragma unroll
                for (int i = 0; i < PB; ++i)
                    pb[n][i] = __builtin_bit_cast(k3v8bf, none[n] ? gm_v4u{0, 0, 0, 0} : p[i]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                gm_v4u p[PA];
                k3v8bf pa[PA];
                ln_split(a[d][h][u], p);
#pragma unroll
                for (int i = 0; i < PA; ++i) pa[i] = __builtin_bit_cast(k3v8bf, p[i]);
#pragma unroll
                for (int n = 0; n < NB; ++n) ln_mma<PA, PB>(pa, pb[n], acc[u][n]);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (d < mine) load(d, d);
    for (int i = 0; i < mine; i += D)
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (i + d >= mine) break;
            sum(d);
            if (i + d + D < mine) load(i + d + D, d);
        }
    if ((K & 63) && wave == full % WV) {
        /* the columns past the last whole chunk */
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 64 * full + 32 * h + 8 * q;
#pragma unroll
            for (int u = 0; u < U; ++u) a[0][h][u] = ln_unit(w[u] + min(k, K - 1), K - k);
#pragma unroll
            for (int n = 0; n < NB; ++n) b[0][h][n] = ln_unit(x[n] + min(k, K - 1), K - k);
        }
        sum(0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < NB; ++n) lds[((wave * U + u) * NB + n) * 64 + lane] = acc[u][n];
    __syncthreads();
    auto total = [&](int i, int l) {
        k3v4f s = lds[i * 64 + l];
#pragma unroll
        for (int v = 1; v < WV; ++v) s += lds[(v * U * NB + i) * 64 + l];
        return s;
    };
    for (int i = wave; i < U * NB; i += WV) {
        const int u = i / NB, n = i - u * NB, col = ft * FW + u * FB + 4 * q, m = min(4, g.NA - col);
        if (16 * n + c >= np || m <= 0 || (GATED && q >= 2)) continue;
        const size_t at = (size_t)(p0 + 16 * n + c) * g.NA + col;
        const k3v4f v = total(i, lane), up = GATED ? total(i, lane + 32) : v;
        k3v4f bias = {0.f, 0.f, 0.f, 0.f}, bias3 = bias;
        if (g.bias) bias = ln_get4(g.bias + (size_t)e * g.NA + col, m);
        if (GATED && g.bias3) bias3 = ln_get4(g.bias3 + (size_t)e * g.NA + col, m);
        auto out = [&](auto *y) {
            using Y = std::remove_pointer_t<decltype(y)>;
            LnRead<LN_FWD, Y> r;
            ln_ask<LN_FWD, Y>(g, y, at, m, r);
            ln_finish<LN_FWD, GATED, Y>(g, y, at, m, v, up, bias, bias3, r);
        };
        if (ydt == K3_WBF16) out((uint16_t *)g.y);
        else out((float *)g.y);
    }
}

template <bool GATED, typename TA, typename TB, int U, int WV, int NB>
static int ln_few_run(const char *who, const LnArgs &g, int ydt, hipStream_t st)
{
    /* chunks under way: what their operands' registers allow */
    constexpr int REGS = 8 * (U * (int)sizeof(TA) / 2 + NB * (int)sizeof(TB) / 2), D = REGS <= 16 ? 6 : REGS <= 32 ? 4 : REGS <= 64 ? 2 : 1;
    const int fw = U * (GATED ? 8 : 16);
    const int64_t blocks = gm_row_items(g.off != nullptr, g.E, g.P, 16 * NB, (g.NA + fw - 1) / fw);
    if (blocks * 64 * WV > UINT32_MAX) {
        fprintf(stderr, "%s: %d rows by %d columns (%d experts) are more than a launch takes\n", who, g.P, g.NA, g.E);
        return -1;
    }
    return k3h_launch(who, k_ln_few<GATED, TA, TB, U, WV, NB, D>, dim3((unsigned)blocks), dim3(64 * WV), st, (LnArgs)g,
                      (int)ydt);
}

/* Row blocks, waves and blocks of places of a workgroup. us, bf16, weights not in the caches:
 *   U, WV, NB                       1, 8, 1   4, 4, 1   1, 8, 2   1, 8, 4
 *   1 x 7168 by 2 x 2048, gated     14.5      37.5      15.9      20.4
 *   1 x 2048 by 7168                8.7       12.4      9.6       13.9
 *   24 x 7168 by 3584               27.9      38.2      22.0      24.5
 * Experts of about a row each and not too many columns (64 x 2 x 1408 by 2048, 16 tokens x 6) take
 * four row blocks and four waves, 82 us against 151 with one and eight and 89 with tiles (8 tokens x 8 by 2 x
 * 2048 x 7168: 564, 569 and 515, so the columns count). */
template <bool GATED, typename TA, typename TB>
static int ln_few_t(const char *who, const LnArgs &g, int ydt, hipStream_t st)
{
    if (g.off) return ln_few_run<GATED, TA, TB, 4, 4, 1>(who, g, ydt, st);
    if (g.P <= 16) return ln_few_run<GATED, TA, TB, 1, 8, 1>(who, g, ydt, st);
    if (g.P <= 32) return ln_few_run<GATED, TA, TB, 1, 8, 2>(who, g, ydt, st);
    return ln_few_run<GATED, TA, TB, 1, 8, 4>(who, g, ydt, st);
}

/* Up to 16 rows, up to 32 by not too many features, up to 64 where the columns are few too: the rows are
 * read again for every 16 features. us, this kernel and the tiles of any types, bf16 and fp32:
 *   1, 16 rows, 7168 -> 7168       19.7 37.6, 28.0 37.5     49 110, 62 113
 *   1, 16 rows, 7168 -> 28672      72 96, 108 102           163 213, 213 219
 *   32 rows, 7168 -> 3584          22.0 23.0                45 71
 *   32 rows, 7168 -> 7168          39.8 39.5                86 115
 *   32 rows, 7168 -> 10240         65 48                    125 118
 *   32 rows, 4096 -> 32000         88 57                    200 141
 *   64 rows, 500 -> 500            5.9 7.6                  7.6 9.3
 *   64 rows, 1024 -> 4096          8.1 7.9                  13.9 13.7
 *   64 rows, 7168 -> 3584          34 22                    71 70 */
bool ln_few_takes(const LnArgs &g, int mode)
{
    if (mode != LN_FWD) return false;
    if (g.off) return g.P <= 2 * (g.E < g.P ? g.E : g.P) && g.K <= 4096;
    const int features = g.a3 ? 2 * g.NA : g.NA;
    return g.P <= 16 || (g.P <= 32 && features <= 8192) || (g.P <= 64 && features <= 4096 && g.K <= 1024);
}

template <bool GATED>
static int ln_few_m(const char *who, const LnArgs &g, int adt, int bdt, int ydt, hipStream_t st)
{
    if (adt == K3_WBF16)
        return bdt == K3_WBF16 ? ln_few_t<GATED, uint16_t, uint16_t>(who, g, ydt, st)
                               : ln_few_t<GATED, uint16_t, float>(who, g, ydt, st);
    return bdt == K3_WBF16 ? ln_few_t<GATED, float, uint16_t>(who, g, ydt, st)
                           : ln_few_t<GATED, float, float>(who, g, ydt, st);
}

int ln_run_few(const char *who, const LnArgs &g, bool gated, int adt, int bdt, int ydt, hipStream_t st)
{
    return gated ? ln_few_m<true>(who, g, adt, bdt, ydt, st) : ln_few_m<false>(who, g, adt, bdt, ydt, st);
}
