/* k3g_groups.h - which rows of which expert a workgroup of a grouped product takes. */
#pragma once

#include "k3g_dev.h"

#define GM_MAX_EXPERTS 1024

/* Row tile `item` of up to TM of the P places of E experts (off NULL: of one, all of them): expert,
 * first place and count; false past the last. Every wave finds it by itself: a lane takes up to 16
 * experts, all their ranges asked for at once, a wave scan of the lanes' tile counts finds the lane
 * that has it. The ranges are clamped to the places there are, whatever off holds. */
template <int TM>
__device__ __forceinline__ bool gm_row_tile(const int32_t *off, int E, int P, int item, int &e, int &p0,
                                            int &np)
{
    if (!off) {
        e = 0;
        p0 = item * TM;
        np = min(TM, P - p0);
        return np > 0;
    }
    const int lane = threadIdx.x & 63;
    constexpr int MOST = GM_MAX_EXPERTS / 64;
    const int per = (E + 63) >> 6, e0 = lane * per;
    int at[MOST + 1], n = 0;
#pragma unroll
    for (int i = 0; i <= MOST; ++i)
        if (i <= per) at[i] = off[min(e0 + i, E)];
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        if (i >= per) continue;
        at[i] = min(max(at[i], 0), P);
        n += (min(max(at[i + 1], at[i]), P) - at[i] + TM - 1) / TM;
    }
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d, K3G_WAVE);
        if (lane >= d) inc += o;
    }
    const uint64_t past = __ballot(inc > item);
    if (!past) return false;
    int left = item - (inc - n), fe = 0, fp = 0, fn = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        if (i >= per) continue;
        const int rows = min(max(at[i + 1], at[i]), P) - at[i], t = (rows + TM - 1) / TM;
        if (left >= 0 && left < t) {
            fe = e0 + i;
            fp = at[i] + left * TM;
            fn = min(TM, rows - left * TM);
        }
        left -= t;
    }
    const int L = __ffsll((unsigned long long)past) - 1;
    e = __builtin_amdgcn_readlane(fe, L);
    p0 = __builtin_amdgcn_readlane(fp, L);
    np = __builtin_amdgcn_readlane(fn, L);
    return true;
}

/* Workgroup b runs on XCD b % 8. One matrix: each XCD takes an eighth of the (feature tile, row
 * tile) pairs in bands of 8 row tiles, so the 64 that run on it at a time are about 8 x 8 and read
 * a sixteenth of what they would alone from past its L2. Experts: the feature tiles are dealt to the
 * XCDs one by one, each with two row tiles one after the other, so an expert's second row tile
 * finds its weights in that L2, and a few experts still fill every XCD. */
template <int TM>
__device__ __forceinline__ bool gm_row_item(const int32_t *off, int E, int P, int nft, int &ft, int &e,
                                            int &p0, int &np)
{
    const int xcd = blockIdx.x & 7, s = blockIdx.x >> 3;
    if (!off) {
        const int tiles = (P + TM - 1) / TM, items = tiles * nft, per = (items + 7) / 8;
        const int i = xcd * per + s;
        if (s >= per || i >= items) return false;
        const int band = i / (8 * nft), in = i - band * 8 * nft, wide = min(8, tiles - 8 * band);
        ft = in / wide;
        return gm_row_tile<TM>(off, E, P, 8 * band + in - ft * wide, e, p0, np);
    }
    const int i = 8 * (s >> 1) + xcd, pair = i / nft;
    ft = i - pair * nft;
    return gm_row_tile<TM>(off, E, P, 2 * pair + (s & 1), e, p0, np);
}

/* as many workgroups as gm_row_item may be asked for: row tiles of tm places by nft feature tiles */
static inline int64_t gm_row_items(bool grouped, int E, int P, int tm, int64_t nft)
{
    if (!grouped) return ((P + (int64_t)tm - 1) / tm * nft + 7) / 8 * 8;
    const int64_t tiles = P / tm + (E < P ? E : P);
    return ((tiles + 1) / 2 * nft + 7) / 8 * 16;
}
