"""MXFP4 quantisation and products (k3g_quant_mxfp4, k3g_dequant_mxfp4, k3g_matmul_mxfp4,
k3g_grouped_mxfp4) against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest

import k3moe
import ops64
from test_gpu_order import DT, Out, dev, floats, graphs, routing, rows_of, sort_tokens

pytestmark = pytest.mark.gpu


def quantise(x, dt):
    """packed, scales of the call for x stored in dt"""
    tag, _, _ = DT[dt]
    rows, cols = x.shape
    b, p = dev(x)
    pk, sc = Out(np.uint8, rows * cols // 2), Out(np.uint8, rows * cols // 32)
    assert k3moe.lib().k3g_quant_mxfp4(p, tag, rows, cols, pk.ptr, sc.ptr, None) == 0
    k3moe.sync()
    return pk.get().reshape(rows, -1), sc.get().reshape(rows, -1)


def spread(rng, rows, cols, lo=-20, hi=20):
    """Normally distributed values, each block of 32 with a size of its own."""
    v = rng.normal(0, 1, (rows, cols // 32, 32)) * np.exp2(rng.integers(lo, hi + 1, (rows, cols // 32, 1)))
    return v.reshape(rows, cols).astype(np.float32)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 7168), (3, 96), (24, 1408), (257, 544), (1000, 2080)])
def test_quantise(gpu, dt, rows, cols):
    print(f"case: k3g_quant_mxfp4 {rows} x {cols}, {dt}", flush=True)
    rng = np.random.default_rng(rows + cols)
    x, xs = rows_of(spread(rng, rows, cols), dt)
    x[0, :32] = 0
    xs[0, :32] = 0
    pk, sc = quantise(xs, dt)
    code, scale = ops64.quant(x)
    assert np.array_equal(sc, scale)
    assert np.array_equal(ops64.unpack(pk), code)


def test_quantise_borders(gpu):
    """Every midpoint between two codes, its neighbours on both sides, signs, zeros of both signs,
    values past 6 units, subnormals and the largest values, infinities and NaN."""
    print("case: k3g_quant_mxfp4 at its borders", flush=True)
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], np.float32)
    near = np.concatenate([mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(9))])
    near = np.concatenate([near, -near, [0.0, -0.0, 2.0 ** -126, 7.9999995, 4.0]]).astype(np.float32)
    near = np.resize(near, (2, 32))
    near[:, 0] = 7.5                            # the block's unit is 1
    blocks = [near[0], near[1]]
    for e in (-149, -148, -140, -130, -127, -126, -125, -124, -100, 0, 100, 124, 125):
        for b in near:
            with np.errstate(over="ignore", under="ignore"):
                v = np.ldexp(b.astype(np.float64), e).astype(np.float32)
            blocks.append(np.where(np.isfinite(v), v, np.float32(1.0)))
    blocks += [np.zeros(32, np.float32), -np.zeros(32, np.float32), np.full(32, 2.0 ** -149, np.float32),
               np.full(32, np.finfo(np.float32).max, np.float32)]
    for bad in (np.inf, -np.inf, np.nan):
        v = np.ones(32, np.float32)
        v[len(blocks) % 32] = bad
        blocks.append(v)
    x = np.stack(blocks)
    pk, sc = quantise(x, "f32")
    code, scale = ops64.quant(x)
    assert np.array_equal(sc, scale)
    assert np.array_equal(ops64.unpack(pk), code)
    assert list(sc[-3:, 0]) == [255, 255, 255]
    xs = ops64.to_bf16(x)
    pk, sc = quantise(xs, "bf16")
    code, scale = ops64.quant(ops64.from_bf16(xs))
    assert np.array_equal(sc, scale)
    assert np.array_equal(ops64.unpack(pk), code)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_read_back(gpu, dt):
    """All 16 codes under all 256 scale bytes, and a second quantisation that changes nothing."""
    print(f"case: k3g_dequant_mxfp4, {dt}", flush=True)
    tag, store, eps = DT[dt]
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 6))
    scale = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 3))
    (bp, pp), (bs, ps) = dev(ops64.pack(code)), dev(scale)
    o = Out(store, code.size)
    assert k3moe.lib().k3g_dequant_mxfp4(pp, ps, 256, 96, o.ptr, tag, None) == 0
    k3moe.sync()
    raw = o.get().reshape(256, 96)
    got = floats(raw, dt).astype(np.float64)
    want = ops64.values(code, scale)
    # subnormal results round to nearest even of what dt holds: half of its smallest step
    half = 2.0 ** -150 if dt == "f32" else 2.0 ** -134
    assert np.all(np.isnan(got[255]))
    with np.errstate(over="ignore"):
        big = np.abs(want[:255]) > np.finfo(np.float32).max
    assert np.all(np.isinf(got[:255][big]))
    err = np.abs(got[:255] - want[:255])
    normal = np.abs(want[:255]) >= 2.0 ** -126
    assert np.all(err[normal & ~big] == 0)
    assert np.all(err[~normal] <= half)
    keep = slice(2, 250)
    pk, sc = quantise(raw[keep], dt)
    assert np.array_equal(sc, scale[keep])
    assert np.array_equal(ops64.unpack(pk), code[keep])


def tiled(pk, sc, n, cols):
    L = k3moe.lib()
    t = k3moe.DevBuf(L.k3g_tiled_mxfp4_bytes(n, cols))
    (bp, pp), (bs, ps) = dev(pk), dev(sc)
    assert L.k3g_tile_mxfp4(C.c_void_p(t.ptr), pp, ps, n, cols, None) == 0
    k3moe.sync()
    return t


def matrix(rng, n, cols, lo=110, hi=130):
    """random codes, scale bytes in [lo, hi]; and their values"""
    code = rng.integers(0, 16, (n, cols)).astype(np.uint8)
    scale = rng.integers(lo, hi + 1, (n, cols // 32)).astype(np.uint8)
    return ops64.pack(code), scale, ops64.values(code, scale)


def bound(xv, w):
    """Sum of the magnitudes of a product's terms, and how far fp32 sums of it may be off: the
    products of two codes are multiples of 1/4 up to 36, so those of a pair of blocks add up
    exactly; each of the cols / 32 block sums then joins a sum in fp32, off by at most 2^-23 of
    the magnitudes met (2^-24 rounded, twice that cut off), and up to 16 partial sums join."""
    mag = np.abs(xv) @ np.abs(w).T
    return mag, (xv.shape[1] // 32 + 16) * 2.0 ** -23 * mag


def activation(g, u, b1, b2):
    s = 1.0 / (1.0 + np.exp(-g))
    a = g * s if b1 >= 2.0 ** 64 else b1 * np.tanh(g / b1) * s
    return a * (u if b2 >= 2.0 ** 64 else b2 * np.tanh(u / b2))


def check(got, want, tol, dt):
    eps = DT[dt][2]
    bad = ~(np.abs(got - want) <= tol + eps * (np.abs(want) + tol) * (1 + 2.0 ** -7))
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


MATS = [(1, 32, 16), (1, 7168, 2048), (2, 544, 48), (3, 128, 4096), (4, 2048, 64), (5, 160, 80), (15, 1056, 272),
        (16, 512, 256), (17, 64, 16), (33, 4128, 208), (64, 1024, 512), (65, 2592, 1040), (129, 96, 336),
        (300, 1536, 640), (513, 576, 528), (500, 160, 6144), (512, 672, 7152), (1000, 160, 6096),
        (2000, 288, 7088)]


@pytest.mark.parametrize("rows,cols,n", MATS)
@pytest.mark.parametrize("xdt,ydt", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_matmul(gpu, rows, cols, n, xdt, ydt):
    print(f"case: k3g_matmul_mxfp4 {rows} x {cols} by {n}, {xdt} -> {ydt}", flush=True)
    rng = np.random.default_rng(rows * 3 + cols + n)
    x, xs = rows_of(spread(rng, rows, cols, -6, 6), xdt)
    pk, sc, w = matrix(rng, n, cols)
    L = k3moe.lib()
    bx, px = dev(xs)
    t = tiled(pk, sc, n, cols)
    size = L.k3g_mxfp4_work_bytes(rows, cols)
    work, y = Out(np.uint8, size), Out(DT[ydt][1], rows * n)
    assert L.k3g_matmul_mxfp4(px, DT[xdt][0], rows, cols, C.c_void_p(t.ptr), n, y.ptr, DT[ydt][0], work.ptr, size,
                              None) == 0
    k3moe.sync()
    work.get()
    got = floats(y.get(), ydt).reshape(rows, n).astype(np.float64)
    xv = ops64.values(*ops64.quant(x))
    check(got, xv @ w.T, bound(xv, w)[1], ydt)


def test_matmul_infinities(gpu):
    """A row with an infinity or a NaN is NaN, its neighbours are not."""
    print("case: k3g_matmul_mxfp4 with infinities", flush=True)
    L = k3moe.lib()
    for rows, n in ((3, 64), (40, 64), (500, 6144)):
        rng = np.random.default_rng(rows)
        x = rng.normal(0, 1, (rows, 1056)).astype(np.float32)
        x[1, 700], x[rows - 1, 1055] = np.inf, np.nan
        pk, sc, w = matrix(rng, n, 1056)
        bx, px = dev(x)
        t = tiled(pk, sc, n, 1056)
        size = L.k3g_mxfp4_work_bytes(rows, 1056)
        work, y = Out(np.uint8, size), Out(np.float32, rows * n)
        assert L.k3g_matmul_mxfp4(px, 0, rows, 1056, C.c_void_p(t.ptr), n, y.ptr, 0, work.ptr, size, None) == 0
        k3moe.sync()
        bad = np.isnan(y.get().reshape(rows, n))
        assert bad[1].all() and bad[rows - 1].all()
        bad[[1, rows - 1]] = False
        assert not bad.any()


def experts(rng, E, cols, n, count, lo=110, hi=130):
    """count tables of E tiled matrices: (buffers, pointer table, values) each"""
    out = []
    for _ in range(count):
        made = [matrix(rng, n, cols, lo, hi) for _ in range(E)]
        bufs = [tiled(pk, sc, n, cols) for pk, sc, _ in made]
        out.append((bufs, np.array([b.ptr for b in bufs], np.uint64), [m[2] for m in made]))
    return out


def grouped(x, xdt, perm, topk, off, tables, n, ydt, P, caps=(2.0 ** 100, 2.0 ** 100), step=8):
    L = k3moe.lib()
    rows, cols = x.shape
    (bx, px), (bo, po) = dev(x), dev(off.astype(np.int32))
    bp, pp = dev(perm.astype(np.int32)) if perm is not None else (None, None)
    ptr = [dev(t) for t in tables] + [(None, None)]
    size = L.k3g_mxfp4_work_bytes(rows, cols)
    work, y = Out(np.uint8, size), Out(DT[ydt][1], P * n)
    assert L.k3g_grouped_mxfp4(px, DT[xdt][0], rows, cols, pp, topk, po, off.size - 1, ptr[0][1], ptr[1][1], step, n,
                               caps[0], caps[1], y.ptr, DT[ydt][0], work.ptr, size, None) == 0
    k3moe.sync()
    work.get()
    return y.get().reshape(P, n)


GROUPS = [(1, 8, 16, 512, 64, 0.0), (3, 2, 5, 96, 48, 0.3), (8, 8, 24, 2048, 256, 0.0), (40, 1, 3, 1056, 80, 0.2),
          (64, 4, 7, 544, 304, 0.0), (100, 16, 40, 64, 16, 0.5), (600, 2, 3, 640, 272, 0.1), (5, 3, 1024, 32, 16, 0.0),
          (300, 4, 40, 1056, 1648, 0.1), (1500, 2, 24, 416, 2832, 0.0)]


@pytest.mark.parametrize("T,k,E,cols,n,drop", GROUPS)
@pytest.mark.parametrize("kind", ["tokens", "gated", "situ", "rows"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_grouped(gpu, T, k, E, cols, n, drop, kind, dt):
    print(f"case: k3g_grouped_mxfp4 {T} x {k} over {E}, {cols} -> {n}, {kind}, {dt}", flush=True)
    rng = np.random.default_rng(T + k + E + cols)
    idx = routing(rng, T, k, E, drop, same=(T == 40))
    perm, off, _ = ops64.order(idx, E)
    P, placed = T * k, perm.size
    full = np.full(P, -1)
    full[:placed] = perm
    by_token = kind != "rows"
    # gates of a few units, where the activation is neither linear nor flat
    x, xs = rows_of(spread(rng, T if by_token else P, cols, -3, 0), dt)
    caps = (4.0, 25.0) if kind == "situ" else (2.0 ** 100, 2.0 ** 100)
    mats = experts(rng, E, cols, n, 2 if kind in ("gated", "situ") else 1, 120, 123)
    raw = grouped(xs, dt, full if by_token else None, k if by_token else 1, off, [m[1] for m in mats], n, dt, P, caps)
    assert np.all(raw[placed:].view(np.uint8) == 0x5A), "rows behind the last place"
    got = floats(raw, dt).astype(np.float64)
    xv = ops64.values(*ops64.quant(x))
    row = perm // k if by_token else np.arange(placed)
    for e in range(E):
        r = slice(off[e], off[e + 1])
        if off[e] == off[e + 1]:
            continue
        a = xv[row[r]]
        want, (_, tol) = a @ mats[0][2][e].T, bound(a, mats[0][2][e])
        if len(mats) == 2:
            u, (_, tu) = a @ mats[1][2][e].T, bound(a, mats[1][2][e])
            g, tg = want, tol
            want = activation(g, u, *caps)
            # |d act / d gate| <= 1.25 |up|, |act| <= |gate| |up|; the activation itself, in fp32, has
            # two tanh (5 roundings of 2^-24 each in all), a sigmoid (5) and 5 products and quotients:
            # 20 of the 32 that 2^-19 is
            tol = 1.25 * tg * (np.abs(u) + tu) + np.abs(g) * tu + 2.0 ** -19 * np.abs(want)
        check(got[r], want, tol, dt)


def test_grouped_on_a_layers_table(gpu):
    """p1 and p3 of a K3ExpertQ table; an expert without matrices gives rows of zeros."""
    print("case: k3g_grouped_mxfp4 on a K3ExpertQ table", flush=True)
    rng = np.random.default_rng(2)
    T, k, E, cols, n = 20, 2, 4, 256, 64
    idx = routing(rng, T, k, E)
    perm, off, _ = ops64.order(idx, E)
    mats = experts(rng, E, cols, n, 2, 120, 123)
    x, xs = rows_of(spread(rng, T, cols, -3, 0), "f32")
    want = grouped(xs, "f32", perm, k, off, [m[1] for m in mats], n, "f32", T * k)
    table = np.zeros((E, 6), np.uint64)
    table[:, 0], table[:, 2] = mats[0][1], mats[1][1]
    table[2] = 0
    b, p = dev(table)
    L = k3moe.lib()
    (bx, px), (bo, po), (bp, pp) = dev(xs), dev(off.astype(np.int32)), dev(perm.astype(np.int32))
    size = L.k3g_mxfp4_work_bytes(T, cols)
    work, y = Out(np.uint8, size), Out(np.float32, T * k * n)
    assert L.k3g_grouped_mxfp4(px, 0, T, cols, pp, k, po, E, C.c_void_p(p.value), C.c_void_p(p.value + 16),
                               C.sizeof(k3moe.K3ExpertQ), n, 2.0 ** 100, 2.0 ** 100, y.ptr, 0, work.ptr, size, None) == 0
    k3moe.sync()
    got = y.get().reshape(T * k, n)
    want[off[2]:off[3]] = 0
    assert np.array_equal(got, want)


def test_grouped_ranges_and_pairs_out_of_range(gpu):
    """Ranges past the places are cut, a pair of no token reads a row of zeros."""
    print("case: k3g_grouped_mxfp4, off and perm out of range", flush=True)
    rng = np.random.default_rng(4)
    T, k, E, cols, n = 6, 2, 3, 64, 32
    mats = experts(rng, E, cols, n, 1)
    x, xs = rows_of(spread(rng, T, cols, -3, 0), "f32")
    perm = np.arange(T * k)
    perm[1], perm[5] = -7, 2 ** 31 - 1
    off = np.array([-4, 3, 2, 2 ** 31 - 1])
    got = grouped(xs, "f32", perm, k, off, [mats[0][1]], n, "f32", T * k).astype(np.float64)
    xv = ops64.values(*ops64.quant(x))
    a = np.zeros((T * k, cols))
    ok = (perm >= 0) & (perm // k < T)
    a[ok] = xv[perm[ok] // k]
    # expert 0 has places 0 to 2, expert 1 none (its end lies before its start), 2 from 2 on: each
    # value of the place that two claim is either's (both write it)
    for e, r in ((0, slice(0, 2)), (2, slice(3, T * k))):
        check(got[r], a[r] @ mats[0][2][e].T, bound(a[r], mats[0][2][e])[1], "f32")
    either = [np.abs(got[2] - a[2] @ mats[0][2][e].T) <= bound(a[2:3], mats[0][2][e])[1][0] + 1e-6 for e in (0, 2)]
    assert (either[0] | either[1]).all()


@pytest.mark.parametrize("T,E,n", [(3, 4, 32), (200, 4, 32), (400, 40, 1648)])
def test_grouped_without_pairs(gpu, T, E, n):
    """Every pair dropped: nothing is written."""
    print(f"case: k3g_grouped_mxfp4 without pairs, {T} tokens", flush=True)
    rng = np.random.default_rng(T)
    mats = experts(rng, E, 64, n, 2)
    x = rng.normal(0, 1, (T, 64)).astype(np.float32)
    raw = grouped(x, "f32", np.full(2 * T, -1), 2, np.zeros(E + 1, int), [m[1] for m in mats], n, "f32", 2 * T)
    assert np.all(raw.view(np.uint8) == 0x5A)


@pytest.mark.parametrize("T", [2, 70])
def test_expert_layer_in_four_bits(gpu, T):
    """A run of the operators as a program uses them: sort, gate and up of the tokens, down of the
    sorted rows, back with weights; weights quantised here."""
    print(f"case: an expert layer in MXFP4, {T} tokens", flush=True)
    rng = np.random.default_rng(T)
    k, E, d, inter = 4, 8, 512, 288
    L = k3moe.lib()
    idx = routing(rng, T, k, E, 0.1)
    wt = rng.random(T * k).astype(np.float32)
    x, xs = rows_of(rng.normal(0, 1, (T, d)), "bf16")
    tabs, vals, keep = [], [], []
    for rows, cols in ((inter, d), (inter, d), (d, inter)):
        t, v = [], []
        for _ in range(E):
            m, ms = rows_of(rng.normal(0, cols ** -0.5, (rows, cols)), "bf16")
            pk, sc = quantise(ms, "bf16")
            t.append(tiled(pk, sc, rows, cols))
            v.append(ops64.values(ops64.unpack(pk), sc))
        keep += t
        tabs.append(np.array([b.ptr for b in t], np.uint64))
        vals.append(v)
    perm, off, pos = sort_tokens(idx, E)
    h = grouped(xs, "bf16", perm, k, off, tabs[:2], inter, "f32", T * k)
    placed = off[-1]
    h[placed:] = 0
    y = grouped(h, "f32", None, 1, off, tabs[2:], d, "f32", T * k)
    y[placed:] = 0
    (by, py), (bp, pp), (bw, pw) = dev(y), dev(pos), dev(wt)
    o = Out(np.float32, T * d)
    assert L.k3g_unpermute(py, 0, T, k, d, pp, pw, None, o.ptr, None) == 0
    k3moe.sync()
    got = o.get().reshape(T, d).astype(np.float64)
    xv = ops64.values(*ops64.quant(x))
    hw, want, size = np.zeros((T * k, inter)), np.zeros((T, d)), np.zeros((T, d))
    for e in range(E):
        for r in range(off[e], off[e + 1]):
            a = xv[perm[r] // k]
            hw[r] = activation(vals[0][e] @ a, vals[1][e] @ a, 2.0 ** 100, 2.0 ** 100)
            # the second quantisation is checked on the h that the call gave
            assert np.all(np.abs(h[r] - hw[r]) <= 1e-5 * np.abs(hw[r]).max())
            q = ops64.values(*ops64.quant(h[r:r + 1]))[0]
            part = wt[perm[r]].astype(np.float64) * (vals[2][e] @ q)
            want[perm[r] // k] += part
            size[perm[r] // k] += wt[perm[r]] * (np.abs(vals[2][e]) @ np.abs(q))
    assert np.all(np.abs(got - want) <= (inter // 32 + 16 + k + 2) * 2.0 ** -23 * size)


@pytest.mark.parametrize("T", [3, 40, 700])
def test_captured_and_replayed(gpu, T):
    """Quantisation and the product inside it, gated and not, in a graph on a stream of its own, with
    new activations before each replay, against eager calls."""
    import torch
    print(f"case: captured products, {T} tokens", flush=True)
    L = k3moe.lib()
    k, E, cols, n = 2, 6, 1056, 272
    rng = np.random.default_rng(T)
    idx = torch.from_numpy(routing(rng, T, k, E, 0.1)).cuda()
    perm, off, _ = ops64.order(idx.cpu().numpy(), E)
    P = T * k
    full = np.full(P, -1, np.int32)
    full[:perm.size] = perm
    perm, off = torch.from_numpy(full).cuda(), torch.from_numpy(off.astype(np.int32)).cuda()
    mats = experts(rng, E, cols, n, 2, 120, 123)
    tab = [torch.from_numpy(m[1].astype(np.int64)).cuda() for m in mats]
    x = torch.empty(T, cols, device="cuda").normal_()
    size = L.k3g_mxfp4_work_bytes(T, cols)
    work = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    y = [torch.zeros(P, n, device="cuda") for _ in range(2)]
    z = [torch.zeros(T, n, device="cuda") for _ in range(2)]
    q = [torch.zeros(T, cols // 2 + cols // 32, dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()

    def run(st, i):
        assert L.k3g_grouped_mxfp4(x.data_ptr(), 0, T, cols, perm.data_ptr(), k, off.data_ptr(), E, tab[0].data_ptr(),
                                   tab[1].data_ptr(), 8, n, 4.0, 25.0, y[i].data_ptr(), 0, work[i].data_ptr(), size,
                                   st) == 0
        assert L.k3g_matmul_mxfp4(x.data_ptr(), 0, T, cols, int(mats[0][1][1]), n, z[i].data_ptr(), 0,
                                  work[i].data_ptr(), size, st) == 0
        assert L.k3g_quant_mxfp4(x.data_ptr(), 0, T, cols, q[i].data_ptr(), q[i].data_ptr() + T * cols // 2, st) == 0

    for _ in graphs(lambda st: run(st, 0)):
        run(None, 1)
        torch.cuda.synchronize()
        assert torch.equal(y[0], y[1]) and torch.equal(z[0], z[1]) and torch.equal(q[0], q[1])
        assert float(z[0].abs().max()) > 0
        x.normal_()
        y[0].zero_()
        z[0].zero_()
        torch.cuda.synchronize()


def test_two_products_at_once(gpu):
    """Two calls on two streams, each with a workspace of its own, give what they give alone."""
    import torch
    print("case: two products at once", flush=True)
    L = k3moe.lib()
    rows, cols, n = 600, 2048, 1024
    rng = np.random.default_rng(0)
    pk, sc, _ = matrix(rng, n, cols)
    t = tiled(pk, sc, n, cols)
    size = L.k3g_mxfp4_work_bytes(rows, cols)
    x = [torch.randn(rows, cols, device="cuda") for _ in range(2)]
    y = [torch.empty(rows, n, device="cuda") for _ in range(2)]
    alone = [torch.empty(rows, n, device="cuda") for _ in range(2)]
    work = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(2):
        assert L.k3g_matmul_mxfp4(x[i].data_ptr(), 0, rows, cols, t.ptr, n, alone[i].data_ptr(), 0, work[0].data_ptr(),
                                  size, None) == 0
        torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            assert L.k3g_matmul_mxfp4(x[i].data_ptr(), 0, rows, cols, t.ptr, n, y[i].data_ptr(), 0, work[i].data_ptr(),
                                      size, st[i].cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(y[0], alone[0]) and torch.equal(y[1], alone[1])


@pytest.mark.parametrize("rows", [1, 4, 5, 16, 40, 130, 257, 520])
def test_rows_do_not_meet(gpu, rows):
    """A row's product is the same bits whatever rows lie beside it in the call."""
    import torch
    print(f"case: rows of one call, {rows}", flush=True)
    L = k3moe.lib()
    cols, n = 3616, 1616
    rng = np.random.default_rng(rows)
    pk, sc, _ = matrix(rng, n, cols)
    t = tiled(pk, sc, n, cols)
    x = torch.randn(rows, cols, device="cuda")
    work = torch.empty(L.k3g_mxfp4_work_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    y = [torch.empty(rows, n, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for i, v in enumerate((x, x.flip(0).contiguous())):
        assert L.k3g_matmul_mxfp4(v.data_ptr(), 0, rows, cols, t.ptr, n, y[i].data_ptr(), 0, work.data_ptr(),
                                  work.numel(), None) == 0
        torch.cuda.synchronize()
    assert torch.equal(y[0], y[1].flip(0))


def test_values_past_32_bits(gpu):
    """More than 2^32 values quantised and read back: the last rows are the first rows' codes."""
    import torch
    print("case: values past 2^32", flush=True)
    L = k3moe.lib()
    rows, cols = 70000, 65536
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    block = torch.randn(100, cols, device="cuda").bfloat16()
    x.view(700, 100, cols)[:] = block
    pk = torch.empty(rows, cols // 2, dtype=torch.uint8, device="cuda")
    sc = torch.empty(rows, cols // 32, dtype=torch.uint8, device="cuda")
    assert L.k3g_quant_mxfp4(x.data_ptr(), 1, rows, cols, pk.data_ptr(), sc.data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert torch.equal(pk[:100], pk[-100:]) and torch.equal(sc[:100], sc[-100:])
    code, scale = ops64.quant(block[:3].float().cpu().numpy())
    assert np.array_equal(ops64.unpack(pk[-100:-97].cpu().numpy()), code)
    assert np.array_equal(sc[-100:-97].cpu().numpy(), scale)
    x.zero_()
    assert L.k3g_dequant_mxfp4(pk.data_ptr(), sc.data_ptr(), rows, cols, x.data_ptr(), 1, None) == 0
    torch.cuda.synchronize()
    assert np.array_equal(x[-100:-97].float().cpu().numpy(), ops64.values(code, scale))
    assert torch.equal(x[:100], x[-100:])


@pytest.mark.parametrize("caps", [(2.0 ** 100, 2.0 ** 100), (4.0, 25.0), (0.5, 2.0 ** 100), (2.0 ** 100, 3.0)])
def test_activation(gpu, caps):
    """The gated epilogue over gates and ups from far below to far above the caps: one column, so a
    row's gate and up are known exactly."""
    print(f"case: the gated product's activation, caps {caps}", flush=True)
    n = 16
    # x: one code a row and scale, gate weights 1, up weights -1 to 1.5 in code steps
    mags = np.array([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    col = np.concatenate([s * mags * 2.0 ** e for e in range(-30, 4) for s in (1.0, -1.0)])
    x = np.zeros((col.size, 32), np.float32)
    x[:, 0] = col
    gate, up = np.zeros((n, 32), np.uint8), np.zeros((n, 32), np.uint8)
    gate[:, 0] = 2                                  # 1.0
    up[:, 0] = np.arange(16)
    one = np.full((n, 1), 127, np.uint8)
    L = k3moe.lib()
    bufs = [tiled(ops64.pack(c), one, n, 32) for c in (gate, up)]
    tab = [np.array([b.ptr], np.uint64) for b in bufs]
    for rows in (2, col.size):
        raw = grouped(x[-rows:], "f32", np.arange(rows), 1, np.array([0, rows]), tab, n, "f32", rows, caps)
        g, u = col[-rows:, None] * np.ones(n), col[-rows:, None] * ops64.values(up, one)[:, 0]
        want = activation(g, u, *caps)
        assert np.all(np.abs(raw - want) <= 2.0 ** -19 * np.abs(want) + 2.0 ** -149), np.abs(raw / want - 1).max()


@pytest.mark.parametrize("caps", [(2.0 ** 100, 2.0 ** 100), (4.0, 25.0), (2.0 ** -100, 2.0 ** -100)])
def test_activation_far(gpu, caps):
    """Gates and ups far from zero: from a gate of -87 down the sigmoid is 0 whatever up is, so the
    result is off by all of the formula's; nothing becomes NaN."""
    print(f"case: the gated product's activation, large gates, caps {caps}", flush=True)
    mags = np.array([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    col = np.concatenate([[0.0]] + [s * mags * 2.0 ** e for e in range(4, 60) for s in (1.0, -1.0)])
    x = np.zeros((col.size, 32), np.float32)
    x[:, 0] = col
    code = np.zeros((2, 16, 32), np.uint8)
    code[0, :, 0], code[1, :, 0] = 2, np.arange(16)
    one = np.full((16, 1), 127, np.uint8)
    bufs = [tiled(ops64.pack(c), one, 16, 32) for c in code]
    tab = [np.array([b.ptr], np.uint64) for b in bufs]
    raw = grouped(x, "f32", np.arange(col.size), 1, np.array([0, col.size]), tab, 16, "f32", col.size, caps)
    g, u = col[:, None] * np.ones(16), col[:, None] * ops64.values(code[1], one)[:, 0]
    with np.errstate(over="ignore"):
        want = activation(g, u, *caps)
    tol = np.where(g <= -87, 1.0, 2.0 ** -19) * np.abs(want) + 2.0 ** -149
    assert np.all(np.abs(raw - want) <= tol), np.argwhere(~(np.abs(raw - want) <= tol))[:4]
