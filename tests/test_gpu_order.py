"""Tokens in expert order and back (k3g_sort_tokens, k3g_permute, k3g_unpermute and their
gradients) against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest

import k3moe
import ops64

pytestmark = pytest.mark.gpu

GUARD = 64                      # bytes past an output's end that must stay as they were


class Out:
    """An output of n elements, filled with a pattern, with a guard behind it and `skew` bytes
    of misalignment before it."""

    def __init__(self, dtype, n, skew=0):
        self.dtype, self.n, self.skew = np.dtype(dtype), n, skew
        self.bytes = n * self.dtype.itemsize
        self.fill = np.full(skew + self.bytes + GUARD, 0x5A, np.uint8)
        self.buf = k3moe.DevBuf.from_array(self.fill)
        self.ptr = C.c_void_p(self.buf.ptr + skew)

    def get(self):
        raw = self.buf.download(np.uint8, self.fill.size)
        assert np.array_equal(raw[:self.skew], self.fill[:self.skew]), "written before the output"
        assert np.array_equal(raw[self.skew + self.bytes:], self.fill[:GUARD]), "written behind the output"
        return raw[self.skew:self.skew + self.bytes].copy().view(self.dtype)


def dev(a, skew=0):
    a = np.ascontiguousarray(a)
    b = k3moe.DevBuf(a.nbytes + skew + 16)
    b.upload(a.view(np.uint8).reshape(-1), offset=skew)
    return b, C.c_void_p(b.ptr + skew)


def rows_of(a, dt):
    """float32 values of an array stored in dt, and the array to store"""
    if dt == "bf16":
        b = ops64.to_bf16(a)
        return ops64.from_bf16(b), b
    return a.astype(np.float32), a.astype(np.float32)


DT = {"f32": (k3moe.K3_WF32, np.float32, 2.0 ** -24), "bf16": (k3moe.K3_WBF16, np.uint16, 2.0 ** -8)}


def floats(out, dt):
    return ops64.from_bf16(out) if dt == "bf16" else out


def routing(rng, T, k, E, drop=0.0, same=False):
    idx = np.argsort(rng.random((T, E)), axis=1)[:, :k] if E >= k and T * E < 1 << 22 else \
        rng.integers(0, E, (T, k))
    if same:
        idx[:] = idx[:, :1]                     # every slot of a token on the same expert
    idx = idx.astype(np.int32)
    if drop:
        idx[rng.random((T, k)) < drop] = -1
    return np.ascontiguousarray(idx)


def sort_tokens(idx, E, want_err=0):
    T, k = idx.shape
    P = T * k
    L = k3moe.lib()
    b, p = dev(idx if P else np.zeros(1, np.int32))
    perm, off, pos = Out(np.int32, P), Out(np.int32, E + 1), Out(np.int32, P)
    err = k3moe.DevBuf.from_array(np.zeros(1, np.int32))
    n = L.k3g_sort_bytes(T, k, E)
    work = Out(np.uint8, n)
    assert L.k3g_sort_tokens(p, T, k, E, perm.ptr, off.ptr, pos.ptr, C.c_void_p(err.ptr), work.ptr, n, None) == 0
    k3moe.sync()
    work.get()
    assert err.download(np.int32, 1)[0] == want_err
    return perm.get(), off.get(), pos.get()


@pytest.mark.parametrize("T,k,E", [(0, 8, 384), (1, 1, 1), (1, 16, 896), (4, 8, 384), (63, 1, 3), (9, 7, 64),
                                   (64, 8, 256), (513, 8, 1024), (511, 8, 1024), (4097, 1, 2),
                                   (700, 6, 64), (4096, 8, 384), (5000, 64, 64), (70001, 1, 1000),
                                   (1025, 1, 40), (2049, 1, 1024), (16385, 8, 300), (131073, 8, 500)])
@pytest.mark.parametrize("kind", ["all", "dropped", "one expert", "none"])
def test_sort(gpu, T, k, E, kind):
    print(f"case: k3g_sort_tokens {T} x {k} over {E}, {kind}", flush=True)
    rng = np.random.default_rng(T * 131 + k + E)
    idx = routing(rng, T, k, E, 0.2 if kind == "dropped" else 0.0)
    if kind == "one expert":
        idx[:] = E - 1
    if kind == "none":
        idx[:] = -1 - (np.arange(idx.size).reshape(idx.shape) % 3)
    perm, off, pos = sort_tokens(idx, E)
    wperm, woff, wpos = ops64.order(idx, E)
    assert np.array_equal(off, woff)
    assert np.array_equal(perm[:wperm.size], wperm)
    assert np.all(perm[wperm.size:].view(np.uint8) == 0x5A), "entries behind the last place"
    assert np.array_equal(pos, wpos)


@pytest.mark.parametrize("T,k", [(3, 8), (2000, 8)])
def test_sort_reports_experts_out_of_range(gpu, T, k):
    print(f"case: k3g_sort_tokens with an expert out of range, {T} x {k}", flush=True)
    idx = routing(np.random.default_rng(5), T, k, 64)
    idx[T // 2, 3] = 64
    idx[T - 1, 0] = 2 ** 31 - 1
    perm, off, pos = sort_tokens(idx, 64, want_err=1)
    wperm, woff, wpos = ops64.order(idx, 64)
    assert np.array_equal(off, woff) and np.array_equal(perm[:wperm.size], wperm)
    assert np.array_equal(pos, wpos)


SIZES = [(1, 1, 1), (1, 16, 3584), (2, 3, 7), (3, 2, 8), (5, 8, 1411), (5, 1, 255), (17, 6, 257), (33, 4, 64),
         (7, 64, 40), (64, 8, 2048), (3, 8, 7168), (300, 5, 129)]


def case(T, k, n, dt, drop, seed=3, place_rows=True):
    rng = np.random.default_rng(seed + T * 7 + k + n)
    idx = routing(rng, T, k, max(k, 16), drop, same=(n == 64))
    _, off, pos = ops64.order(idx, max(k, 16))
    v = lambda *s: rows_of(rng.normal(0, 1, s), dt)
    return rng, pos.astype(np.int32), int(off[-1]), v


@pytest.mark.parametrize("T,k,n", SIZES)
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("skew", [0, 1])
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_permute(gpu, T, k, n, dt, skew, drop):
    print(f"case: k3g_permute {T} x {k}, width {n}, {dt}, skew {skew}, drop {drop}", flush=True)
    tag, store, eps = DT[dt]
    skew *= np.dtype(store).itemsize
    rng, pos, placed, v = case(T, k, n, dt, drop)
    P = T * k
    (x, xs), (g, gs) = v(T, n), v(P, n)
    L = k3moe.lib()
    bp, pp = dev(pos)
    bx, px = dev(xs, skew)
    s = Out(store, P * n, skew)
    assert L.k3g_permute(px, tag, T, k, n, pp, s.ptr, None) == 0
    k3moe.sync()
    got = s.get().reshape(P, n)
    token = np.repeat(np.arange(T), k)
    want = got.copy()
    want[pos[pos >= 0]] = xs[token[pos >= 0]]
    assert np.array_equal(got, want)
    assert np.all(got[placed:].view(np.uint8) == 0x5A), "rows behind the last place"
    # the gradient; a dropped pair's row would be NaN
    gs = gs.copy()
    gs[placed:] = np.array([np.nan], np.float32).view(np.uint32)[0] >> 16 if dt == "bf16" else np.nan
    bg, pg = dev(gs, skew)
    dx = Out(store, T * n, skew)
    assert L.k3g_permute_grad(pg, tag, T, k, n, pp, dx.ptr, None) == 0
    k3moe.sync()
    got = floats(dx.get(), dt).reshape(T, n).astype(np.float64)
    want, size = np.zeros((T, n)), np.zeros((T, n))
    for p in np.flatnonzero(pos >= 0):
        want[token[p]] += g[pos[p]].astype(np.float64)
        size[token[p]] += np.abs(g[pos[p]])
    # k additions in fp32, each off by 2^-24 of a partial sum of at most `size`, and the rounding
    assert np.all(np.abs(got - want) <= k * 2.0 ** -24 * size + eps * np.abs(want) * (1 + 2.0 ** -7))


@pytest.mark.parametrize("T,k,n", SIZES)
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("skew", [0, 1])
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_unpermute(gpu, T, k, n, dt, skew, drop):
    print(f"case: k3g_unpermute {T} x {k}, width {n}, {dt}, skew {skew}, drop {drop}", flush=True)
    tag, store, eps = DT[dt]
    skew *= np.dtype(store).itemsize
    rng, pos, placed, v = case(T, k, n, dt, drop)
    P = T * k
    (s, ss), (a, as_), (g, gs) = v(P, n), v(T, n), v(T, n)
    wt = rng.random(P).astype(np.float32)
    wt[pos < 0] = np.nan                       # a dropped pair's weight is never used
    ss = ss.copy()
    ss[placed:] = np.array([np.inf], np.float32).view(np.uint32)[0] >> 16 if dt == "bf16" else np.inf
    L = k3moe.lib()
    (bp, pp), (bs, ps), (ba, pa), (bg, pg), (bw, pw) = (dev(pos), dev(ss, skew), dev(as_, skew), dev(gs, skew),
                                                        dev(wt))
    token = np.repeat(np.arange(T), k)
    kept = np.flatnonzero(pos >= 0)
    for add in (False, True):
        out = Out(store, T * n, skew)
        assert L.k3g_unpermute(ps, tag, T, k, n, pp, pw, pa if add else None, out.ptr, None) == 0
        k3moe.sync()
        got = floats(out.get(), dt).reshape(T, n).astype(np.float64)
        want, size = np.zeros((T, n)), np.zeros((T, n))
        for p in kept:
            r = wt[p].astype(np.float64) * s[pos[p]]
            want[token[p]] += r
            size[token[p]] += np.abs(r)
        if add:
            want += a
            size += np.abs(a)
        # a product's rounding, then k + 1 additions, then the output's
        assert np.all(np.abs(got - want) <= (k + 2) * 2.0 ** -24 * size + eps * np.abs(want) * (1 + 2.0 ** -7))
    ds, dw = Out(store, P * n, skew), Out(np.float32, P)
    assert L.k3g_unpermute_grad(pg, ps, tag, T, k, n, pp, pw, ds.ptr, dw.ptr, None) == 0
    k3moe.sync()
    got, gotw = ds.get().reshape(P, n), dw.get()
    assert np.all(got[placed:].view(np.uint8) == 0x5A), "rows behind the last place"
    wantw = np.zeros(P)
    for p in kept:
        exact = wt[p].astype(np.float64) * g[token[p]]
        assert np.all(np.abs(floats(got[pos[p]], dt) - exact) <= (eps + 2.0 ** -24) * np.abs(exact))
        prod = s[pos[p]].astype(np.float64) * g[token[p]]
        wantw[p] = prod.sum()
        # n products and additions in fp32: the classical bound, any order
        assert abs(gotw[p] - wantw[p]) <= (n + 1) * 2.0 ** -24 * np.abs(prod).sum()
    assert np.all(gotw[pos < 0] == 0)
    # one gradient at a time gives the same bits
    ds1, dw1 = Out(store, P * n, skew), Out(np.float32, P)
    assert L.k3g_unpermute_grad(pg, None, tag, T, k, n, pp, pw, ds1.ptr, None, None) == 0
    assert L.k3g_unpermute_grad(pg, ps, tag, T, k, n, pp, None, None, dw1.ptr, None) == 0
    k3moe.sync()
    assert np.array_equal(ds1.get().reshape(P, n), got)
    assert np.array_equal(dw1.get(), gotw)


def test_places_out_of_range_are_left_out(gpu):
    print("case: places past the pairs", flush=True)
    T, k, n = 3, 2, 40
    pos = np.array([0, 6, 1, -2 ** 31, 2, 2 ** 31 - 1], np.int32)
    x = np.arange(T * n, dtype=np.float32).reshape(T, n) + 1
    L = k3moe.lib()
    (bp, pp), (bx, px) = dev(pos), dev(x)
    s = Out(np.float32, T * k * n)
    assert L.k3g_permute(px, k3moe.K3_WF32, T, k, n, pp, s.ptr, None) == 0
    k3moe.sync()
    rows = s.get().reshape(T * k, n)
    assert np.array_equal(rows[:3], x) and np.all(rows[3:].view(np.uint8) == 0x5A)
    bs, ps = dev(rows)
    o = Out(np.float32, T * n)
    bw, pw = dev(np.full(T * k, 0.5, np.float32))
    assert L.k3g_unpermute(ps, k3moe.K3_WF32, T, k, n, pp, pw, None, o.ptr, None) == 0
    k3moe.sync()
    assert np.array_equal(o.get().reshape(T, n), 0.5 * x)


def test_unpermute_is_the_layers_combine(gpu):
    """fp32 rows: bit for bit what k3g_combine gives on the same rows in pair order."""
    print("case: k3g_unpermute against k3g_combine", flush=True)
    T, k, n, E = 37, 8, 256, 16
    rng = np.random.default_rng(9)
    idx = routing(rng, T, k, E, 0.2)
    perm, off, pos = ops64.order(idx, E)
    contrib = rng.normal(0, 1, (T * k, n)).astype(np.float32)
    wt, add = rng.random(T * k).astype(np.float32), rng.normal(0, 1, (T, n)).astype(np.float32)
    s = np.zeros_like(contrib)
    s[:perm.size] = contrib[perm]
    (bi, pi), (bc, pc), (bs, ps), (bw, pw), (ba, pa), (bp, pp) = (dev(idx), dev(contrib), dev(s), dev(wt), dev(add),
                                                                 dev(pos.astype(np.int32)))
    L = k3moe.K3gLayer()
    L.hidden = L.latent = L.inter = n
    L.n_experts, L.topk = E, k
    ctx = k3moe.Ctx(L, max_tokens=T)
    a, b = Out(np.float32, T * n), Out(np.float32, T * n)
    ctx.combine(pc.value, pi.value, pw.value, T, k, n, pa.value, a.ptr.value)
    ctx.sync()
    assert k3moe.lib().k3g_unpermute(ps, k3moe.K3_WF32, T, k, n, pp, pw, pa, b.ptr, None) == 0
    k3moe.sync()
    assert np.array_equal(a.get().view(np.uint32), b.get().view(np.uint32))
    ctx.destroy()


def test_gradients_against_differences(gpu):
    """d<out, dout> / d(row element, weight, token element) against the gradients: the calls are
    linear in each, so a difference of any size is exact but for rounding."""
    print("case: gradients against differences", flush=True)
    T, k, n, E = 5, 3, 24, 6
    rng = np.random.default_rng(11)
    idx = routing(rng, T, k, E, 0.2)
    P = T * k
    pos = ops64.order(idx, E)[2].astype(np.int32)
    placed = int((pos >= 0).sum())
    x, g = rng.normal(0, 1, (T, n)).astype(np.float32), rng.normal(0, 1, (T, n)).astype(np.float32)
    wt = rng.random(P).astype(np.float32)
    L = k3moe.lib()
    bp, pp = dev(pos)

    def there_and_back(x, wt):
        (bx, px), (bw, pw) = dev(x), dev(wt)
        s, o = Out(np.float32, P * n), Out(np.float32, T * n)
        assert L.k3g_permute(px, k3moe.K3_WF32, T, k, n, pp, s.ptr, None) == 0
        assert L.k3g_unpermute(s.ptr, k3moe.K3_WF32, T, k, n, pp, pw, None, o.ptr, None) == 0
        k3moe.sync()
        return s, float((o.get().reshape(T, n).astype(np.float64) * g).sum())

    s, base = there_and_back(x, wt)
    (bg, pg), (bw, pw) = dev(g), dev(wt)
    ds, dw, dx = Out(np.float32, P * n), Out(np.float32, P), Out(np.float32, T * n)
    assert L.k3g_unpermute_grad(pg, s.ptr, k3moe.K3_WF32, T, k, n, pp, pw, ds.ptr, dw.ptr, None) == 0
    assert L.k3g_permute_grad(ds.ptr, k3moe.K3_WF32, T, k, n, pp, dx.ptr, None) == 0
    k3moe.sync()
    dw, dx = dw.get(), dx.get().reshape(T, n)
    # outputs of size ~ 3 rounded to 2^-24 each, T n of them against g of ~ 1: below 1e-5 in all
    tol = 2e-5
    for p in rng.integers(0, P, 6):
        w2 = wt.copy()
        w2[p] += 1.0
        assert abs(there_and_back(x, w2)[1] - base - dw[p]) < tol
    for _ in range(6):
        t, i = rng.integers(0, T), rng.integers(0, n)
        x2 = x.copy()
        x2[t, i] += 1.0
        assert abs(there_and_back(x2, wt)[1] - base - dx[t, i]) < tol
    assert placed < P


def graphs(capture, steps=3):
    """Captures `capture(stream)` on a stream of its own and replays it with eager work of the
    program and synchronizations in between; yields after each replay."""
    import torch
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        capture(st.cuda_stream)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        capture(st.cuda_stream)
    other = torch.ones(1 << 16, device="cuda")
    for _ in range(steps):
        with torch.cuda.stream(st):
            g.replay()
        other = other * 1.5 + 1.0
        st.synchronize()
        torch.cuda.synchronize()
        yield


@pytest.mark.parametrize("T,k,n,E", [(3, 8, 100, 24), (900, 8, 72, 64)])
def test_captured_and_replayed(gpu, T, k, n, E):
    """Sort, rows out, back with weights and every gradient in one graph, on a stream that is not
    the default one, with new routing, rows and weights before each replay."""
    import torch
    print(f"case: a captured run of {T} x {k}", flush=True)
    L, P = k3moe.lib(), T * k
    gen = torch.Generator(device="cuda")
    gen.manual_seed(T)
    dev_ = dict(device="cuda")
    x, g = torch.empty(T, n, **dev_), torch.empty(T, n, **dev_)
    idx, wt = torch.empty(T, k, dtype=torch.int32, **dev_), torch.empty(T, k, **dev_)

    def fresh():
        x.normal_(generator=gen)
        g.normal_(generator=gen)
        wt.uniform_(generator=gen)
        i = torch.topk(torch.rand(T, E, generator=gen, **dev_), k, dim=1).indices.int()
        idx.copy_(torch.where(torch.rand(T, k, generator=gen, **dev_) < 0.1, -1, i))
        torch.cuda.synchronize()

    perm, pos = torch.empty(P, dtype=torch.int32, **dev_), torch.empty(P, dtype=torch.int32, **dev_)
    off = torch.empty(E + 1, dtype=torch.int32, **dev_)
    nw = L.k3g_sort_bytes(T, k, E)
    work = torch.empty(max(nw, 1), dtype=torch.uint8, **dev_)
    s, ds = torch.zeros(P, n, **dev_), torch.zeros(P, n, **dev_)
    out, dw, dx = torch.empty(T, n, **dev_), torch.empty(P, **dev_), torch.empty(T, n, **dev_)

    def capture(st):
        assert L.k3g_sort_tokens(idx.data_ptr(), T, k, E, perm.data_ptr(), off.data_ptr(), pos.data_ptr(), None,
                                 work.data_ptr(), nw, st) == 0
        assert L.k3g_permute(x.data_ptr(), 0, T, k, n, pos.data_ptr(), s.data_ptr(), st) == 0
        assert L.k3g_unpermute(s.data_ptr(), 0, T, k, n, pos.data_ptr(), wt.data_ptr(), None, out.data_ptr(), st) == 0
        assert L.k3g_unpermute_grad(g.data_ptr(), s.data_ptr(), 0, T, k, n, pos.data_ptr(), wt.data_ptr(),
                                    ds.data_ptr(), dw.data_ptr(), st) == 0
        assert L.k3g_permute_grad(ds.data_ptr(), 0, T, k, n, pos.data_ptr(), dx.data_ptr(), st) == 0

    fresh()
    for _ in graphs(capture):
        kept = idx.cpu().numpy().reshape(-1) >= 0
        assert np.array_equal(pos.cpu().numpy(), ops64.order(idx.cpu().numpy(), E)[2])
        w64 = np.where(kept, wt.cpu().numpy().reshape(-1).astype(np.float64), 0.0).reshape(T, k)
        xn, gn = x.cpu().numpy().astype(np.float64), g.cpu().numpy().astype(np.float64)
        tol = (2 * k + 4) * 2.0 ** -24
        assert np.all(np.abs(out.cpu().numpy() - w64.sum(1)[:, None] * xn) <= tol * w64.sum(1)[:, None] * np.abs(xn))
        assert np.all(np.abs(dx.cpu().numpy() - w64.sum(1)[:, None] * gn) <= tol * w64.sum(1)[:, None] * np.abs(gn))
        dots = np.where(kept.reshape(T, k), (xn * gn).sum(1)[:, None], 0.0)
        assert np.all(np.abs(dw.cpu().numpy().reshape(T, k) - dots) <= (n + 1) * 2.0 ** -24 * np.abs(xn * gn).sum(1)[:, None])
        fresh()


def test_two_sorts_at_once(gpu):
    """Two calls on two streams, each with a workspace of its own, do not meet."""
    import torch
    print("case: two sorts at once", flush=True)
    L = k3moe.lib()
    T, k, E = 6000, 8, 200
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for i in range(2):
        idx = torch.from_numpy(routing(np.random.default_rng(i), T, k, E, 0.1)).cuda()
        perm, pos = (torch.empty(T * k, dtype=torch.int32, device="cuda") for _ in range(2))
        off = torch.empty(E + 1, dtype=torch.int32, device="cuda")
        work = torch.empty(L.k3g_sort_bytes(T, k, E), dtype=torch.uint8, device="cuda")
        runs.append((idx, perm, off, pos, work))
    torch.cuda.synchronize()
    for _ in range(10):
        for (idx, perm, off, pos, work), s in zip(runs, st):
            assert L.k3g_sort_tokens(idx.data_ptr(), T, k, E, perm.data_ptr(), off.data_ptr(), pos.data_ptr(), None,
                                     work.data_ptr(), work.numel(), s.cuda_stream) == 0
    torch.cuda.synchronize()
    for idx, perm, off, pos, _ in runs:
        wp, wo, wpos = ops64.order(idx.cpu().numpy(), E)
        assert np.array_equal(off.cpu().numpy(), wo) and np.array_equal(pos.cpu().numpy(), wpos)
        assert np.array_equal(perm.cpu().numpy()[:wp.size], wp)


def test_rows_past_32_bits(gpu):
    """Sorted rows of more than 2^32 elements (and 8 GB): the last ones go out and come back."""
    import torch
    print("case: sorted rows past 2^32 elements", flush=True)
    T, k, n = 33000, 2, 65600
    L, P = k3moe.lib(), T * k
    assert P * n > 1 << 32
    pos = torch.arange(P, dtype=torch.int32, device="cuda").flip(0).contiguous()
    x = (torch.arange(T, device="cuda", dtype=torch.int32) % 251).to(torch.bfloat16).unsqueeze(1).expand(T, n).contiguous()
    x[:, -1] = 3.0
    s = torch.empty(P, n, dtype=torch.bfloat16, device="cuda")
    wt = torch.full((P,), 0.5, device="cuda")
    assert L.k3g_permute(x.data_ptr(), 1, T, k, n, pos.data_ptr(), s.data_ptr(), None) == 0
    torch.cuda.synchronize()
    for r in (0, 1, P // 2, P - 2, P - 1):
        assert torch.equal(s[r], x[(P - 1 - r) // k])
    out = torch.empty_like(x)
    assert L.k3g_unpermute(s.data_ptr(), 1, T, k, n, pos.data_ptr(), wt.data_ptr(), None, out.data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, x)                  # two halves of the same value
    dw = torch.empty(P, device="cuda")
    out.fill_(1.0)
    assert L.k3g_unpermute_grad(out.data_ptr(), s.data_ptr(), 1, T, k, n, pos.data_ptr(), wt.data_ptr(), s.data_ptr(),
                                None, None) == 0
    assert L.k3g_unpermute_grad(out.data_ptr(), x.data_ptr(), 1, 1, 1, n, pos[P - 1:].data_ptr(), None, None,
                                dw.data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert bool((s[0] == 0.5).all()) and bool((s[P - 1] == 0.5).all()) and bool((s[P // 2] == 0.5).all())
    assert float(dw[0]) == 3.0                  # token 0's row is zeros but for its last element
