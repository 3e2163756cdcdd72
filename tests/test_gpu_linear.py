"""Products by matrices in plain rows, one or an expert's each, with what follows them, and their
gradients (k3g_matmul, k3g_grouped and their gradients, k3g_act_grad) against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest

import k3moe
import linear64 as L64
import ops64
from test_gpu_order import DT, Out, dev, floats, graphs, routing, rows_of

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16", "bf16"), ("bf16", "bf16", "f32"), ("f32", "bf16", "f32"), ("f32", "bf16", "bf16"),
         ("f32", "f32", "f32"), ("bf16", "f32", "f32")]


def whole(rng, *shape):
    """Whole numbers from -3 to 3: sums of their products are exact in fp32."""
    return rng.integers(-3, 4, shape).astype(np.float32)


def normal(rng, *shape):
    return rng.normal(0, 1, shape).astype(np.float32)


def stored(v, dt):
    """what an exact value becomes in dt"""
    return ops64.to_bf16(np.float32(v)) if dt == "bf16" else np.float32(v)


def table(mats, skew=0):
    """Matrices [E][..] as stored, NULL for None: their buffers and the address of their pointers"""
    bufs = [None if m is None else dev(m, skew) for m in mats]
    ptrs = np.array([0 if b is None else b[1].value for b in bufs], np.uint64)
    t = dev(ptrs)
    return (bufs, t), t[1]


def outs(shape, dt, skew=0, fill=None):
    o = Out(DT[dt][1], int(np.prod(shape)), skew)
    if fill is not None:
        o.buf.upload(np.ascontiguousarray(fill).view(np.uint8).reshape(-1), offset=skew)
    return o


def ranges(rng, E, P, kind):
    """off of P places among E experts; kind: how they share them"""
    if kind == "one":
        c = np.zeros(E, np.int64)
        c[E // 2] = P
    elif kind == "behind":                       # places behind the last one
        c = rng.multinomial(P - P // 4, np.ones(E) / E)
    elif kind == "none":
        c = np.zeros(E, np.int64)
    else:
        p = rng.random(E) ** 3
        p[::3] = 0
        c = rng.multinomial(P, p / p.sum())
    return np.concatenate([[0], np.cumsum(c)]).astype(np.int32)


class Forward:
    """One k3g_matmul or k3g_grouped (E > 0) call on given float32 values, and its 64-bit result."""

    def __init__(self, rng, rows, cols, n, types, act="none", E=0, topk=1, kind="", make=normal, bias=False,
                 residual=False, keep=False, caps=None, skew=0, null=(), inplace=False):
        self.types, self.act, self.E, self.n, self.skew = types, act, E, n, skew
        xdt, wdt, ydt = types
        self.caps = caps or (L64.UNCAPPED, L64.UNCAPPED)
        pair, P, M = act == "situ", rows * topk, max(E, 1)
        self.P, self.M, self.pair, self.rows, self.cols, self.topk = P, M, pair, rows, cols, topk
        self.x, xs = rows_of(make(rng, rows, cols), xdt)
        scale = 1.0 if make is whole else cols ** -0.5
        self.w, ws = zip(*[rows_of(make(rng, n, cols) * np.float32(scale), wdt) for _ in range(M)])
        self.w3, w3s = zip(*[rows_of(make(rng, n, cols) * np.float32(scale), wdt) for _ in range(M)]) if pair else (None, None)
        self.bias = make(rng, M, n) if bias else None
        self.bias3 = make(rng, M, n) if bias and pair else None
        self.res, ress = rows_of(make(rng, P, n), ydt) if residual else (None, None)
        self.off = ranges(rng, E, P, kind) if E else np.array([0, P], np.int32)
        self.kept = int(self.off[-1])
        self.pairs = rng.permutation(P).astype(np.int32) if E and topk > 1 else None
        self.null = null
        # ---- the call
        keepers = [dev(xs if rows else np.zeros(1, np.float32), skew)]
        ep = k3moe.K3gEpilogue()
        ep.act, ep.b1, ep.b2 = L64.ACTS.index(act), *self.caps

        def ptr(a):
            if a is None:
                return None
            keepers.append(dev(a, skew if a.dtype == np.uint16 else skew // 4 * 4))
            return keepers[-1][1].value

        ep.bias, ep.bias3 = ptr(self.bias), ptr(self.bias3)
        self.y = outs((P, n), ydt, skew, ress if inplace else None)
        ep.residual = self.y.ptr.value if inplace else ptr(ress)
        self.z = outs((P, n), ydt, skew) if keep else None
        self.z3 = outs((P, n), ydt, skew) if keep and pair else None
        ep.z, ep.z3 = (None if o is None else o.ptr.value for o in (self.z, self.z3))
        lib, tags = k3moe.lib(), [DT[t][0] for t in types]
        if E:
            t1, a1 = table([None if e in null else ws[e] for e in range(E)], skew)
            t3, a3 = table(list(w3s), skew) if pair else (None, None)
            off = dev(self.off)
            perm = None
            if self.pairs is not None:
                keepers.append(dev(self.pairs))
                perm = keepers[-1][1]
            rc = lib.k3g_grouped(keepers[0][1], tags[0], rows, cols, perm, topk, off[1], E, a1, a3, 8, tags[1], n,
                                 C.byref(ep), self.y.ptr, tags[2], None)
        else:
            rc = lib.k3g_matmul(keepers[0][1], tags[0], rows, cols, ptr(ws[0]), ptr(w3s[0]) if pair else None, tags[1],
                                n, C.byref(ep), self.y.ptr, tags[2], None)
        assert rc == 0
        k3moe.sync()

    def want(self):
        """z, z3, the sums' magnitudes, y (float64), of the kept places"""
        z, z3, size, size3 = [], [], [], []
        for e in range(self.M):
            a, b = (self.off[e], self.off[e + 1]) if self.E else (0, self.P)
            at = np.arange(a, b) if self.pairs is None else self.pairs[a:b] // self.topk
            x = self.x[at].astype(np.float64)
            for w, bias, out, mag in ((self.w, self.bias, z, size), (self.w3, self.bias3, z3, size3)):
                if w is None:
                    continue
                m = w[e].astype(np.float64)
                v, s = x @ m.T, np.abs(x) @ np.abs(m.T)
                if bias is not None:
                    v, s = v + bias[e], s + np.abs(bias[e])
                out.append(v)
                mag.append(s)
        z, size = np.concatenate(z), np.concatenate(size)
        z3, size3 = (np.concatenate(z3), np.concatenate(size3)) if self.pair else (None, None)
        y = L64.act(self.act, z, z3, *self.caps)
        if self.res is not None:
            y = y + self.res[:self.kept]
        return z, z3, size, size3, y

    def got(self, o):
        raw = o.get().reshape(self.P, self.n)
        assert np.all(raw[self.kept:].view(np.uint8) == 0x5A), "rows behind the last place"
        return raw[:self.kept]


SHAPES = [(1, 1, 1), (1, 7168, 64), (3, 40, 130), (17, 33, 5), (64, 512, 384), (127, 95, 129), (128, 128, 128),
          (129, 64, 136), (300, 1411, 709), (513, 264, 1024)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows,cols,n", SHAPES)
def test_matmul_whole_numbers(gpu, rows, cols, n, types):
    print(f"case: k3g_matmul {rows} x {cols} by {n}, {types}", flush=True)
    rng = np.random.default_rng(rows + cols + n)
    f = Forward(rng, rows, cols, n, types, "relu" if n % 2 else "none", make=whole, bias=True, residual=True, keep=True)
    z, _, _, _, y = f.want()
    assert np.array_equal(f.got(f.z), stored(z, types[2]))
    assert np.array_equal(f.got(f.y), stored(y, types[2]))


GROUPS = [(1, 64, 32, 5, 1), (1, 256, 48, 16, 8), (5, 100, 70, 8, 3), (64, 72, 128, 4, 2), (300, 136, 200, 7, 4),
          (1000, 31, 33, 64, 6), (40, 2048, 96, 300, 1)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("T,cols,n,E,topk", GROUPS)
def test_grouped_whole_numbers(gpu, T, cols, n, E, topk, types):
    print(f"case: k3g_grouped {T} x {topk} x {cols} by {E} of {n}, {types}", flush=True)
    rng = np.random.default_rng(T + cols + n)
    for kind in ("uneven", "behind", "one"):
        f = Forward(rng, T, cols, n, types, E=E, topk=topk, kind=kind, make=whole, bias=True, residual=True, keep=True)
        z, _, _, _, y = f.want()
        assert np.array_equal(f.got(f.z), stored(z, types[2])), kind
        assert np.array_equal(f.got(f.y), stored(y, types[2])), kind


@pytest.mark.parametrize("skew", [0, 4, 8])
@pytest.mark.parametrize("cols,n", [(64, 72), (65, 71), (66, 70)])
@pytest.mark.parametrize("types", [("bf16", "bf16", "bf16"), ("f32", "f32", "f32")])
def test_any_address(gpu, cols, n, types, skew):
    """Rows, matrices and outputs at addresses that only their elements have"""
    print(f"case: k3g_grouped at addresses {skew} past 16, {cols} x {n}, {types}", flush=True)
    rng = np.random.default_rng(cols + n)
    s = skew if types[0] == "f32" else skew // 2
    f = Forward(rng, 150, cols, n, types, "none", E=5, topk=2, make=whole, bias=True, residual=True, skew=s)
    assert np.array_equal(f.got(f.y), stored(f.want()[4], types[2]))


def close(got, want, bound, dt):
    """within bound of the value before its rounding to dt, and that rounding"""
    _, _, eps = DT[dt]
    err = np.abs(floats(got, dt).astype(np.float64) - want)
    tol = bound * (1 + eps) + eps * np.abs(want) + 2.0 ** -140
    bad = ~(err <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first {np.argwhere(bad)[0]}: {err[bad][0]} > {tol[bad][0]}"


def act_bound(f, z, z3, size, size3):
    """How far act(z, z3) may be off: the sums' bounds by the slopes' largest magnitudes around
    (1.2 and, of two products, their other factors), and the activation's own 2^-18 of its
    factors. gelu's erfc argument is rounded by 2^-23 of itself: up to z^2 2^-23 of the value."""
    t = f.cols + 2
    d = L64.sum_bound(t, size)
    if not f.pair:
        own = np.abs(z) * 2.0 ** -18 + np.abs(z) ** 3 * np.exp(-0.5 * z * z) * 2.0 ** -22
        return 1.2 * d + (own if f.act != "none" else 0)
    d3 = L64.sum_bound(t, size3)
    return 1.2 * d * (np.abs(z3) + d3) + (np.abs(z) + d) * d3 + np.abs(z * z3) * 2.0 ** -18


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("act", L64.ACTS)
def test_matmul_acts(gpu, act, types):
    print(f"case: k3g_matmul, {act}, {types}", flush=True)
    rng = np.random.default_rng(7)
    for rows, cols, n, caps in ((1, 320, 48, None), (70, 96, 144, (4.0, 25.0)), (150, 333, 91, (0.5, 2.0))):
        f = Forward(rng, rows, cols, n, types, act, bias=True, residual=True, keep=True, caps=caps)
        z, z3, size, size3, y = f.want()
        close(f.got(f.z), z, L64.sum_bound(cols + 2, size), types[2])
        if f.pair:
            close(f.got(f.z3), z3, L64.sum_bound(cols + 2, size3), types[2])
        close(f.got(f.y), y, act_bound(f, z, z3, size, size3) + 2.0 ** -24 * np.abs(y), types[2])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("T,cols,n,E,topk", [(1, 512, 64, 24, 8), (8, 1024, 48, 40, 6), (200, 160, 96, 6, 2),
                                             (333, 97, 61, 12, 3)])
def test_grouped_gated(gpu, T, cols, n, E, topk, types):
    print(f"case: k3g_grouped gated {T} x {topk} x {cols} by {E} of {n}, {types}", flush=True)
    rng = np.random.default_rng(T)
    for kind, caps in (("uneven", None), ("behind", (4.0, 25.0))):
        f = Forward(rng, T, cols, n, types, "situ", E=E, topk=topk, kind=kind, keep=True, caps=caps)
        z, z3, size, size3, y = f.want()
        close(f.got(f.z), z, L64.sum_bound(cols, size), types[2])
        close(f.got(f.z3), z3, L64.sum_bound(cols, size3), types[2])
        close(f.got(f.y), y, act_bound(f, z, z3, size, size3), types[2])


def test_residual_in_place(gpu):
    print("case: k3g_matmul onto its own output", flush=True)
    for types in TYPES:
        rng = np.random.default_rng(3)
        f = Forward(rng, 90, 120, 77, types, make=whole, residual=True, inplace=True)
        assert np.array_equal(f.got(f.y), stored(f.want()[4], types[2]))


@pytest.mark.parametrize("rows,cols,n", [(20, 64, 96), (300, 64, 96)])
def test_missing_matrices_give_zeros(gpu, rows, cols, n):
    print(f"case: k3g_grouped with experts without a matrix, {rows}", flush=True)
    rng = np.random.default_rng(11)
    f = Forward(rng, rows, cols, n, ("bf16", "bf16", "f32"), E=6, make=whole, bias=True, keep=True, null=(1, 4))
    y = f.want()[4]
    for e in f.null:
        y[f.off[e]:f.off[e + 1]] = 0
    assert np.array_equal(f.got(f.y), stored(y, "f32"))


# ------------------------------------------------------------------------ gradients ----

class BackX:
    def __init__(self, rng, rows, n, cols, types, E=0, kind="", make=normal, pair=False, add=False, act="none",
                 caps=None, skew=0, inplace=False):
        ddt, wdt, xdt = types
        self.types, self.rows, self.n, self.cols, self.E, self.act = types, rows, n, cols, E, act
        self.caps = caps or (L64.UNCAPPED, L64.UNCAPPED)
        M = max(E, 1)
        self.M = M
        self.off = ranges(rng, E, rows, kind) if E else np.array([0, rows], np.int32)
        self.kept = int(self.off[-1])
        scale = 1.0 if make is whole else n ** -0.5
        self.sets = []
        keep = []

        def ptr(a):
            if a is None:
                return None
            keep.append(dev(a, skew))
            return keep[-1][1].value

        args = []
        for _ in range(2 if pair else 1):
            d, ds = rows_of(make(rng, rows, n), ddt)
            w, ws = zip(*[rows_of(make(rng, n, cols) * np.float32(scale), wdt) for _ in range(M)])
            self.sets.append((d, w))
            if E:
                t, a = table(list(ws), skew)
                keep.append(t)
            else:
                a = ptr(ws[0])
            args.append((ptr(ds), a))
        args.append((None, None))
        self.add, adds = rows_of(make(rng, rows, cols), xdt) if add else (None, None)
        back = k3moe.K3gBack()
        self.dx = outs((rows, cols), xdt, skew, adds if inplace else None)
        back.add = self.dx.ptr.value if inplace else ptr(adds)
        self.dz3 = self.z3 = self.z = None
        if act != "none":
            back.act, back.b1, back.b2 = L64.ACTS.index(act), *self.caps
            self.z, zs = rows_of(make(rng, rows, cols) * 2, xdt)
            back.z = ptr(zs)
            if act == "situ":
                self.z3, z3s = rows_of(make(rng, rows, cols) * 2, xdt)
                back.z3 = ptr(z3s)
                self.dz3 = outs((rows, cols), xdt, skew)
                back.dz3 = self.dz3.ptr.value
        lib, tags = k3moe.lib(), [DT[t][0] for t in types]
        (d1, a1), (d3, a3) = args[:2]
        if E:
            off = dev(self.off)
            rc = lib.k3g_grouped_grad_x(d1, d3, tags[0], rows, n, off[1], E, a1, a3, 8, tags[1], cols, C.byref(back),
                                        self.dx.ptr, tags[2], None)
        else:
            rc = lib.k3g_matmul_grad_x(d1, d3, tags[0], rows, n, a1, a3, tags[1], cols, C.byref(back), self.dx.ptr,
                                       tags[2], None)
        assert rc == 0
        k3moe.sync()

    def want(self):
        g, size = np.zeros((self.kept, self.cols)), np.zeros((self.kept, self.cols))
        for d, w in self.sets:
            for e in range(self.M):
                r = slice(self.off[e], self.off[e + 1])
                g[r] += d[r].astype(np.float64) @ w[e]
                size[r] += np.abs(d[r].astype(np.float64)) @ np.abs(w[e])
        if self.add is not None:
            g += self.add[:self.kept]
            size += np.abs(self.add[:self.kept])
        return g, size

    def got(self, o):
        raw = o.get().reshape(self.rows, self.cols)
        assert np.all(raw[self.kept:].view(np.uint8) == 0x5A), "rows behind the last place"
        return raw[:self.kept]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows,n,cols,E", [(1, 1, 1, 0), (1, 640, 72, 0), (33, 65, 257, 0), (128, 128, 128, 0),
                                           (300, 709, 311, 0), (260, 200, 384, 0), (1, 32, 64, 9), (500, 72, 136, 6),
                                           (700, 33, 131, 40), (200, 512, 264, 3)])
def test_grad_x_whole_numbers(gpu, rows, n, cols, E, types):
    print(f"case: gradient of rows, {rows} x {n} by {cols}, {E} experts, {types}", flush=True)
    rng = np.random.default_rng(rows + n)
    for pair, add, kind in ((False, False, "uneven"), (True, True, "behind")):
        b = BackX(rng, rows, n, cols, types, E, kind, whole, pair, add)
        assert np.array_equal(b.got(b.dx), stored(b.want()[0], types[2]))


def test_grad_x_onto_its_output(gpu):
    print("case: gradient of rows added to its own output", flush=True)
    for types in TYPES:
        b = BackX(np.random.default_rng(2), 70, 80, 90, types, 0, "", whole, False, True, inplace=True)
        assert np.array_equal(b.got(b.dx), stored(b.want()[0], types[2]))


def slope_bound(act, z, z3, d, d3):
    """The slopes' own errors, in 2^-19 of their factors: sums of a few terms whose magnitudes
    are at most 1 + |z| (times the other factor)."""
    if act == "situ":
        return (2 + np.abs(z)) * np.abs(z3) * 2.0 ** -18, (1 + np.abs(z)) * 2.0 ** -18
    return (2 + np.abs(z)) * 2.0 ** -18, None


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("act", L64.ACTS[1:])
@pytest.mark.parametrize("E", [0, 5])
def test_grad_x_through_the_activation(gpu, E, act, types):
    print(f"case: gradient of rows through {act}, {E} experts, {types}", flush=True)
    rng = np.random.default_rng(9)
    for caps, (rows, n, cols) in ((None, (150, 96, 136)), ((4.0, 25.0), (90, 77, 61))):
        b = BackX(rng, rows, n, cols, types, E, "behind", normal, False, E == 0, act, caps)
        g, size = b.want()
        z = b.z[:b.kept].astype(np.float64)
        z3 = b.z3[:b.kept].astype(np.float64) if b.z3 is not None else None
        d, d3 = L64.slopes(act, z, z3, *b.caps)
        own, own3 = slope_bound(act, z, z3, d, d3)
        e = L64.sum_bound(n + 1, size)
        close(b.got(b.dx), g * d, e * np.abs(d) + (np.abs(g) + e) * own, types[2])
        if d3 is not None:
            close(b.got(b.dz3), g * d3, e * np.abs(d3) + (np.abs(g) + e) * own3, types[2])


class BackW:
    def __init__(self, rng, rows, n, cols, types, E=0, topk=1, kind="", make=whole, accumulate=0, bias=True, skew=0,
                 null=(), poison=False):
        ddt, xdt, wdt = types
        P, M = rows * topk, max(E, 1)
        self.types, self.n, self.cols, self.E, self.M, self.null = types, n, cols, E, M, null
        self.off = ranges(rng, E, P, kind) if E else np.array([0, P], np.int32)
        kept = int(self.off[-1])
        pairs = rng.permutation(P).astype(np.int32) if E and topk > 1 else None
        self.x, xs = rows_of(make(rng, rows, cols), xdt)
        self.d, ds = rows_of(make(rng, P, n), ddt)
        if poison:                               # rows that no expert has
            ds[kept:] = stored(np.nan, ddt)
            if pairs is None:
                xs[kept:] = stored(np.inf, xdt)
        self.old, olds = rows_of(make(rng, M, n, cols), wdt)
        self.oldb = make(rng, M, n)
        self.acc = accumulate
        self.dw = [outs((n, cols), wdt, skew, olds[e] if accumulate else None) for e in range(M)]
        self.db = outs((M, n), "f32", 0, self.oldb if accumulate else None) if bias else None
        self.at = np.arange(P) if pairs is None else pairs // topk
        lib, tags = k3moe.lib(), [DT[t][0] for t in types]
        dx, dd = dev(xs if rows else np.zeros(1), skew), dev(ds if rows else np.zeros(1), skew)
        db = None if self.db is None else self.db.ptr
        if E:
            t = dev(np.array([0 if e in null else self.dw[e].ptr.value for e in range(E)], np.uint64))
            off = dev(self.off)
            perm = dev(pairs) if pairs is not None else (None, None)
            rc = lib.k3g_grouped_grad_w(dd[1], tags[0], dx[1], tags[1], rows, n, cols, perm[1], topk, off[1], E,
                                        accumulate, t[1], 8, tags[2], db, None)
        else:
            rc = lib.k3g_matmul_grad_w(dd[1], tags[0], dx[1], tags[1], rows, n, cols, accumulate, self.dw[0].ptr,
                                       tags[2], db, None)
        assert rc == 0
        k3moe.sync()

    def want(self, e):
        r = slice(self.off[e], self.off[e + 1])
        d, x = self.d[r].astype(np.float64), self.x[self.at[r]].astype(np.float64)
        w, b, size = d.T @ x, d.sum(0), np.abs(d.T) @ np.abs(x)
        return (w + self.old[e], b + self.oldb[e], size) if self.acc else (w, b, size)

    def check(self):
        gb = None if self.db is None else self.db.get().reshape(self.M, self.n)
        for e in range(self.M):
            raw = self.dw[e].get().reshape(self.n, self.cols)
            if e in self.null:
                assert np.all(raw.view(np.uint8) == 0x5A) or self.acc
                continue
            w, b, _ = self.want(e)
            assert np.array_equal(raw, stored(w, self.types[2])), e
            if gb is not None:
                assert np.array_equal(gb[e], np.float32(b)), e


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows,n,cols,E,topk", [
    (0, 40, 33, 0, 1), (1, 1, 1, 0, 1), (1, 130, 140, 0, 1), (31, 64, 72, 0, 1), (300, 129, 260, 0, 1),
    (1000, 136, 128, 0, 1), (257, 61, 35, 0, 1), (0, 32, 40, 3, 1), (1, 64, 48, 5, 1), (400, 72, 136, 7, 1),
    (150, 264, 130, 5, 3), (90, 33, 41, 20, 6), (700, 128, 256, 3, 2)])
def test_grad_w_whole_numbers(gpu, rows, n, cols, E, topk, types):
    print(f"case: gradient of matrices, {rows} x {topk}, {n} x {cols}, {E} experts, {types}", flush=True)
    rng = np.random.default_rng(rows + n + cols)
    for acc, kind in ((0, "uneven"), (1, "behind"), (0, "one")):
        BackW(rng, rows, n, cols, types, E, topk, kind, accumulate=acc).check()


@pytest.mark.parametrize("topk", [1, 4])
def test_grad_w_rows_of_others_do_not_count(gpu, topk):
    """NaN and infinities in the rows behind the last place, and wanted and unwanted gradients"""
    print(f"case: gradient of matrices beside rows of NaN, topk {topk}", flush=True)
    for types in TYPES:
        rng = np.random.default_rng(4)
        BackW(rng, 203, 72, 136, types, 6, topk, "behind", poison=True, null=(2, 5)).check()


@pytest.mark.parametrize("types", TYPES)
def test_grad_w_random(gpu, types):
    print(f"case: gradient of matrices, normal values, {types}", flush=True)
    rng = np.random.default_rng(8)
    b = BackW(rng, 600, 70, 90, types, 4, 2, "uneven", normal)
    gb = b.db.get().reshape(b.M, b.n)
    for e in range(b.M):
        w, s, size = b.want(e)
        rows = int(b.off[e + 1] - b.off[e])
        close(b.dw[e].get().reshape(70, 90), w, L64.sum_bound(rows, size), types[2])
        close(gb[e], s, L64.sum_bound(rows, np.abs(b.d[b.off[e]:b.off[e + 1]].astype(np.float64)).sum(0)), "f32")


# -------------------------------------------------------------- through the activation ----

@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", L64.ACTS)
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 4095), (33, 257), (700, 1408)])
def test_act_grad(gpu, rows, n, act, dt):
    print(f"case: k3g_act_grad {rows} x {n}, {act}, {dt}", flush=True)
    rng = np.random.default_rng(rows + n)
    tag = DT[dt][0]
    for caps, skew in (((L64.UNCAPPED, L64.UNCAPPED), 0), ((4.0, 25.0), 4)):
        spread = np.exp2(rng.integers(-12, 6, (rows, n))).astype(np.float32)
        (h, hs), (z, zs), (z3, z3s) = (rows_of(normal(rng, rows, n) * s, dt) for s in (1, spread, spread))
        pair = act == "situ"
        dz, dz3 = outs((rows, n), dt, skew), outs((rows, n), dt, skew) if pair else None
        bh, bz, b3 = dev(hs, skew), dev(zs, skew), dev(z3s, skew)
        assert k3moe.lib().k3g_act_grad(bh[1], tag, rows, n, L64.ACTS.index(act), *caps, bz[1], b3[1] if pair else None,
                                        dz.ptr, dz3.ptr if pair else None, None) == 0
        k3moe.sync()
        h, z, z3 = (v.astype(np.float64) for v in (h, z, z3))
        d, d3 = L64.slopes(act, z, z3, *caps)
        own, own3 = slope_bound(act, z, z3, d, d3)
        close(dz.get().reshape(rows, n), h * d, np.abs(h) * own, dt)
        if pair:
            close(dz3.get().reshape(rows, n), h * d3, np.abs(h) * own3, dt)
