"""Products with weights of one's own as programs use them: a layer's experts there and back, captured
graphs, calls at once on several streams, pairs that are none, extreme values, rows and outputs past 32
bits."""
import ctypes as C
import math

import numpy as np
import pytest

import k3moe
import linear64 as L64
from test_gpu_order import DT, graphs

pytestmark = pytest.mark.gpu

UNCAPPED = 2.0 ** 100


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def table(t):
    """the device address of the pointers to t[0], t[1], ..."""
    import torch
    return t.data_ptr() + t.stride(0) * t.element_size() * torch.arange(t.shape[0], device="cuda")


def tag(t):
    import torch
    return k3moe.K3_WBF16 if t.dtype == torch.bfloat16 else k3moe.K3_WF32


def ok(rc):
    assert rc == 0


class Experts:
    """Tokens through experts of one's own and back, every buffer made beforehand."""

    def __init__(self, T, topk, E, d, n, dtype, caps, gen):
        import torch
        self.T, self.k, self.E, self.d, self.n, self.caps = T, topk, E, d, n, caps
        new = lambda *s, **a: torch.randn(*s, device="cuda", generator=gen, **a)
        self.x, self.dout = new(T, d).to(dtype), new(T, d).to(dtype)
        self.w1, self.w3 = (new(E, n, d).mul_(d ** -0.5).to(dtype) for _ in range(2))
        self.w2 = new(E, d, n).mul_(n ** -0.5).to(dtype)
        self.wt = torch.rand(T, topk, device="cuda", generator=gen)
        self.idx = torch.empty(T, topk, dtype=torch.int32, device="cuda")
        P = T * topk
        i32 = dict(dtype=torch.int32, device="cuda")
        self.perm, self.pos, self.off = torch.full((P,), -1, **i32), torch.empty(T, topk, **i32), torch.empty(E + 1, **i32)
        self.work = torch.empty(max(k3moe.lib().k3g_sort_bytes(T, topk, E), 1), dtype=torch.uint8, device="cuda")
        zero = lambda *s, dt=dtype: torch.zeros(*s, dtype=dt, device="cuda")
        self.z, self.z3, self.h, self.dh, self.du = (zero(P, n) for _ in range(5))
        self.y, self.dy, self.dxs = (zero(P, d) for _ in range(3))
        self.out, self.dx = zero(T, d), zero(T, d)
        self.dwt = zero(T, topk, dt=torch.float32)
        self.dw1, self.dw3, self.dw2 = (zero(*w.shape, dt=torch.float32) for w in (self.w1, self.w3, self.w2))
        self.tables = [table(t) for t in (self.w1, self.w3, self.w2, self.dw1, self.dw3, self.dw2)]
        self.ep, self.back = k3moe.K3gEpilogue(), k3moe.K3gBack()
        self.ep.act, self.ep.b1, self.ep.b2 = k3moe.K3G_ACT_SITU, *caps
        self.ep.z, self.ep.z3 = ptr(self.z), ptr(self.z3)
        self.back.act, self.back.b1, self.back.b2 = k3moe.K3G_ACT_SITU, *caps
        self.back.z, self.back.z3, self.back.dz3 = ptr(self.z), ptr(self.z3), ptr(self.du)
        self.route(gen)

    def route(self, gen, drop=0.1):
        import torch
        i = torch.topk(torch.rand(self.T, self.E, generator=gen, device="cuda"), self.k, dim=1).indices.int()
        lost = torch.rand(self.T, self.k, generator=gen, device="cuda") < drop
        self.idx.copy_(torch.where(lost, -1, i))

    def run(self, st):
        L, T, k, E, d, n = k3moe.lib(), self.T, self.k, self.E, self.d, self.n
        P, t, f32 = T * k, tag(self.x), k3moe.K3_WF32
        w1, w3, w2, g1, g3, g2 = (v.data_ptr() for v in self.tables)
        ok(L.k3g_sort_tokens(ptr(self.idx), T, k, E, ptr(self.perm), ptr(self.off), ptr(self.pos), None, ptr(self.work),
                             self.work.numel(), st))
        ok(L.k3g_grouped(ptr(self.x), t, T, d, ptr(self.perm), k, ptr(self.off), E, w1, w3, 8, t, n, C.byref(self.ep),
                         ptr(self.h), t, st))
        ok(L.k3g_grouped(ptr(self.h), t, P, n, None, 1, ptr(self.off), E, w2, None, 8, t, d, None, ptr(self.y), t, st))
        ok(L.k3g_unpermute(ptr(self.y), t, T, k, d, ptr(self.pos), ptr(self.wt), None, ptr(self.out), st))
        ok(L.k3g_unpermute_grad(ptr(self.dout), ptr(self.y), t, T, k, d, ptr(self.pos), ptr(self.wt), ptr(self.dy),
                                ptr(self.dwt), st))
        ok(L.k3g_grouped_grad_w(ptr(self.dy), t, ptr(self.h), t, P, d, n, None, 1, ptr(self.off), E, 0, g2, 8, f32, None, st))
        ok(L.k3g_grouped_grad_x(ptr(self.dy), None, t, P, d, ptr(self.off), E, w2, None, 8, t, n, C.byref(self.back),
                                ptr(self.dh), t, st))
        ok(L.k3g_grouped_grad_x(ptr(self.dh), ptr(self.du), t, P, n, ptr(self.off), E, w1, w3, 8, t, d, None,
                                ptr(self.dxs), t, st))
        ok(L.k3g_grouped_grad_w(ptr(self.dh), t, ptr(self.x), t, T, n, d, ptr(self.perm), k, ptr(self.off), E, 0, g1, 8, f32,
                                None, st))
        ok(L.k3g_grouped_grad_w(ptr(self.du), t, ptr(self.x), t, T, n, d, ptr(self.perm), k, ptr(self.off), E, 0, g3, 8, f32,
                                None, st))
        ok(L.k3g_permute_grad(ptr(self.dxs), t, T, k, d, ptr(self.pos), ptr(self.dx), st))

    def results(self):
        return {k: getattr(self, k) for k in ("out", "dx", "dwt", "dw1", "dw3", "dw2")}

    def loss64(self, x, w1, w3, w2, wt):
        """The layer's outputs and sum(out * dout) in 64 bits, a token and slot at a time by expert"""
        import torch
        b1, b2 = self.caps
        cap = lambda v, b: v if b >= 2.0 ** 64 else b * torch.tanh(v / b)
        out = torch.zeros(self.T, self.d, dtype=torch.float64, device="cuda")
        for e in range(self.E):
            t, j = torch.nonzero(self.idx == e, as_tuple=True)
            if t.numel():
                g, u = x[t] @ w1[e].t(), x[t] @ w3[e].t()
                h = cap(g, b1) * torch.sigmoid(g) * cap(u, b2)
                out = out.index_add(0, t, wt[t, j].unsqueeze(1) * (h @ w2[e].t()))
        return out, (out * self.dout.double()).sum()


@pytest.mark.parametrize("T,k,E,d,n", [(40, 3, 7, 96, 56), (33, 2, 5, 71, 45), (700, 4, 6, 264, 136)])
def test_a_layer_of_ones_own_experts(gpu, T, k, E, d, n):
    """fp32 throughout, against the 64-bit formula's results and gradients, and those against
    differences of the 64-bit loss. The products' sums are off by less than (6 K + 16) 2^-24 of their
    magnitudes' sum (linear64.sum_bound), the activation by 2^-18: over four products in a row, normal
    values and the norm of many values, 2^-15 is more than all of it."""
    import torch
    print(f"case: experts there and back, {T} x {k} over {E}, {d} x {n}", flush=True)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(T)
    for caps in ((UNCAPPED, UNCAPPED), (4.0, 25.0)):
        m = Experts(T, k, E, d, n, torch.float32, caps, gen)
        m.run(stream())
        leaves = [v.double().requires_grad_() for v in (m.x, m.w1, m.w3, m.w2, m.wt)]
        out, loss = m.loss64(*leaves)
        loss.backward()
        got = m.results()
        want = dict(out=out.detach(), dx=leaves[0].grad, dw1=leaves[1].grad, dw3=leaves[2].grad, dw2=leaves[3].grad,
                    dwt=leaves[4].grad)
        for key, v in want.items():
            rel = ((got[key].double() - v).norm() / v.norm()).item()
            assert rel < 2.0 ** -15, (key, rel)
        # the formula against differences, along one direction for all leaves
        eps = 1e-5
        way = [torch.randn(v.shape, dtype=torch.float64, device="cuda", generator=gen) for v in leaves]
        with torch.no_grad():
            up = m.loss64(*[v + eps * s for v, s in zip(leaves, way)])[1]
            down = m.loss64(*[v - eps * s for v, s in zip(leaves, way)])[1]
        slope = sum((v.grad * s).sum() for v, s in zip(leaves, way))
        assert abs(((up - down) / (2 * eps) - slope).item()) < 1e-6 * abs(slope.item()) + 1e-5


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,k,E,d,n", [(3, 2, 9, 136, 64), (300, 2, 3, 520, 1032)])
def test_captured_and_replayed(gpu, T, k, E, d, n, dtype):
    import torch
    print(f"case: a captured layer and its gradients, {T} x {k} over {E}, {d} x {n}, {dtype}", flush=True)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(T + d)
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    m = Experts(T, k, E, d, n, dt, (UNCAPPED, UNCAPPED), gen)

    def fresh():
        m.route(gen)
        for v in (m.x, m.dout):
            v.copy_(torch.randn(v.shape, device="cuda", generator=gen))
        torch.cuda.synchronize()

    for _ in graphs(m.run, steps=4):
        got = {key: v.clone() for key, v in m.results().items()}
        m.run(stream())
        torch.cuda.synchronize()
        for key, v in m.results().items():
            assert torch.equal(got[key], v), key
        fresh()


def test_streams_at_once(gpu):
    """The same layers on four streams, twice each, give what they give one after the other"""
    import torch
    print("case: layers on four streams at once", flush=True)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    shapes = [(300, 2, 3, 520, 1032, torch.bfloat16), (40, 3, 7, 96, 56, torch.float32), (4, 8, 64, 1024, 256, torch.bfloat16),
              (617, 2, 9, 71, 45, torch.float32)]
    layers = [Experts(*s, (4.0, 25.0), gen) for s in shapes]
    alone = []
    for m in layers:
        m.run(stream())
        torch.cuda.synchronize()
        alone.append({key: v.clone() for key, v in m.results().items()})
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(2):
        for m, st in zip(layers, streams):
            for v in m.results().values():
                v.zero_()
        torch.cuda.synchronize()
        for m, st in zip(layers, streams):
            m.run(st.cuda_stream)
        torch.cuda.synchronize()
        for m, want in zip(layers, alone):
            for key, v in m.results().items():
                assert torch.equal(v, want[key]), key


@pytest.mark.parametrize("T,topk,E,K,n,dtype", [(3, 2, 4, 136, 72, "bf16"), (40, 3, 4, 71, 45, "f32"), (200, 2, 3, 64, 200, "bf16"),
                                                (500, 3, 4, 72, 6000, "bf16")])
def test_pairs_that_are_none(gpu, T, topk, E, K, n, dtype):
    """perm entries outside the pairs are rows of zeros, and add nothing to a gradient; off past the
    places ends at them."""
    import torch
    print(f"case: pairs that are none, {T} x {topk} x {K} by {E} of {n}, {dtype}", flush=True)
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    gen = torch.Generator(device="cuda")
    gen.manual_seed(T)
    P = T * topk
    whole = lambda *s: torch.randint(-3, 4, s, device="cuda", generator=gen).to(dt)
    x, w, dy = whole(T, K), whole(E, n, K), whole(P, n)
    perm = torch.randperm(P, device="cuda", generator=gen).int()
    gone = torch.rand(P, device="cuda", generator=gen) < 0.2
    perm = torch.where(gone, torch.where(torch.arange(P, device="cuda") % 2 == 0, -1, P + 5).int(), perm)
    cuts = torch.sort(torch.randint(0, P + 1, (E - 1,), device="cuda", generator=gen)).values
    off = torch.cat([torch.zeros(1, device="cuda"), cuts.float(), torch.tensor([P + 9.0], device="cuda")]).int()
    bias = torch.randint(-3, 4, (E, n), device="cuda", generator=gen).float()
    y, dw = torch.zeros(P, n, device="cuda"), torch.zeros(E, n, K, device="cuda")
    ep = k3moe.K3gEpilogue()
    ep.bias = ptr(bias)
    L, t, tw, td = k3moe.lib(), tag(x), table(w), table(dw)
    ok(L.k3g_grouped(ptr(x), t, T, K, ptr(perm), topk, ptr(off), E, ptr(tw), None, 8, t, n, C.byref(ep), ptr(y), 0, stream()))
    ok(L.k3g_grouped_grad_w(ptr(dy), t, ptr(x), t, T, n, K, ptr(perm), topk, ptr(off), E, 0, ptr(td), 8, 0, None, stream()))
    rows = x.double()[perm.clamp(0, P - 1).long() // topk] * (~gone).double().unsqueeze(1)
    o = off.clamp(max=P).tolist()
    for e in range(E):
        a, b = o[e], o[e + 1]
        assert torch.equal(y[a:b].double(), rows[a:b] @ w[e].double().t() + bias[e].double())
        assert torch.equal(dw[e].double(), dy[a:b].double().t() @ rows[a:b])


def test_extremes(gpu):
    """fp32 values near the largest and near the smallest that are held in three pieces, infinities and
    NaN: each row's outputs are its own."""
    import torch
    print("case: extreme values", flush=True)
    L = k3moe.lib()
    for K, n in ((64, 48), (70, 33)):
        for rows in (4, 200):
            x = torch.zeros(rows, K, device="cuda")
            w = torch.eye(n, K, device="cuda")
            x[:, :n] = torch.randn(rows, n, device="cuda")
            x[0, :n] = 3.4e38 * torch.sign(x[0, :n])
            x[1, :n] *= 2.0 ** -100
            x[2, 3], x[2, 5], x[2, 7] = math.inf, -math.inf, math.nan
            for wdt in (torch.float32, torch.bfloat16):
                wm, y = w.to(wdt), torch.empty(rows, n, device="cuda")
                ok(L.k3g_matmul(ptr(x), 0, rows, K, ptr(wm), None, tag(wm), n, None, ptr(y), 0, stream()))
                keep = torch.ones(rows, dtype=torch.bool, device="cuda")
                keep[2] = False
                # one product of 1 a sum: the pieces give the value back, all 24 bits
                assert torch.equal(y[keep], x[keep][:, :n])
                assert not torch.isfinite(y[2, [3, 5, 7]]).any()
    # infinities by bf16 matrices without zeros are infinities
    x, w = torch.ones(3, 64, device="cuda"), torch.ones(32, 64, device="cuda", dtype=torch.bfloat16)
    x[1, 9], x[2, 9] = math.inf, -math.inf
    for xx in (x, x.bfloat16()):
        y = torch.empty(3, 32, device="cuda")
        ok(L.k3g_matmul(ptr(xx), tag(xx), 3, 64, ptr(w), None, 1, 32, None, ptr(y), 0, stream()))
        assert (y[0] == 64).all() and (y[1] == math.inf).all() and (y[2] == -math.inf).all()


def test_activations_at_their_ends(gpu):
    """Values far out: the activations and slopes reach 0, z or 1 without NaN."""
    import torch
    print("case: activations far out", flush=True)
    L = k3moe.lib()
    z = torch.tensor([-3e38, -1e20, -1e4, -300.0, -100.0, -60.0, 60.0, 100.0, 300.0, 1e4, 1e20, 3e38], device="cuda")
    one = torch.ones_like(z)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        a = L64.ACTS.index(act)
        dz, y = torch.empty_like(z), torch.empty_like(z)
        ok(L.k3g_act_grad(ptr(one), 0, 1, z.numel(), a, 0.0, 0.0, ptr(z), None, ptr(dz), None, stream()))
        ep = k3moe.K3gEpilogue()
        ep.act = a
        ok(L.k3g_matmul(ptr(z), 0, z.numel(), 1, ptr(one), None, 0, 1, C.byref(ep), ptr(y), 0, stream()))
        assert torch.allclose(dz, (z > 0).float(), rtol=0, atol=2.0 ** -22), act
        assert torch.equal(y[6:], z[6:]) and (y[:6].abs() < 2.0 ** -60).all(), act


def test_past_32_bits(gpu):
    """Gathered rows of 4.6 GB, outputs of 4.6 GB, and gradients' rows of 4.6 GB"""
    import torch
    print("case: rows and outputs past 32 bits", flush=True)
    L, bf = k3moe.lib(), torch.bfloat16
    T, K = 320000, 7168
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randint(-3, 4, (T, K), device="cuda", generator=gen, dtype=torch.int8).to(bf)
    E, n = 2, 40
    w = torch.randint(-3, 4, (E, n, K), device="cuda", generator=gen).to(bf)
    perm = torch.randperm(T, device="cuda", generator=gen).int()
    off = torch.tensor([0, T // 3, T], device="cuda", dtype=torch.int32)
    y = torch.empty(T, n, device="cuda")
    for p in (perm, None):
        ok(L.k3g_grouped(ptr(x), 1, T, K, ptr(p), 1, ptr(off), E, ptr(table(w)), None, 8, 1, n, None, ptr(y), 0, stream()))
        at = torch.cat([torch.arange(0, T, 9973, device="cuda"), torch.arange(T - 70, T, device="cuda")])
        rows = x[(p.long() if p is not None else torch.arange(T, device="cuda"))[at]].double()
        want = torch.where((at < T // 3).unsqueeze(1), rows @ w[0].double().t(), rows @ w[1].double().t())
        assert torch.equal(y[at].double(), want)
    # x's gradient rows, 7168 wide: dx = dy W, and W's from all rows
    dy, dx = torch.randint(-1, 2, (T, 8), device="cuda", generator=gen).to(bf), torch.empty_like(x)
    wg = torch.randint(-3, 4, (8, K), device="cuda", generator=gen).to(bf)
    ok(L.k3g_matmul_grad_x(ptr(dy), None, 1, T, 8, ptr(wg), None, 1, K, None, ptr(dx), 1, stream()))
    assert torch.equal(dx[at].double(), dy[at].double() @ wg.double())
    dw = torch.empty(8, K, device="cuda")
    ok(L.k3g_matmul_grad_w(ptr(dy), 1, ptr(x), 1, T, 8, K, 0, ptr(dw), 0, None, stream()))
    want = torch.zeros(8, K, dtype=torch.float64, device="cuda")
    for a in range(0, T, 40000):
        want += dy[a:a + 40000].double().t() @ x[a:a + 40000].double()
    assert torch.equal(dw.double(), want)


TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")]


def whole(gen, dt, *shape):
    """Whole numbers from -3 to 3: sums of their products are exact in fp32."""
    import torch
    v = torch.randint(-3, 4, shape, device="cuda", generator=gen)
    return v.to(torch.float32 if dt == "f32" else torch.bfloat16)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("size", [500, 1101, 2999, 4103])
def test_from_few_tiles_to_many(gpu, size, types):
    """Squares of odd width, from few outputs to many: all three products, exactly"""
    import torch
    print(f"case: {size} x {size} x {size}, {types}", flush=True)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(size)
    L, (xdt, wdt) = k3moe.lib(), types
    x, dy, w = whole(gen, xdt, size, size), whole(gen, xdt, size, size), whole(gen, wdt, size, size)
    o, bias = torch.empty(size, size, device="cuda"), torch.empty(size, device="cuda")
    ok(L.k3g_matmul(ptr(x), tag(x), size, size, ptr(w), None, tag(w), size, None, ptr(o), 0, stream()))
    assert torch.equal(o.double(), x.double() @ w.double().t().contiguous())
    ok(L.k3g_matmul_grad_x(ptr(dy), None, tag(dy), size, size, ptr(w), None, tag(w), size, None, ptr(o), 0, stream()))
    assert torch.equal(o.double(), dy.double() @ w.double())
    ok(L.k3g_matmul_grad_w(ptr(dy), tag(dy), ptr(x), tag(x), size, size, size, 0, ptr(o), 0, ptr(bias), stream()))
    assert torch.equal(o.double(), dy.double().t().contiguous() @ x.double())
    assert torch.equal(bias.double(), dy.double().sum(0))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65])
def test_few_rows(gpu, rows, pair, types):
    """Up to a few rows by matrices of few features to many, with one product or two, exactly"""
    import torch
    print(f"case: {rows} rows, {types}, {'two products' if pair else 'one'}", flush=True)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    L, (xdt, wdt) = k3moe.lib(), types
    for K in (40, 130, 1100):
        for n in (5, 333, 7001):
            x, w, w3 = whole(gen, xdt, rows, K), whole(gen, wdt, n, K), whole(gen, wdt, n, K)
            y, z, z3 = (torch.full((rows + 1, n), 7.0, device="cuda") for _ in range(3))
            ep = k3moe.K3gEpilogue()
            ep.act, ep.b1, ep.b2 = k3moe.K3G_ACT_SITU if pair else k3moe.K3G_ACT_RELU, UNCAPPED, UNCAPPED
            ep.z, ep.z3 = ptr(z), ptr(z3) if pair else None
            ok(L.k3g_matmul(ptr(x), tag(x), rows, K, ptr(w), ptr(w3) if pair else None, tag(w), n, C.byref(ep), ptr(y), 0,
                            stream()))
            want = x.double() @ w.double().t().contiguous()
            assert torch.equal(z[:rows].double(), want)
            if pair:
                want3 = x.double() @ w3.double().t().contiguous()
                assert torch.equal(z3[:rows].double(), want3)
                # SwiGLU of exact factors: the sigmoid and two products, 2^-18 of it
                s = want * torch.sigmoid(want) * want3
                assert ((y[:rows].double() - s).abs() <= 2.0 ** -18 * s.abs() + 2.0 ** -100).all()
            else:
                assert torch.equal(y[:rows].double(), want.clamp(min=0))
            for o in (y, z, z3):
                assert (o[rows:] == 7).all()


def test_a_matrix_for_several_experts(gpu):
    """Experts may share a matrix; their gradients of the rows are each one's own."""
    import torch
    print("case: experts that share matrices", flush=True)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    L, P, K, n, E = k3moe.lib(), 190, 72, 104, 5
    x, dy, w = whole(gen, "bf16", P, K), whole(gen, "bf16", P, n), whole(gen, "bf16", 2, n, K)
    which = torch.tensor([0, 1, 0, 0, 1], device="cuda")
    tw = w.data_ptr() + w.stride(0) * 2 * which
    off = torch.tensor([0, 40, 41, 41, 150, 190], device="cuda", dtype=torch.int32)
    y, dx = torch.empty(P, n, device="cuda"), torch.empty(P, K, device="cuda")
    ok(L.k3g_grouped(ptr(x), 1, P, K, None, 1, ptr(off), E, ptr(tw), None, 8, 1, n, None, ptr(y), 0, stream()))
    ok(L.k3g_grouped_grad_x(ptr(dy), None, 1, P, n, ptr(off), E, ptr(tw), None, 8, 1, K, None, ptr(dx), 0, stream()))
    for e in range(E):
        a, b, m = off[e].item(), off[e + 1].item(), w[which[e]].double()
        assert torch.equal(y[a:b].double(), x[a:b].double() @ m.t().contiguous())
        assert torch.equal(dx[a:b].double(), dy[a:b].double() @ m)
