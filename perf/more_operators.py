"""What the speed of products with weights of one's own is measured on.

Matrix products grouped by expert over ragged ranges of sorted rows, one matrix product with
bias, activation and residual in its epilogue, and the gradients of both: what a program with
bf16 or fp32 experts runs between the sort of the tokens and the way back, and beside them for
its shared expert and its projections.

Every case is one pass through an operator as a program calls it. Widths, expert counts and
top-k are those of the layers this repository is measured on (Kimi-K2 and a smaller layer) or
generic; inputs come from the case's seed alone, made on the GPU with torch.

`own` False: the operators in elementary torch operations. `own` True: k3moe's entry points.
"""
from __future__ import annotations

import ctypes as C
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
# the activations: of one product, or (situ) of a gate and an up product with caps
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh", "situ"]
UNCAPPED = 2.0**100


def _k3moe():
    path = os.path.join(ROOT, "kimi-k3-in-rust_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import k3moe
    return k3moe


# --------------------------------------------------------------------------- cases ----

def _grouped(T, topk, experts, cols, n, dt, wdt, gated, keep=False, drop=0.0, caps=False):
    """The experts' products over the sorted pairs: gated, T tokens by each expert's gate and up
    matrices and the activation; else the pairs' own rows by each expert's one matrix. keep: and
    the values before the activation, for a backward pass. drop: the share of pairs without an
    expert."""
    return dict(op="grouped", T=T, topk=topk, experts=experts, cols=cols, n=n, dt=dt, wdt=wdt, gated=gated,
                keep=keep and gated, drop=drop, caps=caps)


def _grouped_back(T, topk, experts, cols, n, dt, wdt, gated, drop=0.0, caps=False):
    """Their gradients. gated, from those of both products: the gathered rows' and both matrices'.
    Else, from the outputs': those before the activation that gave the rows, and the matrices'."""
    return dict(op="grouped_back", T=T, topk=topk, experts=experts, cols=cols, n=n, dt=dt, wdt=wdt, gated=gated,
                drop=drop, caps=caps)


def _matmul(rows, cols, n, dt, wdt, act, bias=False, residual=False, keep=False, caps=False):
    """One product (situ: two) with what follows it."""
    return dict(op="matmul", rows=rows, cols=cols, n=n, dt=dt, wdt=wdt, act=act, bias=bias, residual=residual,
                keep=keep and act != "none", caps=caps)


def _matmul_back(rows, cols, n, dt, wdt, gated, bias=False, add=False):
    """Its gradients, from those before the activation: the rows' (add: onto a gradient that they
    have already), the matrices' and the biases'."""
    return dict(op="matmul_back", rows=rows, cols=cols, n=n, dt=dt, wdt=wdt, gated=gated, bias=bias, add=add)


def _act_back(rows, n, dt, act, caps=False):
    """Through the activation: the gradients of the values before it from that of its result."""
    return dict(op="act_back", rows=rows, n=n, dt=dt, act=act, caps=caps)


def listed():
    return [
        # eight streams decoding: gate and up of the experts they meet
        dict(_grouped(8, 8, 384, 7168, 2048, "bf16", "bf16", True), name="grouped_decode_8"),
        # a long prompt: the down product of every expert
        dict(_grouped(4096, 8, 384, 2048, 7168, "bf16", "bf16", False), name="grouped_prefill_4096"),
        # training in fp32 on ragged widths, a tenth of the pairs dropped by capacity
        dict(_grouped(617, 6, 64, 1411, 709, "f32", "f32", True, keep=True, drop=0.1, caps=True),
             name="grouped_ragged_617"),
        # a batch of 4,096 tokens in training: gradients of gate and up, then of down
        dict(_grouped_back(4096, 6, 64, 2048, 1408, "bf16", "bf16", True), name="grouped_back_up_4096"),
        dict(_grouped_back(4096, 6, 64, 1408, 2048, "bf16", "bf16", False), name="grouped_back_down_4096"),
        # one stream decoding: gate and up of the shared expert, on the engine's fp32 hidden state
        dict(_matmul(1, 7168, 2048, "f32", "bf16", "situ"), name="matmul_decode_1"),
        # a batch of streams: a projection with a bias, its activation, onto the hidden state
        dict(_matmul(24, 7168, 3584, "bf16", "bf16", "gelu", bias=True, residual=True), name="matmul_step_24"),
        # a batch in training: gate and up of the shared expert, values kept for the way back
        dict(_matmul(4096, 7168, 2048, "bf16", "bf16", "situ", keep=True), name="matmul_train_4096"),
        # and its way back, onto the routed experts' gradient
        dict(_matmul_back(4096, 7168, 2048, "bf16", "bf16", True, add=True), name="matmul_back_4096"),
        # a small fp32 batch of ragged widths on bf16 weights
        dict(_matmul_back(617, 1411, 709, "f32", "bf16", False, bias=True), name="matmul_back_ragged_617"),
        # the activation's part of a way back: the pairs of the training batch, and a small batch
        dict(_act_back(24576, 1408, "bf16", "situ"), name="act_back_24576"),
        dict(_act_back(617, 709, "f32", "gelu"), name="act_back_617"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    w = _log(rng, 64, 7168)
    return w if rng.random() < 0.3 else max(w // 32 * 32, 64)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["grouped", "grouped", "grouped_back", "grouped_back", "matmul", "matmul", "matmul_back",
                         "act_back"])
        dt, wdt = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
        experts = _log(rng, 8, 384)
        topk = rng.randint(1, min(12, experts))
        drop = rng.choice([0.0, 0.0, 0.1])
        cols, n, caps = _width(rng), _width(rng), rng.random() < 0.3
        if op == "grouped":
            c = _grouped(_log(rng, 1, 4096), topk, experts, cols, n, dt, wdt, rng.random() < 0.5,
                         rng.random() < 0.5, drop, caps)
        elif op == "grouped_back":
            c = _grouped_back(_log(rng, 16, 4096), topk, experts, cols, n, dt, wdt, rng.random() < 0.5, drop, caps)
        elif op == "matmul":
            c = _matmul(_log(rng, 1, 4096), cols, n, dt, wdt, rng.choice(ACTS), rng.random() < 0.5,
                        rng.random() < 0.5, rng.random() < 0.5, caps)
        elif op == "matmul_back":
            c = _matmul_back(_log(rng, 16, 4096), cols, n, dt, wdt, rng.random() < 0.5, rng.random() < 0.5,
                             rng.random() < 0.5)
        else:
            c = _act_back(_log(rng, 1, 32768), _log(rng, 64, 4096), dt, rng.choice(ACTS[1:]), caps)
        if op.startswith("grouped") and experts * cols * n * (2 if c["gated"] else 1) > 384 * 2048 * 7168:
            continue
        if _cost(c) <= most:
            return c


# ------------------------------------------------------------------------- inputs ----

def _generator(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + stream)
    return g


def _normal(shape, seed, stream, std=1.0, dt="f32"):
    v = torch.empty(shape, dtype=TYPES[dt], device="cuda")
    return v.normal_(0.0, std, generator=_generator(seed, stream))


def _activations(rows, cols, seed, stream, dt):
    """Normally distributed, a few channels ten times as large, as a hidden state's are."""
    v = _normal((rows, cols), seed, stream)
    c = torch.randperm(cols, device="cuda", generator=_generator(seed, stream + 1))[:max(cols // 100, 1)]
    v[:, c] *= 10.0
    return v.to(TYPES[dt])


def _routing(case, seed):
    """idx [T][topk], each token's experts distinct, popular experts among them, -1 for a dropped
    pair."""
    T, k, E = case["T"], case["topk"], case["experts"]
    bias = _normal((E,), seed, 50, 0.5)
    idx = torch.topk(_normal((T, E), seed, 51) + bias, k, dim=1).indices
    if case["drop"]:
        lost = torch.rand((T, k), device="cuda", generator=_generator(seed, 52)) < case["drop"]
        idx = torch.where(lost, -1, idx)
    return idx


def _order(idx, E):
    """perm and off of the pairs grouped by expert (perm -1 behind the last kept one)."""
    key = idx.reshape(-1)
    key = torch.where(key < 0, E, key)
    order = torch.sort(key, stable=True)
    off = torch.searchsorted(order.values, torch.arange(E + 1, device=key.device), right=False)
    kept = torch.arange(key.numel(), device=key.device) < off[E]
    return torch.where(kept, order.indices, -1).to(torch.int32), off.to(torch.int32)


class _State:
    pass


def _inputs(case, seed):
    s, c = _State(), case
    s.case, op, dt = c, c["op"], c["dt"]
    n = c["n"]
    if op == "act_back":
        s.dh = _normal((c["rows"], n), seed, 1, dt=dt)
        s.z = _normal((c["rows"], n), seed, 2, 2.0, dt)
        s.z3 = _normal((c["rows"], n), seed, 3, 2.0, dt) if c["act"] == "situ" else None
        return s
    cols = c["cols"]
    pair = c["act"] == "situ" if op == "matmul" else c["gated"]
    lead = ()
    if op.startswith("grouped"):
        s.perm, s.off = _order(_routing(c, seed), c["experts"])
        lead, P = (c["experts"],), c["T"] * c["topk"]
        # gated products read the tokens' rows by perm, single ones the sorted rows
        rows, places = (c["T"] if c["gated"] else P), P
    else:
        rows = places = c["rows"]
    s.x = _activations(rows, cols, seed, 10, dt)
    # weights that keep a row's size about one
    std = 1.0 / math.sqrt(cols)
    s.w = _normal(lead + (n, cols), seed, 12, std, c["wdt"])
    s.w3 = _normal(lead + (n, cols), seed, 13, std, c["wdt"]) if pair else None
    if op.endswith("back"):
        s.dy = _normal((places, n), seed, 14, dt=dt)
        s.dy3 = _normal((places, n), seed, 15, dt=dt) if pair else None
        if op == "matmul_back":
            s.add = _normal((rows, cols), seed, 16, dt=dt) if c["add"] else None
        elif not c["gated"]:
            s.z, s.z3 = _normal((P, cols), seed, 17, 2.0, dt), _normal((P, cols), seed, 18, 2.0, dt)
    elif op == "matmul":
        s.bias = _normal((n,), seed, 19, 0.2) if c["bias"] else None
        s.bias3 = _normal((n,), seed, 20, 0.2) if c["bias"] and pair else None
        s.residual = _normal((rows, n), seed, 21, dt=dt) if c["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"].startswith("grouped"):
        # a program that loops over the experts on the host knows their ranges there
        s.ranges = s.off.tolist()
    if own:
        _own_state(s)
    torch.cuda.synchronize()
    return s


def _caps(c):
    return (4.0, 25.0) if c.get("caps") else (UNCAPPED, UNCAPPED)


def _own_state(s):
    """The tables of weights and the output buffers a program keeps."""
    k3, c = _k3moe(), s.case
    s.lib, s.k3 = k3.lib(), k3
    s.tags = {"f32": k3.K3_WF32, "bf16": k3.K3_WBF16}
    op, dt, n = c["op"], TYPES[c["dt"]], c["n"]

    def buf(*shape, dtype=dt):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    def table(t):
        return t.data_ptr() + t.stride(0) * t.element_size() * torch.arange(t.shape[0], device="cuda")

    def ptr(t):
        return None if t is None else t.data_ptr()

    b1, b2 = _caps(c)
    if op == "act_back":
        s.dz = torch.empty_like(s.z)
        s.dz3 = torch.empty_like(s.z) if c["act"] == "situ" else None
        return
    cols = c["cols"]
    grouped = op.startswith("grouped")
    places = c["T"] * c["topk"] if grouped else c["rows"]
    if grouped:
        s.table, s.table3 = table(s.w), table(s.w3) if c["gated"] else None
    if op in ("grouped", "matmul"):
        act = ("situ" if c["gated"] else "none") if grouped else c["act"]
        s.y = buf(places, n)
        s.z = buf(places, n) if c["keep"] else None
        s.z3 = buf(places, n) if c["keep"] and act == "situ" else None
        s.ep = k3.K3gEpilogue()
        s.ep.act, s.ep.b1, s.ep.b2 = getattr(k3, "K3G_ACT_" + act.upper()), b1, b2
        s.ep.z, s.ep.z3 = ptr(s.z), ptr(s.z3)
        if op == "matmul":
            s.ep.bias, s.ep.bias3, s.ep.residual = ptr(s.bias), ptr(s.bias3), ptr(s.residual)
        return
    s.dx = buf(places, cols)
    s.dw = buf(*s.w.shape, dtype=torch.float32)
    s.dw3 = buf(*s.w.shape, dtype=torch.float32) if c["gated"] else None
    s.back = k3.K3gBack()
    if grouped:
        s.dtable, s.dtable3 = table(s.dw), table(s.dw3) if c["gated"] else None
        if not c["gated"]:
            s.dz3 = buf(places, cols)
            s.back.act, s.back.b1, s.back.b2 = k3.K3G_ACT_SITU, b1, b2
            s.back.z, s.back.z3, s.back.dz3 = ptr(s.z), ptr(s.z3), ptr(s.dz3)
    else:
        s.back.add = ptr(s.add)
        s.db = buf(n, dtype=torch.float32) if c["bias"] else None
        s.db3 = buf(n, dtype=torch.float32) if c["bias"] and c["gated"] else None


# --------------------------------------------------------------------------- passes ----

def run(s):
    return (_run_own if own else _run_plain)(s)


def _ok(rc):
    if rc != 0:
        raise RuntimeError("a k3moe call failed")


def _run_own(s):
    c, L, st = s.case, s.lib, torch.cuda.current_stream().cuda_stream
    op, dt, n = c["op"], s.tags[c["dt"]], c["n"]

    def ptr(t):
        return None if t is None else t.data_ptr()

    if op == "act_back":
        b1, b2 = _caps(c)
        _ok(L.k3g_act_grad(ptr(s.dh), dt, c["rows"], n, getattr(s.k3, "K3G_ACT_" + c["act"].upper()), b1, b2,
                           ptr(s.z), ptr(s.z3), ptr(s.dz), ptr(s.dz3), st))
        return {"dz": s.dz, "dz3": s.dz3} if c["act"] == "situ" else {"dz": s.dz}
    cols, wdt = c["cols"], s.tags[c["wdt"]]
    if op == "matmul":
        _ok(L.k3g_matmul(ptr(s.x), dt, c["rows"], cols, ptr(s.w), ptr(s.w3), wdt, n, C.byref(s.ep), ptr(s.y), dt, st))
    elif op == "grouped":
        gated = c["gated"]
        _ok(L.k3g_grouped(ptr(s.x), dt, s.x.shape[0], cols, ptr(s.perm) if gated else None, c["topk"] if gated else 1,
                          ptr(s.off), c["experts"], ptr(s.table), ptr(s.table3), 8, wdt, n, C.byref(s.ep), ptr(s.y),
                          dt, st))
    if op in ("matmul", "grouped"):
        out = {"y": s.y}
        if s.z is not None:
            out["z"] = s.z
        if s.z3 is not None:
            out["z3"] = s.z3
        return out
    f32 = s.tags["f32"]
    if op == "matmul_back":
        rows = c["rows"]
        _ok(L.k3g_matmul_grad_x(ptr(s.dy), ptr(s.dy3), dt, rows, n, ptr(s.w), ptr(s.w3), wdt, cols, C.byref(s.back),
                                ptr(s.dx), dt, st))
        _ok(L.k3g_matmul_grad_w(ptr(s.dy), dt, ptr(s.x), dt, rows, n, cols, 0, ptr(s.dw), f32, ptr(s.db), st))
        out = {"dx": s.dx, "dw": s.dw}
        if c["gated"]:
            _ok(L.k3g_matmul_grad_w(ptr(s.dy3), dt, ptr(s.x), dt, rows, n, cols, 0, ptr(s.dw3), f32, ptr(s.db3), st))
            out["dw3"] = s.dw3
        if c["bias"]:
            out["db"] = s.db
            if c["gated"]:
                out["db3"] = s.db3
        return out
    gated, E, P = c["gated"], c["experts"], c["T"] * c["topk"]
    _ok(L.k3g_grouped_grad_x(ptr(s.dy), ptr(s.dy3), dt, P, n, ptr(s.off), E, ptr(s.table), ptr(s.table3), 8, wdt,
                             cols, C.byref(s.back), ptr(s.dx), dt, st))
    perm, topk = (ptr(s.perm), c["topk"]) if gated else (None, 1)
    _ok(L.k3g_grouped_grad_w(ptr(s.dy), dt, ptr(s.x), dt, s.x.shape[0], n, cols, perm, topk, ptr(s.off), E, 0,
                             ptr(s.dtable), 8, f32, None, st))
    if not gated:
        return {"dz": s.dx, "dz3": s.dz3, "dw": s.dw}
    _ok(L.k3g_grouped_grad_w(ptr(s.dy3), dt, ptr(s.x), dt, s.x.shape[0], n, cols, perm, topk, ptr(s.off), E, 0,
                             ptr(s.dtable3), 8, f32, None, st))
    return {"dx": s.dx, "dw": s.dw, "dw3": s.dw3}


def _plain_act(act, z, z3, b1, b2):
    if act == "none":
        return z
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return z * torch.sigmoid(math.sqrt(8.0 / math.pi) * (z + 0.044715 * z * z * z))
    a, u = (z, z3) if b1 == UNCAPPED else (b1 * torch.tanh(z / b1), b2 * torch.tanh(z3 / b2))
    return a * torch.sigmoid(z) * u


def _plain_act_grad(act, g, z, z3, b1, b2):
    """g times the activation's derivative by z (and by z3)."""
    if act == "relu":
        return torch.where(z > 0.0, g, 0.0), None
    s = torch.sigmoid(z)
    if act == "silu":
        return g * s * (1.0 + z * torch.sigmoid(-z)), None
    if act == "gelu":
        return g * (0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)), None
    if act == "gelu_tanh":
        k = math.sqrt(8.0 / math.pi)
        v = k * (z + 0.044715 * z * z * z)
        t = torch.sigmoid(v)
        return g * t * (1.0 + z * torch.sigmoid(-v) * k * (1.0 + 3.0 * 0.044715 * z * z)), None
    if b1 == UNCAPPED:
        a, da, u, du = z, 1.0, z3, 1.0
    else:
        a, da = b1 * torch.tanh(z / b1), 1.0 / torch.cosh(z / b1)**2
        u, du = b2 * torch.tanh(z3 / b2), 1.0 / torch.cosh(z3 / b2)**2
    return g * s * (da + a * torch.sigmoid(-z)) * u, g * a * s * du


def _run_plain(s):
    c = s.case
    op, dt = c["op"], TYPES[c["dt"]]
    b1, b2 = _caps(c)
    if op == "act_back":
        z3 = s.z3.float() if s.z3 is not None else None
        dz, dz3 = _plain_act_grad(c["act"], s.dh.float(), s.z.float(), z3, b1, b2)
        return {"dz": dz.to(dt), "dz3": dz3.to(dt)} if z3 is not None else {"dz": dz.to(dt)}
    if op == "matmul":
        x = s.x.float()
        z = x @ s.w.float().T
        z3 = x @ s.w3.float().T if s.w3 is not None else None
        if s.bias is not None:
            z = z + s.bias
            z3 = z3 + s.bias3 if z3 is not None else None
        y = _plain_act(c["act"], z, z3, b1, b2)
        if s.residual is not None:
            y = y + s.residual.float()
        out = {"y": y.to(dt)}
        if c["keep"]:
            out["z"] = z.to(dt)
            if z3 is not None:
                out["z3"] = z3.to(dt)
        return out
    if op == "matmul_back":
        dy, x = s.dy.float(), s.x.float()
        dx = dy @ s.w.float()
        out = {"dw": dy.T @ x}
        if c["bias"]:
            out["db"] = dy.sum(0)
        if c["gated"]:
            dy3 = s.dy3.float()
            dx = dx + dy3 @ s.w3.float()
            out["dw3"] = dy3.T @ x
            if c["bias"]:
                out["db3"] = dy3.sum(0)
        if s.add is not None:
            dx = dx + s.add.float()
        out["dx"] = dx.to(dt)
        return out
    P, n, cols, gated = c["T"] * c["topk"], c["n"], c["cols"], c["gated"]
    token = s.perm.long() // c["topk"] if gated else None

    def zeros(*shape, dtype=dt):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    if op == "grouped":
        out = {"y": zeros(P, n)}
        if c["keep"]:
            out["z"], out["z3"] = zeros(P, n), zeros(P, n)
    else:
        out = {k: zeros(P, cols) for k in (("dx",) if gated else ("dz", "dz3"))}
        out["dw"] = zeros(*s.w.shape, dtype=torch.float32)
        if gated:
            out["dw3"] = zeros(*s.w.shape, dtype=torch.float32)
    for e in range(c["experts"]):
        a, b = s.ranges[e], s.ranges[e + 1]
        if a == b:
            continue
        x = (s.x[token[a:b]] if gated else s.x[a:b]).float()
        w = s.w[e].float()
        w3 = s.w3[e].float() if gated else None
        if op == "grouped":
            z = x @ w.T
            if gated:
                z3 = x @ w3.T
                if c["keep"]:
                    out["z"][a:b], out["z3"][a:b] = z.to(dt), z3.to(dt)
                z = _plain_act("situ", z, z3, b1, b2)
            out["y"][a:b] = z.to(dt)
            continue
        dy = s.dy[a:b].float()
        out["dw"][e] = dy.T @ x
        g = dy @ w
        if gated:
            dy3 = s.dy3[a:b].float()
            out["dw3"][e] = dy3.T @ x
            out["dx"][a:b] = (g + dy3 @ w3).to(dt)
        else:
            dz, dz3 = _plain_act_grad("situ", g, s.z[a:b].float(), s.z3[a:b].float(), b1, b2)
            out["dz"][a:b], out["dz3"][a:b] = dz.to(dt), dz3.to(dt)
    return out


# ------------------------------------------------------------------ what it costs ----

def _met(c):
    """Distinct experts that a call of these sizes meets, from scores as the inputs' are."""
    rng = np.random.default_rng(7)
    E = c["experts"]
    bias = rng.normal(0.0, 0.5, E)
    met = np.zeros(E, bool)
    for t0 in range(0, c["T"], 512):
        z = rng.normal(0.0, 1.0, (min(512, c["T"] - t0), E)) + bias
        met[np.argpartition(-z, c["topk"] - 1, axis=1)[:, :c["topk"]].reshape(-1)] = True
        if met.all():
            break
    return int(met.sum())


def work(case):
    c, op, n = case, case["op"], case["n"]
    b = SIZE[c["dt"]]
    if op == "act_back":
        v = c["rows"] * n
        return {"bytes": v * b * (5 if c["act"] == "situ" else 3), "flops": 20 * v}
    cols, wb = c["cols"], SIZE[c["wdt"]]
    if op.startswith("grouped"):
        kept = c["T"] * c["topk"] * (1.0 - c["drop"])
        met, gated = _met(c), c["gated"]
        read = c["T"] if gated else kept           # rows of x
        index = 4 * (c["experts"] + 1) + (4 * kept if gated else 0)
        w = (2 if gated else 1) * n * cols
        flops = 2 * kept * w
        if op == "grouped":
            byt = index + b * read * cols + wb * met * w + b * kept * n * (3 if c["keep"] else 1)
            return {"bytes": int(byt), "flops": int(flops)}
        # the gradients' rows in, the rows out (down: both values before the activation in, both
        # gradients out), weights in, their gradients out
        byt = index + b * kept * n * (2 if gated else 1) + b * read * cols + b * kept * cols * (1 if gated else 4)
        byt += wb * met * w + 4 * c["experts"] * w
        return {"bytes": int(byt), "flops": int(2 * flops)}
    rows = c["rows"]
    m = 2 if (c["act"] == "situ" if op == "matmul" else c["gated"]) else 1
    flops = 2 * rows * m * n * cols
    if op == "matmul":
        byt = b * rows * cols + wb * m * n * cols + b * rows * n * (1 + c["residual"] + (m if c["keep"] else 0))
        return {"bytes": byt + (4 * m * n if c["bias"] else 0), "flops": flops}
    byt = b * rows * (m * n + cols * (2 + c["add"])) + (wb + 4) * m * n * cols + (4 * m * n if c["bias"] else 0)
    return {"bytes": byt, "flops": 2 * flops}


def _cost(c):
    w = work(c)
    # fp32 values cost several matrix products of bf16 ones
    return w["bytes"] / 5e12 + w["flops"] / (1e15 if c["dt"] == "bf16" else 2e14)


# ------------------------------------------------------------------- in 64 bits ----

def _exact_act(act, z, z3, b1, b2, grad=None):
    """The activation, or, given the gradient of its result, those of z and z3."""
    one = torch.ones((), dtype=torch.float64, device=z.device)
    sig = one / (one + torch.exp(-z))
    if act == "none":
        v, d = z, torch.ones_like(z)
    elif act == "relu":
        v, d = torch.where(z > 0, z, 0.0), (z > 0).double()
    elif act == "silu":
        v, d = z * sig, sig + z * sig * (1 - sig)
    elif act == "gelu":
        phi = torch.special.ndtr(z)
        v, d = z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    elif act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z**3))
        v = 0.5 * z * (1 + t)
        d = 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    else:
        a, ga = z, torch.ones_like(z)
        u, gu = z3, torch.ones_like(z)
        if b1 != UNCAPPED:
            ta, tu = torch.tanh(z / b1), torch.tanh(z3 / b2)
            a, ga, u, gu = b1 * ta, 1 - ta * ta, b2 * tu, 1 - tu * tu
        if grad is None:
            return a * sig * u
        return grad * u * (ga * sig + a * sig * (1 - sig)), grad * a * sig * gu
    return v if grad is None else (grad * d, None)


def exact(case, seed):
    s, c = _inputs(case, seed), case
    op = c["op"]
    b1, b2 = _caps(c)
    if op == "act_back":
        z3 = None if s.z3 is None else s.z3.double()
        dz, dz3 = _exact_act(c["act"], s.z.double(), z3, b1, b2, s.dh.double())
        return {"dz": dz} if z3 is None else {"dz": dz, "dz3": dz3}
    if op == "matmul":
        x, out = s.x.double(), {}
        z, z3 = torch.mm(x, s.w.double().t()), None
        if s.w3 is not None:
            z3 = torch.mm(x, s.w3.double().t())
        if c["bias"]:
            z += s.bias.double()
            if z3 is not None:
                z3 += s.bias3.double()
        out["y"] = _exact_act(c["act"], z, z3, b1, b2)
        if c["residual"]:
            out["y"] = out["y"] + s.residual.double()
        if c["keep"]:
            out["z"] = z
            if z3 is not None:
                out["z3"] = z3
        return out
    if op == "matmul_back":
        dy, x = s.dy.double(), s.x.double()
        dx = torch.mm(dy, s.w.double())
        out = {"dw": torch.mm(dy.t(), x)}
        if c["gated"]:
            dy3 = s.dy3.double()
            dx += torch.mm(dy3, s.w3.double())
            out["dw3"] = torch.mm(dy3.t(), x)
        if c["bias"]:
            out["db"] = dy.sum(0)
            if c["gated"]:
                out["db3"] = dy3.sum(0)
        out["dx"] = dx + s.add.double() if c["add"] else dx
        return out
    E, k, n, cols, gated = c["experts"], c["topk"], c["n"], c["cols"], c["gated"]
    P = c["T"] * k
    key = _routing(c, seed).reshape(-1).cpu().numpy()
    kept = np.flatnonzero(key >= 0)
    pairs = kept[np.argsort(key[kept], kind="stable")]
    off = np.concatenate([[0], np.cumsum(np.bincount(key[kept], minlength=E))])

    def empty(*shape):
        return torch.zeros(shape, dtype=torch.float64, device="cuda")

    if op == "grouped":
        out = {"y": empty(P, n)}
        if c["keep"]:
            out.update(z=empty(P, n), z3=empty(P, n))
    elif gated:
        out = dict(dx=empty(P, cols), dw=empty(E, n, cols), dw3=empty(E, n, cols))
    else:
        out = dict(dz=empty(P, cols), dz3=empty(P, cols), dw=empty(E, n, cols))
    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        if r.start == r.stop:
            continue
        at = torch.from_numpy(pairs[r] // k).cuda() if gated else torch.arange(r.start, r.stop, device="cuda")
        x, w = s.x[at].double(), s.w[e].double()
        if op == "grouped":
            z = torch.mm(x, w.t())
            if gated:
                z3 = torch.mm(x, s.w3[e].double().t())
                if c["keep"]:
                    out["z"][r], out["z3"][r] = z, z3
                z = _exact_act("situ", z, z3, b1, b2)
            out["y"][r] = z
            continue
        dy = s.dy[r].double()
        out["dw"][e] = torch.mm(dy.t(), x)
        g = torch.mm(dy, w)
        if gated:
            dy3 = s.dy3[r].double()
            out["dw3"][e] = torch.mm(dy3.t(), x)
            out["dx"][r] = g + torch.mm(dy3, s.w3[e].double())
        else:
            out["dz"][r], out["dz3"][r] = _exact_act("situ", s.z[r].double(), s.z3[r].double(), b1, b2, g)
    return out
