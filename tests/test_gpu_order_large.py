"""Token rows in expert order and back at the sizes where the calls run on other kernels than small
ones do: bf16 gradients four slots at a time (4096 pairs and more, topk of 3 and more), and sorted
rows of more than 256 MB, which are streamed past the caches. Against plain 64-bit forms."""
import pytest

import k3moe
import test_gpu_order as small

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,n", [(1366, 3, 257), (820, 5, 1411), (683, 6, 1024), (512, 8, 1025), (512, 8, 64),
                                   (700, 6, 2051), (600, 7, 7), (1024, 4, 4096)])
@pytest.mark.parametrize("skew,drop", [(0, 0.0), (1, 0.3)])
def test_gradients_of_four_slots_together(gpu, T, k, n, skew, drop):
    """topk that leaves one, two or three slots in a token's last four, rows of a wave (up to 1024
    elements) and of four, dropped pairs among the four; each gradient also without the other."""
    assert T * k >= 4096
    small.test_unpermute(gpu, T, k, n, "bf16", skew, drop)


def streamed(T, k, n, dt):
    """Inputs of T x k pairs whose sorted rows are more than 256 MB, on the GPU."""
    import torch
    tag, _, eps = small.DT[dt]
    t = torch.bfloat16 if dt == "bf16" else torch.float32
    assert T * k * n * (2 if dt == "bf16" else 4) > 1 << 28
    gen = torch.Generator(device="cuda")
    gen.manual_seed(T + n)

    def normal(*s):
        return torch.empty(s, device="cuda").normal_(generator=gen).to(t)

    P = T * k
    order = torch.randperm(P, device="cuda", generator=gen)
    lost = torch.rand(P, device="cuda", generator=gen) < 0.1
    pos = torch.where(lost, -1, order).int()
    wt = torch.rand(P, device="cuda", generator=gen)
    return tag, eps, P, pos, wt, normal


@pytest.mark.parametrize("T,k,n,dt", [(2400, 8, 3600, "f32"), (20000, 8, 500, "f32"), (70000, 8, 125, "f32"),
                                      (3700, 5, 7300, "bf16"), (20000, 7, 1000, "bf16"), (70000, 8, 250, "bf16")])
def test_streamed(gpu, T, k, n, dt):
    """Every row of every call, there and back."""
    import torch
    print(f"case: streamed rows, {T} x {k}, width {n}, {dt}", flush=True)
    L = k3moe.lib()
    tag, eps, P, pos, wt, normal = streamed(T, k, n, dt)
    kept = (pos >= 0).nonzero()[:, 0]
    token, place = kept // k, pos[kept].long()
    x, s, g, add = normal(T, n), normal(P, n), normal(T, n), normal(T, n)
    torch.cuda.synchronize()

    def close(got, want, size, rounds, what):
        bad = (got.double() - want).abs() > rounds * 2.0 ** -24 * size + eps * want.abs() * (1 + 2.0 ** -7)
        assert not bool(bad.any()), what

    def by_token(v):
        return torch.zeros(T, n, dtype=torch.float64, device="cuda").index_add_(0, token, v)

    # rows out: copies; a place that no pair has stays as it was
    out = torch.full((P, n), 7.0, dtype=x.dtype, device="cuda")
    assert L.k3g_permute(x.data_ptr(), tag, T, k, n, pos.data_ptr(), out.data_ptr(), None) == 0
    torch.cuda.synchronize()
    want = torch.full_like(out, 7.0)
    want[place] = x[token]
    assert torch.equal(out, want)
    # their gradient: k additions; and rows back: a product, k + 1 additions; then the output's rounding
    rows = s[place].double()
    dx = torch.empty_like(x)
    assert L.k3g_permute_grad(s.data_ptr(), tag, T, k, n, pos.data_ptr(), dx.data_ptr(), None) == 0
    torch.cuda.synchronize()
    close(dx, by_token(rows), by_token(rows.abs()), k, "gradient of rows out")
    y = torch.empty_like(x)
    assert L.k3g_unpermute(s.data_ptr(), tag, T, k, n, pos.data_ptr(), wt.data_ptr(), add.data_ptr(), y.data_ptr(),
                           None) == 0
    torch.cuda.synchronize()
    w = wt[kept].double().unsqueeze(1)
    close(y, by_token(w * rows) + add.double(), by_token(w * rows.abs()) + add.double().abs(), k + 2, "rows back")
    # gradients: one product each; and dots of n products and additions in any order
    out.fill_(7.0)
    dw = torch.full((P,), 7.0, device="cuda")
    assert L.k3g_unpermute_grad(g.data_ptr(), s.data_ptr(), tag, T, k, n, pos.data_ptr(), wt.data_ptr(),
                                out.data_ptr(), dw.data_ptr(), None) == 0
    torch.cuda.synchronize()
    go = g[token].double()
    exact = w * go
    close(out[place], exact, exact.abs(), 1, "gradient of the rows")
    free = torch.ones(P, dtype=torch.bool, device="cuda")
    free[place] = False
    assert bool((out[free] == 7.0).all())
    dots = (rows * go).sum(1)
    assert bool(((dw[kept].double() - dots).abs() <= (n + 1) * 2.0 ** -24 * (rows * go).abs().sum(1)).all())
    assert bool((dw[pos < 0] == 0).all())
