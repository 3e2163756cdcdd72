"""The gated product's activation on gates and ups of 24 bits: in fp32, within 2^-19 of its value.

A gate is a sum of 12 blocks that hold two bits of it each (a block's one value, 1 to 3 times a power
of two, is exact in MXFP4), by weights of 1; an up is 12 blocks more, which the other matrix reads.
All terms of a sum are multiples of its last bit, so any order of adding them up in fp32 is exact."""
import numpy as np
import pytest

import k3moe
import ops64
import test_gpu_mx as small

pytestmark = pytest.mark.gpu

BLOCKS = 12


def digits(v):
    """v (at most 24 bits each) as BLOCKS values of two bits: [len][BLOCKS], largest first"""
    m, e = np.frexp(v.astype(np.float64))
    m = np.abs(m * 2.0 ** 24).astype(np.int64)
    k = 2 * np.arange(BLOCKS - 1, -1, -1)
    d = (m[:, None] >> k) & 3
    return np.sign(v)[:, None] * d * np.exp2((e[:, None] - 24 + k).astype(np.float64))


def pairs(count, seed):
    """gates and ups of random 24 bits, their sizes spread evenly from 2^-10 to 2^7; gates above -87"""
    rng = np.random.default_rng(seed)
    v = np.exp2(rng.uniform(-10, 7, (2, count))) * rng.choice([-1.0, 1.0], (2, count))
    g, u = v.astype(np.float32)
    return np.where(g <= -87, -g, g), u


def gated(g, u, n, caps):
    """The gated product of one expert whose gate and up of row r are g[r] and u[r] in all n features"""
    rows, cols = g.size, 32 * 2 * BLOCKS + 32
    x = np.zeros((rows, cols), np.float32)
    x[:, :32 * BLOCKS:32] = digits(g)
    x[:, 32 * BLOCKS:64 * BLOCKS:32] = digits(u)
    code = np.zeros((2, n, cols), np.uint8)
    code[0, :, :32 * BLOCKS:32] = 2
    code[1, :, 32 * BLOCKS:64 * BLOCKS:32] = 2
    one = np.full((n, cols // 32), 127, np.uint8)
    bufs = [small.tiled(ops64.pack(c), one, n, cols) for c in code]
    tabs = [np.array([b.ptr], np.uint64) for b in bufs]
    off, perm = np.array([0, rows]), np.arange(rows)
    # the sums are the gates and ups themselves
    for t, v in zip(tabs, (g, u)):
        alone = small.grouped(x, "f32", perm, 1, off, [t], n, "f32", rows)
        assert np.array_equal(alone, np.repeat(v[:, None], n, axis=1))
    return small.grouped(x, "f32", perm, 1, off, tabs, n, "f32", rows, caps)


# 2 rows are quantised in the kernel; 9 and 40 run by 16 and 32 places, 4096 by 512 features by 64 and
# by 1024 by 128
@pytest.mark.parametrize("rows,n", [(2, 16), (9, 16), (40, 16), (4096, 16), (4096, 512), (4096, 1024)])
@pytest.mark.parametrize("caps", [(2.0 ** 100, 2.0 ** 100), (4.0, 25.0), (3.7, 3.7), (1.3, 5.5), (0.3, 2.0 ** 100),
                                  (2.0 ** 100, 7.9)])
def test_activation_of_24_bits(gpu, rows, n, caps):
    print(f"case: the activation of {rows} gates, {n} features, caps {caps}", flush=True)
    g, u = pairs(rows, rows + n)
    got = gated(g, u, n, caps).astype(np.float64)
    assert np.array_equal(got, np.repeat(got[:, :1], n, axis=1)), "features differ"
    b1, b2 = (np.float64(np.float32(c)) for c in caps)
    want = small.activation(g.astype(np.float64), u.astype(np.float64), b1, b2)
    off = np.abs(got[:, 0] - want)
    normal = np.abs(want) >= 2.0 ** -126
    print(f"largest error {(off / np.spacing(np.abs(want).astype(np.float32)))[normal].max():.2f} units in the last "
          f"place, {(off / np.abs(want))[normal].max() * 2 ** 24:.2f} of 2^-24", flush=True)
    # in units of 2^-24, with a reciprocal and a power of two off by one unit in the last place: the
    # sigmoid at most 5.3, each tanh 4.9, each quotient by a cap 2, four products 4: 23 of 32. A gate
    # near -87 leaves products below 2^-126: the one with the sigmoid, then rounded to within 2^-150
    # and multiplied by at most |up|, and the last one, rounded to within 2^-150
    assert np.all(off <= 2.0 ** -19 * np.abs(want) + 2.0 ** -150 * (np.abs(u.astype(np.float64)) + 1))


def test_activation_where_roundings_add_up(gpu):
    """Gates and ups whose parts are off most, and on one side: 10 to 12.5 units in the last place by a
    search over what correctly rounded reciprocals and powers of two would give."""
    print("case: the activation where its roundings add up", flush=True)
    for cap, gate, up in ((3.0, "-0x1.3ab9f4p-4", "-0x1.b2e912p-2"), (3.7, "-0x1.11a2ccp-3", "0x1.00673cp-4"),
                          (5.5, "-0x1.1afe66p-2", "0x1.5fa366p+2"), (6.0, "0x1.b8ec06p-6", "0x1.7eec94p+2"),
                          (4.0, "-0x1.c2b0b6p+1", "0x1.fbfe46p+1"), (3.0, "-0x1.11d778p-5", "0x1.78838cp+1")):
        g, u = np.array([float.fromhex(gate)] * 2, np.float32), np.array([1, -1], np.float32) * np.float32(float.fromhex(up))
        got = gated(g, u, 16, (cap, cap))[:, 0].astype(np.float64)
        c = np.float64(np.float32(cap))
        want = small.activation(g.astype(np.float64), u.astype(np.float64), c, c)
        off = np.abs(got - want)
        print(f"cap {cap}: {(off / np.spacing(np.abs(want).astype(np.float32))).max():.2f} units in the last place, "
              f"{(off / np.abs(want)).max() * 2 ** 24:.2f} of 2^-24", flush=True)
        assert np.all(off <= 2.0 ** -19 * np.abs(want))
