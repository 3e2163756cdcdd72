"""Plain 64-bit (and integer) forms of the operators around the experts, for the tests."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def order(idx, E):
    """perm, off, pos of the pairs idx [T][k] grouped by expert (a stable sort)."""
    key = np.asarray(idx).reshape(-1)
    kept = np.flatnonzero((key >= 0) & (key < E))
    perm = kept[np.argsort(key[kept], kind="stable")]
    off = np.concatenate([[0], np.cumsum(np.bincount(key[kept], minlength=E))])
    pos = np.full(key.size, -1)
    pos[perm] = np.arange(perm.size)
    return perm, off, pos


def to_bf16(a):
    """float -> bf16 bits, nearest even"""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = ((u >> 16) & 1) + 0x7FFF
    out = ((u + r) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), out).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint32) << 16).view(np.float32)


def quant(x):
    """MXFP4 codes [rows][cols] (0..15) and scale bytes [rows][cols / 32] of float values: nearest
    of the eight magnitudes, a tie to the even code."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[0], -1, 32)
    m = np.abs(b).max(2)
    bad = ~np.isfinite(m)
    safe = np.where(bad | (m == 0), 1.0, m)
    e = np.maximum(np.floor(np.log2(safe)) - 2, -127)
    e = np.where(m == 0, -127, e)
    v = np.abs(np.where(bad[..., None], 0.0, b)) / np.exp2(e)[..., None]
    d = np.abs(v[..., None] - E2M1)
    code = d.argmin(3)                        # the lower of two equally near codes
    up = np.minimum(code + 1, 7)
    tie = (code < 7) & (np.take_along_axis(d, up[..., None], 3)[..., 0] == d.min(3)) & (code % 2 == 1)
    code = np.where(tie, up, code) + 8 * np.signbit(b)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    scale = np.where(bad, 255, e + 127).astype(np.uint8)
    return code.reshape(x.shape), scale


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    out = np.empty((packed.shape[0], 2 * packed.shape[1]), np.uint8)
    out[:, 0::2], out[:, 1::2] = packed & 15, packed >> 4
    return out


def values(code, scale):
    """The float64 values of codes and scale bytes (255: NaN)."""
    v = np.where(code >= 8, -1.0, 1.0) * E2M1[code & 7]
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=1)
