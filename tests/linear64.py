"""Plain 64-bit forms of the products with weights of one's own and of what follows them, and the
bounds that fp32 sums of their terms keep."""
import math

import numpy as np

UNCAPPED = 2.0 ** 100
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh", "situ"]
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def cap(v, b):
    return (v, np.ones_like(v)) if b >= 2.0 ** 64 else (b * np.tanh(v / b), 1.0 / np.cosh(np.minimum(np.abs(v / b), 300)) ** 2)


def act(name, z, z3=None, b1=UNCAPPED, b2=UNCAPPED):
    if name == "none":
        return z
    if name == "relu":
        return np.maximum(z, 0.0)
    if name == "silu":
        return z * sigmoid(z)
    if name == "gelu":
        return 0.5 * z * _erfc(-z / math.sqrt(2.0))
    if name == "gelu_tanh":
        return z * sigmoid(math.sqrt(8.0 / math.pi) * (z + 0.044715 * z ** 3))
    return cap(z, b1)[0] * sigmoid(z) * cap(z3, b2)[0]


def slopes(name, z, z3=None, b1=UNCAPPED, b2=UNCAPPED):
    """d act / dz and (situ) d act / dz3"""
    s = sigmoid(z)
    if name == "none":
        return np.ones_like(z), None
    if name == "relu":
        return (z > 0).astype(np.float64), None
    if name == "silu":
        return s * (1 + z * sigmoid(-z)), None
    if name == "gelu":
        return 0.5 * _erfc(-z / math.sqrt(2.0)) + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), None
    if name == "gelu_tanh":
        k = math.sqrt(8.0 / math.pi)
        v = k * (z + 0.044715 * z ** 3)
        return sigmoid(v) * (1 + z * sigmoid(-v) * k * (1 + 3 * 0.044715 * z * z)), None
    (a, da), (u, du) = cap(z, b1), cap(z3, b2)
    return s * (da + a * sigmoid(-z)) * u, a * s * du


def sum_bound(terms, size):
    """How far an fp32 sum of `terms` products, in any order, may be off where their magnitudes add
    up to `size`: every addition rounds by 2^-24 of a partial sum; products of fp32 operands in
    pieces are six terms each and leave out 2^-21 at most."""
    return size * (6 * terms + 16) * 2.0 ** -24
