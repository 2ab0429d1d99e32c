"""AdamW in 64 bits, and the 8-bit moments restated on numpy integers: what the kernels are compared with."""
import numpy as np

U = 2.0 ** -24  # half a step of float32, relative


def step64(p, g, m, v, t, lr, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2, factor=1.0):
    """(p, m, v, bounds): one step in float64 and how far a float32 evaluation may be off each.

    m: b1, 1 - b1 and the factor as float32, the products and the sum round once each (with a factor the gradient's product too, and the factor
    itself carries the norm's error: eight float32 additions of squares, a root and three roundings). v likewise with the factor
    twice. p: two products and a difference, the update with its root, product, sum, quotient and product, and with m's and
    half of v's error."""
    g = g * factor
    clip = 0 if factor is None or factor == 1.0 else 10
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    off_m = (4 + clip) * U * (b1 * abs(m) + (1 - b1) * abs(g))
    # 1 - b2 as float32 of 1 - 0.999 has the relative error of any float32
    off_v = (6 + 2 * clip) * U * v1
    scale, root = lr / (1 - b1 ** t), 1 / np.sqrt(1 - b2 ** t)
    denominator = np.sqrt(v1) * root + eps
    with np.errstate(divide='ignore', invalid='ignore'):
        update = scale * m1 / denominator
        off_p = 3 * U * abs(p) + scale * off_m / denominator + abs(update) * (10 + clip + 3) * U
    p1 = p * (1 - lr * wd) - update
    return p1, m1, v1, (off_p + U * abs(p1), off_m, off_v)


def _mix(x):
    x = x.astype(np.uint32)
    with np.errstate(over='ignore'):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0xBB67AE85)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0x3C6EF373)
    return x ^ (x >> np.uint32(16))


def noise(n, t, seed, first=0):
    """The two numbers in [0, 1) of every element, from `first` on."""
    key = _mix(np.array([(t + seed * 0x9E3779B1) & 0xFFFFFFFF], dtype=np.uint64))[0]
    at = (np.arange(first, first + n, dtype=np.uint64) * np.uint64(0x9E3779B1) + np.uint64(key)) & np.uint64(0xFFFFFFFF)
    h = _mix(at)
    return (h & np.uint32(0xFFFF)).astype(np.float64) / 65536, (h >> np.uint32(16)).astype(np.float64) / 65536


def magnitudes(bits):
    """What the codes stand for in units of the largest binade's power of two; `bits` of exponent, three of fraction."""
    codes = np.arange(8 << bits)
    exponent, fraction = codes >> 3, codes & 7
    return np.where(exponent == 0, fraction / 8, (1 + fraction / 8) * 2.0 ** (exponent - 1.0)) * 2.0 ** (2 - (1 << bits))


def unpack(state, n):
    """(m, v) in float64 of a state's bytes."""
    b = (n + 255) // 256
    state = np.asarray(state)
    exponents = state[512 * b:].reshape(b, 2).astype(np.float64)
    codes = state[:512 * b].reshape(2, b, 256).astype(np.int64)
    m = magnitudes(4)[codes[0] & 127] * np.where(codes[0] > 127, -1, 1) * 2.0 ** (exponents[:, :1] - 127)
    v = magnitudes(5)[codes[1]] * 2.0 ** (exponents[:, 1:] - 127)
    m[exponents[:, 0] == 255], v[exponents[:, 1] == 255] = np.nan, np.nan
    return m.reshape(-1)[:n], v.reshape(-1)[:n]


def rounded(x, u, bits):
    """(kept, spacing) of x >= 0 in blocks of 256: rounded down after u spacings have been added, at most the largest code's value."""
    n = len(x)
    b = (n + 255) // 256
    pad = lambda a: np.concatenate([a, np.zeros(b * 256 - n)]).reshape(b, 256)
    x, u = pad(x), pad(u)
    top = x.max(axis=1, keepdims=True)
    highest = np.where(top > 0, np.floor(np.log2(np.maximum(top, 2.0 ** -126))), -126)
    highest = highest + (top > 1.875 * 2.0 ** highest)
    binade = np.maximum(np.floor(np.log2(np.maximum(x, 2.0 ** -300))), highest - ((1 << bits) - 2))
    spacing = 2.0 ** (binade - 3)
    kept = np.minimum(np.floor(x / spacing + u) * spacing, 2.0 ** highest * (2 - 1 / 8))
    return kept.reshape(-1)[:n], spacing.reshape(-1)[:n]
