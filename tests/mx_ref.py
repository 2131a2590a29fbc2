"""Plain 64-bit forms of microscaled rows, for the tests: decoded by tables, quantised by
looking for the nearest code."""
import numpy as np

INT8, FP4 = 0, 1
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)
TOP = {INT8: 127 / 64, FP4: 6.0}
LOW = {INT8: 4, FP4: 0}


def quantise(x, fmt):
    """(codes as stored, scale bytes) of fp32 rows."""
    x = np.asarray(x, np.float32).astype(np.float64)
    rows, cols = x.shape
    b = x.reshape(rows, cols // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    amax = np.abs(b).max(-1)
    s = np.full(amax.shape, LOW[fmt])
    for byte in range(LOW[fmt], 254):      # the smallest scale that holds the block, 254 at most
        s = np.where(amax > TOP[fmt] * 2.0 ** (byte - 127), byte + 1, s)
    q = np.ldexp(b, (127 - s)[..., None])
    if fmt == INT8:
        c = np.clip(np.rint(q * 64), -127, 127).astype(np.int8)
    else:
        middle = (GRID[1:] + GRID[:-1]) / 2
        a = np.abs(q)[..., None]
        even = np.arange(7) % 2 == 1       # at the middle: up where the upper code is even
        c = ((a > middle) | ((a == middle) & even)).sum(-1).astype(np.uint8)
        c |= np.signbit(q).astype(np.uint8) << 3
    c = np.where(bad[..., None], 0, c)
    s = np.where(bad, 255, s).astype(np.uint8)
    return pack(c.reshape(rows, cols), fmt), s


def pack(codes, fmt):
    if fmt == INT8:
        return codes.astype(np.int8)
    codes = codes.astype(np.uint8)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def values(codes, s, fmt):
    """float64 rows that stored codes and scales stand for."""
    if fmt == FP4:
        c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
        v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    else:
        v = codes.astype(np.float64) / 64
    scale = np.where(s == 255, np.nan, 2.0 ** (s.astype(np.float64) - 127))
    return (v.reshape(*s.shape, 32) * scale[..., None]).reshape(codes.shape[0], -1)


def norm(x, w, eps, unit):
    """fp32 rows of rmsnorm in 64 bits."""
    with np.errstate(invalid="ignore", over="ignore"):
        v = x.astype(np.float64)
        v = v / np.sqrt((v * v).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        if w is not None:
            v = v * (w.astype(np.float64) + (1.0 if unit else 0.0))
        return v.astype(np.float32)


def act(kind, v):
    v = v.astype(np.float64)
    if kind == "silu":
        return v / (1 + np.exp(-v))
    if kind == "sigmoid":
        return 1 / (1 + np.exp(-v))
    if kind == "identity":
        return v
    if kind == "gelu_tanh":
        return v / (1 + np.exp(-2 * 0.7978845608028654 * (v + 0.044715 * v ** 3)))
    t = 1 / (1 + 0.3275911 * np.abs(v) * 0.7071067811865476)
    p = ((((1.061405429 * t - 1.453152027) * t + 1.421413741) * t - 0.284496736) * t
         + 0.254829592) * t * np.exp(-v * v / 2)
    return 0.5 * v * np.where(v < 0, p, 2 - p)
