"""Plain 64-bit forms of the paged cache and of attention with a window and
sinks, for the tests: loops over sequences and heads, no page left out."""
import numpy as np

TOP = {1: np.float32(127), 2: np.float32(7)}


def quantise(x, dt):
    """(codes as integers, fp32 scales) of vectors along the last axis: the scale
    and the quotient in fp32, halves away from zero (include/aero/kv.hpp:62-92)."""
    x = np.asarray(x, np.float32)
    amax = np.abs(x).max(-1)
    scale = np.where(amax > 0, amax / TOP[dt], np.float32(1)).astype(np.float32)
    r = (x / scale[..., None]).astype(np.float64)
    c = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -TOP[dt], TOP[dt])
    return c.astype(np.int8), scale


def pack(codes, dt):
    """Stored bytes of codes."""
    if dt == 1:
        return codes.view(np.uint8)
    c = codes.astype(np.uint8) & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)


def unpack(raw, dt):
    if dt == 1:
        return raw.view(np.int8)
    both = np.stack([raw & 15, raw >> 4], -1).reshape(*raw.shape[:-1], -1).astype(np.int8)
    return np.where(both > 7, both - 16, both).astype(np.int8)


def seen(qpos, kpos, window, sinks):
    qpos, kpos = np.asarray(qpos, np.int64)[:, None], np.asarray(kpos, np.int64)[None]
    keep = kpos <= qpos
    if window > 0:
        keep &= (qpos - kpos < window) | (kpos < sinks)
    return keep


def attention(q, K, V, keep, scale):
    """q [T, H, D], K [S, HK, D], V [S, HK, DV], keep [T, S] -> [T, H, DV] in
    float64; what is not kept is never touched."""
    q, K, V = (np.asarray(a, np.float64) for a in (q, K, V))
    T, H, _ = q.shape
    rep = H // K.shape[1]
    out = np.zeros((T, H, V.shape[2]))
    for t in range(T):
        at = np.nonzero(keep[t])[0]
        if at.size == 0:
            continue
        for kh in range(K.shape[1]):
            s = q[t, kh * rep:(kh + 1) * rep] @ K[at, kh].T * scale
            w = np.exp(s - s.max(1, keepdims=True))
            out[t, kh * rep:(kh + 1) * rep] = w @ V[at, kh] / w.sum(1, keepdims=True)
    return out
