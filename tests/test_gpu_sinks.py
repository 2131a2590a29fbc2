"""GPU: attention with a sliding window and sinks over contiguous caches
(ops.attention with sinks, aero_hip_attention_sinks) against plain attention in
64 bits, within 1e-5 of the output's scale (the contiguous attention's
tolerance; tests/test_gpu_paged.py has the arithmetic)."""
import numpy as np
import pytest

import paged_ref as R
from conftest import RTOL, bits_equal, rel_to_scale
from aero_amd import ops
from aero_amd.device import DeviceArray as DA, Plan, Stream, synchronize

pytestmark = pytest.mark.gpu


def cache(rng, n_kv, HK, D, dt):
    """(device array, scales or None, the values stored in float64)"""
    x = rng.standard_normal((n_kv, HK, D)).astype(np.float32)
    if dt == 0:
        return DA.from_numpy(x), None, x.astype(np.float64)
    c, s = R.quantise(x, dt)
    return (DA.from_numpy(R.pack(c, dt)), DA.from_numpy(s),
            c.astype(np.float64) * s[..., None].astype(np.float64))


def call(q, k, v, n_kv, HK, window, sinks, dt, qpos=None, kpos=None, scale=0.1, DV=None,
         stream=None):
    T, H, D = q.shape
    DV = DV or D
    out = DA.from_numpy(np.full((T, H, DV), 7.0, np.float32))
    dev = lambda a: None if a is None else DA.from_numpy(np.asarray(a, np.int32))
    ops.attention(DA.from_numpy(q), k[0], v[0], out, T, H, HK, D, DV, n_kv, scale, qpos=dev(qpos),
                  kpos=dev(kpos), window=window, kv_dt=dt, k_scale=k[1], v_scale=v[1],
                  stream=stream, sinks=sinks)
    if stream is not None:
        stream.synchronize()
    return out.numpy()


SHAPES = [
    # H, HK, D, DV, n_q, n_kv, window, sinks
    (32, 8, 128, 128, 1, 5000, 1000, 4), (32, 8, 128, 128, 1, 1, 1, 1), (14, 2, 64, 64, 1, 333, 64, 16),
    (8, 4, 256, 256, 1, 2052, 512, 4), (16, 2, 256, 256, 3, 700, 100, 33), (20, 1, 64, 64, 2, 90, 7, 1),
    (8, 8, 128, 128, 5, 300, 16, 16), (32, 8, 128, 128, 4, 4000, 33, 300), (4, 4, 80, 48, 1, 200, 30, 3),
    (4, 1, 32, 32, 70, 100, 11, 2), (6, 2, 20, 100, 9, 50, 49, 1), (32, 8, 64, 64, 257, 300, 100, 4),
    (32, 8, 128, 128, 200, 200, 1000, 4), (8, 4, 256, 256, 130, 600, 64, 5),
    (32, 8, 128, 128, 700, 700, 128, 20), (14, 2, 64, 64, 1001, 2500, 300, 64),
    (8, 4, 256, 256, 1400, 1400, 200, 4), (64, 8, 128, 128, 333, 3000, 90, 2000),
]


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_sinks(hip, shape, dt):
    H, HK, D, DV, T, n_kv, window, sinks = shape
    rng = np.random.default_rng([H, D, T, dt])
    k, v = cache(rng, n_kv, HK, D, dt), cache(rng, n_kv, HK, DV, dt)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    qpos = np.arange(n_kv - T, n_kv)
    got = call(q, k, v, n_kv, HK, window, sinks, dt, qpos, DV=DV)
    keep = R.seen(qpos, np.arange(n_kv), window, sinks)
    assert rel_to_scale(got, R.attention(q, k[2], v[2], keep, 0.1)) <= RTOL


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("D,T", [(64, 5), (128, 3), (256, 2), (48, 4), (128, 400)])
def test_positions(hip, D, T, dt):
    """Query positions in any order, before every key, at the sinks, past the
    cache; key positions of a ring and shuffled ones; absent positions."""
    rng = np.random.default_rng([D, T, dt])
    HK, H, n_kv, window, sinks = 2, 8, 400, 60, 6
    k, v = cache(rng, n_kv, HK, D, dt), cache(rng, n_kv, HK, D, dt)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    ring = np.arange(n_kv)
    ring[sinks:] = 1000 + (ring[sinks:] * 7) % (n_kv - sinks)
    for qpos in (None, rng.integers(-3, 900, T), np.full(T, 5), np.full(T, -1), np.full(T, 2**31 - 1),
                 np.resize([0, 399, 58, 1400], T)):
        for kpos in (None, ring, rng.permutation(n_kv)):
            got = call(q, k, v, n_kv, HK, window, sinks, dt, qpos, kpos)
            keep = R.seen(np.arange(T) if qpos is None else qpos,
                          np.arange(n_kv) if kpos is None else kpos, window, sinks)
            want = R.attention(q, k[2], v[2], keep, 0.1)
            assert np.isfinite(got).all()
            assert not got[~keep.any(1)].any()
            if want.any():
                assert rel_to_scale(got, want) <= RTOL


@pytest.mark.parametrize("D", [64, 128, 256, 48])
@pytest.mark.parametrize("T", [1, 4, 40, 600])
def test_values_that_no_query_may_see(hip, D, T):
    """NaN and infinities in keys and values that some or all queries do not keep
    reach none of those; one that a query keeps reaches that query."""
    rng = np.random.default_rng([D, T])
    H, HK, n_kv, window, sinks = 16, 4, 700, 50, 3
    k = rng.standard_normal((n_kv, HK, D)).astype(np.float32)
    v = rng.standard_normal((n_kv, HK, D)).astype(np.float32)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    qpos = np.arange(n_kv - T, n_kv)
    hidden = ~R.seen(qpos, np.arange(n_kv), window, sinks).any(0)
    k[hidden], v[hidden] = np.nan, np.inf
    v[n_kv - 1] = np.inf                      # only the last query keeps it
    k[n_kv - 1, 1] = np.nan
    dev = lambda x: (DA.from_numpy(x), None)
    got = call(q, dev(k), dev(v), n_kv, HK, window, sinks, 0, qpos)
    keep = R.seen(qpos, np.arange(n_kv), window, sinks)
    if T > 1:
        want = R.attention(q[:-1], k, v, keep[:-1], 0.1)
        assert np.isfinite(got[:-1]).all()
        assert rel_to_scale(got[:-1], want) <= RTOL
    assert not np.isfinite(got[-1]).any()


@pytest.mark.parametrize("dt", [0, 1], ids=["fp32", "int8"])
def test_without_window_or_sinks_it_is_attention(hip, dt):
    rng = np.random.default_rng(dt)
    k, v = cache(rng, 500, 2, 128, dt), cache(rng, 500, 2, 128, dt)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    qpos = np.arange(497, 500)
    a = call(q, k, v, 500, 2, 0, 0, dt, qpos)
    assert bits_equal(a, call(q, k, v, 500, 2, 0, 9, dt, qpos))
    # sinks past the window's first key add nothing to its keys
    want = R.attention(q, k[2], v[2], R.seen(qpos, np.arange(500), 1 << 30, 7), 0.1)
    assert rel_to_scale(call(q, k, v, 500, 2, 1 << 30, 7, dt, qpos), want) <= RTOL
    # the same bits twice, and on another stream
    b = call(q, k, v, 500, 2, 100, 4, dt, qpos)
    s = Stream()
    assert bits_equal(b, call(q, k, v, 500, 2, 100, 4, dt, qpos))
    assert bits_equal(b, call(q, k, v, 500, 2, 100, 4, dt, qpos, stream=s))
    s.destroy()


@pytest.mark.parametrize("dt", [0, 1], ids=["fp32", "int8"])
def test_recorded_step(hip, dt):
    """One token's step over a ring with sinks, recorded; positions move on
    between the replays."""
    rng = np.random.default_rng(40 + dt)
    H, HK, D, window, sinks = 32, 8, 128, 512, 4
    n_kv = window + sinks
    k, v = cache(rng, n_kv, HK, D, dt), cache(rng, n_kv, HK, D, dt)
    q = rng.standard_normal((1, H, D)).astype(np.float32)
    dq, out = DA.from_numpy(q), DA.empty((1, H, D))
    qp, kp = DA.empty(1, np.int32), DA.empty(n_kv, np.int32)
    plan = Plan()
    with plan:
        ops.attention(dq, k[0], v[0], out, 1, H, HK, D, D, n_kv, 0.1, qpos=qp, kpos=kp,
                      window=window, kv_dt=dt, k_scale=k[1], v_scale=v[1], sinks=sinks)
    slots = np.arange(n_kv)
    for last in (600, 601, 1300, 5000):
        newest = last - (last - sinks - (slots - sinks)) % window
        kpos = np.where(slots < sinks, slots, newest)
        qp.copy_from(np.asarray([last], np.int32))
        kp.copy_from(kpos.astype(np.int32))
        plan.launch()
        want = R.attention(q, k[2], v[2], R.seen([last], kpos, window, sinks), 0.1)
        got = out.numpy()
        assert rel_to_scale(got, want) <= RTOL
        assert bits_equal(got, call(q, k, v, n_kv, HK, window, sinks, dt, [last], kpos))
    plan.destroy()


# Calls with enough query vectors for the prompt kernels (128 workgroups and more):
# every width, and one, two and four waves on the same queries.
PROMPTS = [(64, 16, 32, 500), (64, 32, 64, 500), (64, 64, 128, 400), (128, 16, 16, 900),
           (128, 64, 128, 400), (256, 32, 32, 420)]
PROMPT_IDS = ["-".join(map(str, s)) for s in PROMPTS]


def values(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def heads_of(q, HK, heads):
    """The query heads of the kv heads `heads` (the oracle need not do them all)."""
    rep = q.shape[1] // HK
    return np.concatenate([np.arange(h * rep, (h + 1) * rep) for h in heads])


def prompt(q, k, v, qpos, window, sinks, scale=0.1, kpos=None, heads=(0, -1)):
    """(got, want, keep) for the query heads of the kv heads `heads`."""
    HK, n_kv = k.shape[1], k.shape[0]
    heads = [h % HK for h in heads]
    got = call(q, (DA.from_numpy(k), None), (DA.from_numpy(v), None), n_kv, HK, window, sinks, 0,
               qpos, kpos, scale)
    keep = R.seen(np.arange(len(q)) if qpos is None else qpos,
                  np.arange(n_kv) if kpos is None else kpos, window, sinks)
    at = heads_of(q, HK, heads)
    return got[:, at], R.attention(q[:, at], k[:, heads], v[:, heads], keep, scale), keep


@pytest.mark.parametrize("shape", PROMPTS, ids=PROMPT_IDS)
def test_prompt_positions(hip, shape):
    """Consecutive positions from 0 and from the middle of a 32-key tile on; in any
    order and too far apart for the tiles there is room for; key positions of a
    ring, shuffled and absent."""
    D, HK, H, T = shape
    rng = np.random.default_rng([D, H, T])
    window, sinks, n_kv = 70, 5, T + 1500
    k, v, q = values(rng, n_kv, HK, D), values(rng, n_kv, HK, D), values(rng, T, H, D)
    short = 300
    ring = np.arange(short)
    ring[sinks:] = 900 + (ring[sinks:] * 7) % (short - sinks)
    for qpos, kpos in ((None, None), (np.arange(1217, 1217 + T), None),
                       (rng.permutation(T) + 900, None), (rng.integers(-5, n_kv + 50, T), None),
                       (np.full(T, -1), None), (np.full(T, 2**31 - 1), None),
                       (rng.integers(880, 1250, T), ring), (np.arange(T), rng.permutation(short)),
                       (np.arange(T) - 40, np.full(short, 2**31 - 1))):
        n = n_kv if kpos is None else short
        got, want, keep = prompt(q, k[:n], v[:n], qpos, window, sinks, kpos=kpos)
        assert np.isfinite(got).all()
        assert not got[~keep.any(1)].any()
        if want.any():
            assert rel_to_scale(got, want) <= RTOL


@pytest.mark.parametrize("shape", PROMPTS, ids=PROMPT_IDS)
def test_prompt_values(hip, shape):
    """NaN and infinities that nobody keeps stay out; one that the last query keeps
    reaches it alone, within a tile that others keep keys of."""
    D, HK, H, T = shape
    rng = np.random.default_rng([D, H, T, 1])
    window, sinks, n_kv = 50, 3, T + 100
    k, v, q = values(rng, n_kv, HK, D), values(rng, n_kv, HK, D), values(rng, T, H, D)
    qpos = np.arange(n_kv - T, n_kv)
    hidden = ~R.seen(qpos, np.arange(n_kv), window, sinks).any(0)
    k[hidden], v[hidden] = np.nan, np.inf
    got, want, _ = prompt(q, k, v, qpos, window, sinks)
    assert np.isfinite(got).all()
    assert rel_to_scale(got, want) <= RTOL
    v[n_kv - 1] = np.inf
    k[n_kv - 1, 1] = np.nan
    got, want, _ = prompt(q[:, :H], k, v, qpos, window, sinks)
    assert np.isfinite(got[:-1]).all()
    assert rel_to_scale(got[:-1], want[:-1]) <= RTOL
    assert not np.isfinite(got[-1]).any()
    q[T // 2, 0, 1] = np.nan       # a query's own
    got, want, _ = prompt(q, k, v, qpos, window, sinks)
    assert np.isnan(got[T // 2, 0]).all()
    ok = np.ones(T, bool)
    ok[[T // 2, T - 1]] = False
    assert rel_to_scale(got[ok], want[ok]) <= RTOL


@pytest.mark.parametrize("shape", PROMPTS, ids=PROMPT_IDS)
@pytest.mark.parametrize("what", ["rows", "dimensions", "tiny", "huge"])
def test_prompt_ranges(hip, shape, what):
    """Values far apart in size: each part of the result to its own scale. (Of 50
    kept values of one size the largest error is a few units of 2^-22 of it, as
    where all are of a size.)"""
    D, HK, H, T = shape
    rng = np.random.default_rng([D, H, T, 2])
    window, sinks, n_kv = 50, 3, T + 100
    k, v, q = values(rng, n_kv, HK, D), values(rng, n_kv, HK, D), values(rng, T, H, D)
    qpos = np.arange(n_kv - T, n_kv)
    if what == "rows":             # the first keys' and a run's in the middle, sinks too
        v[:n_kv // 2] *= np.float32(2.0**-30)
    elif what == "dimensions":
        v[:, :, ::3] *= np.float32(2.0**-40)
    elif what == "tiny":
        v *= np.float32(2.0**-100)
        k *= np.float32(2.0**-100)
        q *= np.float32(2.0**60)
    else:
        v *= np.float32(2.0**100)
        k *= np.float32(2.0**60)
        q *= np.float32(2.0**-60)
    got, want, _ = prompt(q, k, v, qpos, window, sinks)
    if what == "rows":
        # queries that keep small values alone, and those that keep a large one
        small = np.abs(want).max((1, 2)) < 2.0**-20
        assert small.any() and not small.all()
        assert rel_to_scale(got[small], want[small]) <= RTOL
        assert rel_to_scale(got[~small], want[~small]) <= RTOL
    elif what == "dimensions":
        assert rel_to_scale(got[..., ::3], want[..., ::3]) <= RTOL
        assert rel_to_scale(got[..., 1::3], want[..., 1::3]) <= RTOL
    else:
        assert rel_to_scale(got * np.float32(1 / np.abs(want).max()),
                            want / np.abs(want).max()) <= RTOL


@pytest.mark.parametrize("shape", PROMPTS, ids=PROMPT_IDS)
def test_prompt_large_scores(hip, shape):
    """Scores of thousands. A score's error in fp32 is at most e = (D + 3) 2^-24 of
    scale * sum |q k|, a probability's e^(2e) - 1 of it, and the output's that of
    the largest value, twice (numerator and sum)."""
    D, HK, H, T = shape
    rng = np.random.default_rng([D, H, T, 3])
    window, sinks, n_kv = 50, 3, T + 100
    k, v, q = values(rng, n_kv, HK, D), values(rng, n_kv, HK, D), values(rng, T, H, D)
    q *= np.float32(1600 / D**0.5)
    qpos = np.arange(n_kv - T, n_kv)
    got, want, keep = prompt(q, k, v, qpos, window, sinks, scale=1.0, heads=(0,))
    size = np.einsum("thd,kd->thk", np.abs(q[:, :H // HK]).astype(np.float64), np.abs(k[:, 0]))
    e = (D + 3) * 2.0**-24 * (size * keep[:, None]).max(2)
    limit = 2 * np.expm1(2 * e) * np.abs(v[:, 0]).max()
    assert (np.abs(got - want).max(2) <= limit).all()


def test_prompt_recorded(hip):
    """A prompt's chunk recorded; positions and cache rows move on between the
    replays, which each give the eager call's bits."""
    rng = np.random.default_rng(50)
    H, HK, D, T, n_kv, window, sinks = 32, 16, 64, 500, 1600, 200, 4
    k, v, q = values(rng, n_kv, HK, D), values(rng, n_kv, HK, D), values(rng, T, H, D)
    dk, dv, dq, out = DA.from_numpy(k), DA.from_numpy(v), DA.from_numpy(q), DA.empty((T, H, D))
    qp = DA.empty(T, np.int32)
    plan = Plan()
    with plan:
        ops.attention(dq, dk, dv, out, T, H, HK, D, D, n_kv, 0.1, qpos=qp, window=window,
                      sinks=sinks)
    for first in (0, 500, 1000, 333):
        k[first:first + T] *= np.float32(0.5)
        dk.copy_from(k)
        qpos = np.arange(first, first + T)
        qp.copy_from(qpos.astype(np.int32))
        plan.launch()
        got = out.numpy()
        eager, want, _ = prompt(q, k, v, qpos, window, sinks)
        at = heads_of(q, HK, (0, HK - 1))
        assert bits_equal(got[:, at], eager)
        assert rel_to_scale(eager, want) <= RTOL
    plan.destroy()


def test_more_tiles_than_a_grid_side(hip):
    """70,000 tokens of four heads: 70,000 query tiles of one kv head; the rows at
    both ends and around the 65,535th tile."""
    rng = np.random.default_rng(60)
    T, H, D, window, sinks = 70000, 4, 8, 5, 2
    k, v = cache(rng, T, 1, D, 1), cache(rng, T, 1, D, 1)
    q = values(rng, T, H, D)
    qpos = np.arange(T)
    got = call(q, k, v, T, 1, window, sinks, 1, qpos)
    at = np.r_[0:40, T - 65535 - 20:T - 65535 + 20, 65515:65555, T - 40:T]
    want = R.attention(q[at], k[2], v[2], R.seen(qpos[at], qpos, window, sinks), 0.1)
    assert rel_to_scale(got[at], want) <= RTOL
    assert np.isfinite(got).all() and np.abs(got).max(2).min() > 0


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("D", [64, 128, 256, 48])
@pytest.mark.parametrize("e", [-140, -100, 90])
def test_sizes_of_queries(hip, dt, D, e):
    """Queries of 2^e, one row of them zeros, at the scale that undoes it as far as a
    scale of normal floats can."""
    rng = np.random.default_rng([D, dt, e + 200])
    H, HK, T, n_kv, window, sinks = 8, 2, 3, 700, 300, 4
    k, v = cache(rng, n_kv, HK, D, dt), cache(rng, n_kv, HK, D, dt)
    q = np.ldexp(values(rng, T, H, D), e).astype(np.float32)
    q[1, 3] = 0
    qpos = np.arange(n_kv - T, n_kv)
    scale = float(np.float32(min(np.ldexp(0.1, -e), 2.0**120)))
    got = call(q, k, v, n_kv, HK, window, sinks, dt, qpos, scale=scale)
    keep = R.seen(qpos, np.arange(n_kv), window, sinks)
    assert rel_to_scale(got, R.attention(q, k[2], v[2], keep, scale)) <= RTOL


@pytest.mark.parametrize("dt", [1, 2], ids=["int8", "int4"])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 5), (256, 2), (128, 70)])
def test_sizes_of_scales(hip, dt, D, T):
    """Value scales that fall and rise by 2^40 along the keys, key scales by 2^10:
    each query to the scale of what it keeps."""
    rng = np.random.default_rng([D, T, dt, 9])
    H, HK, n_kv, window, sinks = 8, 2, 900, 64, 3
    k, v = cache(rng, n_kv, HK, D, dt), cache(rng, n_kv, HK, D, dt)
    for step, qpos in ((300, np.sort(rng.integers(0, n_kv, T))), (64, np.arange(n_kv - T, n_kv))):
        ev = -40 * ((np.arange(n_kv) // step) % 2)
        ek = -10 * ((np.arange(n_kv) // 50) % 2)
        ks = np.ldexp(k[1].numpy(), ek[:, None]).astype(np.float32)
        vs = np.ldexp(v[1].numpy(), ev[:, None]).astype(np.float32)
        K, V = np.ldexp(k[2], ek[:, None, None]), np.ldexp(v[2], ev[:, None, None])
        q = values(rng, T, H, D)
        got = call(q, (k[0], DA.from_numpy(ks)), (v[0], DA.from_numpy(vs)), n_kv, HK, window,
                   sinks, dt, qpos)
        want = R.attention(q, K, V, R.seen(qpos, np.arange(n_kv), window, sinks), 0.1)
        for t in range(T):
            assert rel_to_scale(got[t], want[t]) <= RTOL, (step, t)


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("D,DV", [(80, 80), (96, 96), (192, 128), (16, 240), (40, 104), (72, 100),
                                  (8, 8), (252, 4)])
@pytest.mark.parametrize("T", [1, 37])
def test_widths(hip, D, DV, T, dt):
    """Other widths, with and without key positions; values that no query keeps
    are not finite (fp32)."""
    rng = np.random.default_rng([D, DV, T, dt])
    HK, H, n_kv, window, sinks = 3, 6, 650, 300, 5
    k, v = cache(rng, n_kv, HK, D, dt), cache(rng, n_kv, HK, DV, dt)
    q = values(rng, T, H, D)
    qpos = np.arange(n_kv - T, n_kv)
    keep = R.seen(qpos, np.arange(n_kv), window, sinks)
    if dt == 0:
        for x, bad in ((k, np.nan), (v, np.inf)):
            a = x[0].numpy().copy()
            a[~keep.any(0)] = bad
            x[0].copy_from(a)
    want = R.attention(q, k[2], v[2], keep, 0.1)
    for kpos in (None, np.arange(n_kv)):
        got = call(q, k, v, n_kv, HK, window, sinks, dt, qpos, kpos, DV=DV)
        assert rel_to_scale(got, want) <= RTOL


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("D,T,n_kv", [(128, 2, 300), (64, 600, 700), (256, 1, 2000)])
def test_rows_that_are_not_aligned(hip, D, T, n_kv, dt):
    """Queries and outputs at any 4-byte address, codes at any byte (fp32 caches
    are refused then), prompts among them."""
    from test_gpu_paged import shifted
    rng = np.random.default_rng([D, T, dt, 5])
    HK, H, window, sinks = 16, 32, 100, 4
    k, v = cache(rng, n_kv, HK, D, dt), cache(rng, n_kv, HK, D, dt)
    q = values(rng, T, H, D)
    qpos = np.arange(n_kv - T, n_kv)
    at = np.r_[0:T:max(1, T // 20), T - 1]
    want = R.attention(q[at], k[2], v[2], R.seen(qpos[at], np.arange(n_kv), window, sinks), 0.1)
    dq, qp = DA.from_numpy(q), DA.from_numpy(qpos.astype(np.int32))
    blank = np.ones((T, H, D), np.float32)
    for dq, out, dk, dv in ((shifted(q), DA.empty((T, H, D)), k[0], v[0]),
                            (dq, shifted(blank), k[0], v[0]),
                            (dq, DA.empty((T, H, D)), shifted(k[0].numpy()), v[0]),
                            (dq, DA.empty((T, H, D)), k[0], shifted(v[0].numpy()))):
        run = lambda: ops.attention(dq, dk, dv, out, T, H, HK, D, D, n_kv, 0.1, qpos=qp,
                                    window=window, kv_dt=dt, k_scale=k[1], v_scale=v[1],
                                    sinks=sinks)
        if dt == 0 and (dk is not k[0] or dv is not v[0]):
            with pytest.raises(Exception, match="aligned"):
                run()
            continue
        run()
        assert rel_to_scale(out.numpy()[at], want) <= RTOL
