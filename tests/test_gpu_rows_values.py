"""GPU: attention over few query rows (paged caches, and contiguous ones with a
window and sinks) where the values are not of a size, against plain attention in
64 bits: what is not finite in a cut item's parts, and integer caches whose value
scales lie far apart.

Tolerances are those of tests/test_gpu_paged.py: 1e-5 of a token's own scale."""
import numpy as np
import pytest

import paged_ref as R
from conftest import RTOL, rel_to_scale
from test_gpu_paged import Cache
from test_gpu_sinks import cache, call
from aero_amd.device import DeviceArray as DA

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
INTS = pytest.mark.parametrize("dt", [1, 2], ids=["int8", "int4"])


def by_token(got, want, which=None):
    """Every token's rows (of `which`) finite and within RTOL of their own scale."""
    for t in np.ndindex(got.shape[:-2]):
        if which is None or which[t]:
            assert np.isfinite(got[t]).all(), t
            assert rel_to_scale(got[t], want[t]) <= RTOL, (t, rel_to_scale(got[t], want[t]))


# ------------------------------------------------------- parts that are not finite
# (the longest sequence and the window are well past the keys that stay one part: 20
# and more parts an item, in some of the widths 8 of a lane group in flight)
N, WINDOW, SINKS = 3000, 2500, 4
BAD = slice(800, 1400)      # keys: a whole part of any variant, and more


@DTS
@pytest.mark.parametrize("D", [64, 128, 256, 20])
@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_queries_that_are_not_finite(hip, D, T, dt, bad):
    """A query of NaN or an infinity gives NaN, cut or not; its neighbours' results
    are their own."""
    rng = np.random.default_rng([D, T, dt, 70])
    H, HK = 8, 2
    c = Cache(rng, dt, 16, HK, D, D, [N, 100])
    q = rng.standard_normal((2, T, H, D)).astype(np.float32)
    want = c.ref(q, 0.1)
    keep = np.ones((2, T, H), bool)
    for s in range(2):           # cut, and of one part
        q[s, T - 1, 5, D // 2] = bad
        keep[s, T - 1, 5] = False
    got = c.attend(q, 0.1)
    assert np.isnan(got[~keep]).all()
    got[~keep] = want[~keep]
    by_token(got, want)

    k, v = cache(rng, N, HK, D, dt), cache(rng, N, HK, D, dt)
    qpos = np.arange(N - T, N)
    seen = R.seen(qpos, np.arange(N), WINDOW, SINKS)
    for kpos in (None, np.arange(N)):
        got = call(q[0], k, v, N, HK, WINDOW, SINKS, dt, qpos, kpos)
        want = R.attention(np.where(np.isfinite(q[0]), q[0], 0), k[2], v[2], seen, 0.1)
        assert np.isnan(got[~keep[0]]).all()
        got[~keep[0]] = want[~keep[0]]
        by_token(got, want)


@DTS
@pytest.mark.parametrize("D", [64, 128, 256, 20])
@pytest.mark.parametrize("T", [1, 4])
def test_parts_of_nan_keys(hip, D, T, dt):
    """Keys of NaN (their scales, in integer caches) that fill whole parts of one kv
    head: every query of that head that keeps them is NaN, the other head's are right."""
    rng = np.random.default_rng([D, T, dt, 71])
    H, HK = 8, 2
    c = Cache(rng, dt, 16, HK, D, D, [N, 100])
    pos = np.arange(N)[BAD]
    a = (c.raw if dt == 0 else c.scales)[0]
    a[0, c.table[0, pos // 16], 1, pos % 16] = np.nan
    (c.pool.k if dt == 0 else c.pool.k_scale).copy_from(a)
    q = rng.standard_normal((2, T, H, D)).astype(np.float32)
    got, want = c.attend(q, 0.1), c.ref(q, 0.1)
    assert np.isnan(got[0, :, H // 2:]).all()
    by_token(got[:1, :, :H // 2], want[:1, :, :H // 2])
    by_token(got[1:], want[1:])

    k, v = cache(rng, N, HK, D, dt), cache(rng, N, HK, D, dt)
    a = (k[0] if dt == 0 else k[1]).numpy().copy()
    a[BAD, 1] = np.nan
    (k[0] if dt == 0 else k[1]).copy_from(a)
    qpos = np.arange(N - T, N)
    got = call(q[0], k, v, N, HK, WINDOW, SINKS, dt, qpos)
    want = R.attention(q[0], k[2], v[2], R.seen(qpos, np.arange(N), WINDOW, SINKS), 0.1)
    assert np.isnan(got[:, H // 2:]).all()
    by_token(got[:, :H // 2], want[:, :H // 2])


# --------------------------------------------- value scales far apart (integer caches)
def scaled_values(c, dt, power):
    """The cache's values times 2^power[j] at key j of every sequence."""
    a = c.scales[1]
    for s, n in enumerate(c.lens):
        j = np.arange(n)
        at = (c.layer, c.table[s, j // c.page], slice(None), j % c.page)
        a[at] = np.ldexp(a[at], power[:n, None])
        c.V[s] = np.ldexp(c.V[s], power[:n, None, None])
    c.pool.v_scale.copy_from(a)


@INTS
@pytest.mark.parametrize("D", [64, 128, 256, 80, 20])
@pytest.mark.parametrize("low", [-14, -24, -40, -100])
@pytest.mark.parametrize("window", [0, 5])
def test_tokens_that_keep_small_values_alone(hip, D, low, window, dt):
    """Tokens of one tile on both sides of a step of the value scales, up and (in a
    window) down: each token's result has the bits of what it keeps."""
    rng = np.random.default_rng([D, -low, dt, window])
    H, HK, n, T = 8, 2, 300, 11
    q = rng.standard_normal((1, T, H, D)).astype(np.float32)
    pos = np.arange(n - T, n)
    for first, last in ((low, 0), (0, low)) if window else ((low, 0),):
        c = Cache(rng, dt, 16, HK, D, D, [n])
        power = np.where(np.arange(n) < n - T // 2, first, last)
        scaled_values(c, dt, power)
        want = c.ref(q, 0.1, window)
        small = np.abs(want).max((0, 2, 3)) < 2.0 ** (low / 2 - 4)
        # tokens that keep small values alone, beside others in their tile of 16 / 4
        assert any(small[t:t + 4].any() and not small[t:t + 4].all() for t in range(0, T, 4))
        by_token(c.attend(q, 0.1, window), want)
        # the same over a contiguous cache; its sink keeps the small side
        if window:
            j = np.arange(n)
            at = (0, c.table[0, j // 16], slice(None), j % 16)
            power[0] = low
            vs = np.ldexp(c.scales[1][at], (power - np.where(j < n - T // 2, first, last))[:, None])
            V = c.V[0] * (vs / c.scales[1][at])[..., None]
            got = call(q[0], (DA.from_numpy(c.raw[0][at]), DA.from_numpy(c.scales[0][at])),
                       (DA.from_numpy(c.raw[1][at]), DA.from_numpy(vs)), n, HK, window, 1, dt, pos)
            by_token(got, R.attention(q[0], c.K[0], V, R.seen(pos, j, window, 1), 0.1))


@INTS
@pytest.mark.parametrize("D", [64, 128, 256, 80])
@pytest.mark.parametrize("up", [16, 30, 60])
def test_large_values_of_no_weight(hip, D, up, dt):
    """Keys with values 2^up times the others' and a weight below 2^-70: the result
    has the bits of the others, wherever those keys lie."""
    rng = np.random.default_rng([D, up, dt])
    HK, n = 4, 900
    q = rng.standard_normal((1, 1, HK, D)).astype(np.float32)
    for far in ([3], [n - 1], list(range(0, n, 33))):
        c = Cache(rng, dt, 16, HK, D, D, [n])
        # keys against their head's query: a score of -6 |q|
        size = np.linalg.norm(q[0, 0], axis=1)
        codes, sc = R.quantise(-q[0, 0], dt)
        sc = (sc * (600 + 10 * up) / size**2).astype(np.float32)
        at = (0, c.table[0, np.asarray(far) // 16], slice(None), np.asarray(far) % 16)
        c.raw[0][at], c.scales[0][at] = R.pack(codes, dt), sc
        c.K[0][far] = codes.astype(np.float64) * sc[:, None].astype(np.float64)
        c.pool.k.copy_from(c.raw[0])
        c.pool.k_scale.copy_from(c.scales[0])
        power = np.zeros(n, np.int32)
        power[far] = up
        scaled_values(c, dt, power)
        s = np.einsum("hd,jhd->jh", q[0, 0], c.K[0]) * 0.1
        assert (s[far] - s.max(0) < -(70 + up) * np.log(2)).all()
        by_token(c.attend(q, 0.1), c.ref(q, 0.1))


@INTS
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_scale_that_is_not_finite_stays_with_its_token(hip, dt, bad):
    """The newest token's value scale is not finite: it alone loses its result,
    whatever the size of the others' values."""
    rng = np.random.default_rng([dt, 72])
    H, HK, D, n, T = 8, 2, 128, 300, 4
    for power in (-60, 0, 20, 100):
        c = Cache(rng, dt, 16, HK, D, D, [n])
        scaled_values(c, dt, np.full(n, power))
        c.scales[1][0, c.table[0, (n - 1) // 16], :, (n - 1) % 16] = bad
        c.pool.v_scale.copy_from(c.scales[1])
        q = rng.standard_normal((1, T, H, D)).astype(np.float32)
        got, want = c.attend(q, 0.1), c.ref(q, 0.1)
        assert not np.isfinite(got[0, T - 1]).any()
        by_token(got[:, :T - 1] / np.float32(2.0**power), want[:, :T - 1] / 2.0**power)
