"""GPU: attention over few query rows (paged caches, and contiguous ones with a
window and sinks) against plain attention in 64 bits: what is not finite in a cut
item's parts.

Tolerances are those of tests/test_gpu_paged.py: 1e-5 of a token's own scale."""
import numpy as np
import pytest

import paged_ref as R
from conftest import RTOL, rel_to_scale
from test_gpu_paged import Cache
from test_gpu_sinks import cache, call

pytestmark = pytest.mark.gpu

DTS = pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])


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
