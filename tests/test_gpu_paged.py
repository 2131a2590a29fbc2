"""GPU: the paged KV cache (aero_amd/paged.py, ops.paged_* and kv_pages_copy)
against plain 64-bit forms (tests/paged_ref.py).

Attention: <= 1e-5 of the output's scale, the tolerance of the contiguous
attention's tests (tests/test_gpu_attention.py). Where it comes from: a score of
D products rounds by about sqrt(D) 2^-24 of sum |q k| scale (D = 256: 1e-6 of
scores of a few units), which is a probability's relative error; the sums of p v
over n keys add sqrt(n) 2^-24 of the largest term and the splits 2^-22 an
operand: some 1e-6 in all, below 1e-5 with room for the largest of many rows.
Rows written: codes, scales and fp32 rows bit for bit. Copies: bit for bit.

Everything that no query may see is poisoned: NaN in fp32 pages, NaN scales and
arbitrary codes in integer ones."""
import numpy as np
import pytest

import paged_ref as R
from conftest import RTOL, bits_equal, rel_to_scale
from aero_amd import _lib, ops, paged
from aero_amd.device import DeviceArray as DA, Plan, Stream, synchronize, tune_set

pytestmark = pytest.mark.gpu


class Cache:
    """Sequences of `lens` tokens in shuffled pages of a poisoned pool; K, V hold
    the values stored, per sequence, in float64."""

    def __init__(self, rng, dt, page, HK, D, DV, lens, n_layers=1, layer=0, spare=3,
                 max_pages=None, k_mul=1.0):
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        self.dt, self.page, self.lens, self.layer = dt, page, np.asarray(lens, np.int32), layer
        self.max_pages = max_pages or max(1, max(need))
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), self.max_pages), -1, np.int32)
        shape = (n_layers, self.n_pages, HK, page)
        raw, scales, vals = [], [], []
        for dim, mul in ((D, k_mul), (DV, 1.0)):
            if dt == 0:
                raw.append(np.full((*shape, dim), np.nan, np.float32))
                scales.append(None)
            else:
                raw.append(rng.integers(0, 256, (*shape, dim // (2 if dt == 2 else 1))).astype(np.uint8))
                scales.append(np.full(shape, np.nan, np.float32))
            vals.append([(rng.standard_normal((n, HK, dim)) * mul).astype(np.float32)
                         for n in lens])
        at = 0
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
        self.K, self.V = [], []
        for side, (new, keep) in enumerate(((vals[0], self.K), (vals[1], self.V))):
            for s, n in enumerate(lens):
                x = new[s]
                pos = np.arange(n)
                pg, off = self.table[s, pos // page], pos % page
                if dt == 0:
                    raw[side][layer, pg, :, off] = x
                    keep.append(x.astype(np.float64))
                else:
                    c, sc = R.quantise(x, dt)
                    raw[side][layer, pg, :, off] = R.pack(c, dt)
                    scales[side][layer, pg, :, off] = sc
                    keep.append(c.astype(np.float64) * sc[..., None].astype(np.float64))
        self.raw, self.scales = raw, scales
        self.pool = paged.KvPool(dt, DA.from_numpy(raw[0]), DA.from_numpy(raw[1]), self.n_pages,
                                 page, HK, D, DV, n_layers,
                                 *(None if a is None else DA.from_numpy(a) for a in scales))
        self.HK, self.D, self.DV = HK, D, DV

    def attend(self, q, scale, window=0, sinks=0, table=None, lens=None, stream=None, bad=None):
        S, nq, H, _ = q.shape
        out = DA.from_numpy(np.full((S, nq, H, self.DV), 7.0, np.float32))
        ops.paged_attention(self.pool, self.layer, DA.from_numpy(q), out,
                            DA.from_numpy(self.table if table is None else table),
                            DA.from_numpy(self.lens if lens is None else lens), S, H, scale,
                            n_q=nq, window=window, sinks=sinks, bad=bad, stream=stream)
        if stream is not None:
            stream.synchronize()
        return out.numpy()

    def ref(self, q, scale, window=0, sinks=0, lens=None, hidden=lambda s, j: False):
        S, nq, H, _ = q.shape
        out = np.zeros((S, nq, H, self.DV))
        for s in range(S):
            n = int((self.lens if lens is None else lens)[s])
            pos = np.arange(n - nq, n)
            keep = R.seen(pos, np.arange(n), window, sinks) & (pos >= 0)[:, None]
            for j in range(n):
                if hidden(s, j):
                    keep[:, j] = False
            out[s] = R.attention(q[s], self.K[s][:n], self.V[s][:n], keep, scale)
        return out


def check(got, want, lens, nq):
    """Every row within RTOL of its own sequence's scale, rows of nothing zero."""
    for s in range(len(lens)):
        assert np.isfinite(got[s]).all(), s
        if not want[s].any():
            assert not got[s].any(), s
        else:
            assert rel_to_scale(got[s], want[s]) <= RTOL, (s, rel_to_scale(got[s], want[s]))


SHAPES = [
    # H, HK, D, DV, page, lens, n_q, window, sinks
    (32, 8, 128, 128, 16, [1, 0, 16, 17, 333, 4000], 1, 0, 0),
    (14, 2, 64, 64, 16, [333], 1, 0, 0),
    (8, 4, 256, 256, 32, [700, 33, 5, 32], 1, 0, 0),
    (64, 8, 128, 128, 64, [2049, 64, 65], 1, 0, 0),
    (32, 8, 64, 64, 128, [500, 128, 127], 1, 0, 0),
    (16, 2, 256, 256, 256, [1100], 1, 0, 0),
    (20, 1, 64, 64, 16, [300, 90], 1, 0, 0),               # 20 heads a kv head: two query tiles
    (8, 8, 128, 128, 16, [1000, 40], 1, 0, 0),             # a head of its own each
    (7, 1, 128, 128, 32, [200, 1, 2], 3, 0, 0),
    (32, 8, 128, 128, 16, [700, 2, 0, 31, 48], 5, 0, 0),   # fewer tokens than the step's
    (8, 4, 256, 256, 32, [6000, 1024, 1025, 1030, 3], 3, 1024, 4),
    (32, 8, 128, 128, 16, [3000, 100, 17, 16], 1, 64, 4),
    (32, 8, 128, 128, 16, [3000, 130], 1, 100, 0),
    (32, 8, 64, 64, 64, [3000, 500], 2, 33, 70),           # sinks over a page
    (32, 8, 128, 128, 256, [5000], 1, 1, 1),               # the newest token and the first
    (16, 2, 256, 256, 16, [900, 20], 1, 16, 17),
    (6, 6, 80, 48, 16, [130, 5, 64], 1, 0, 0),             # any width, value_dim < head_dim
    (4, 1, 32, 32, 16, [200, 33], 2, 20, 3),
    (4, 2, 20, 100, 32, [77], 1, 0, 0),
    (4, 2, 256, 8, 16, [50, 300], 1, 0, 0),
    (32, 8, 128, 128, 16, [300, 299], 40, 0, 0),           # a short prompt after cached tokens
]


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_paged_attention(hip, shape, dt):
    H, HK, D, DV, page, lens, nq, window, sinks = shape
    rng = np.random.default_rng([H, D, nq, len(lens), dt])
    c = Cache(rng, dt, page, HK, D, DV, lens)
    q = rng.standard_normal((len(lens), nq, H, D)).astype(np.float32)
    scale = D ** -0.5
    check(c.attend(q, scale, window, sinks), c.ref(q, scale, window, sinks), lens, nq)


@pytest.mark.parametrize("dt", [0, 1], ids=["fp32", "int8"])
def test_many_ragged_sequences(hip, dt):
    """More sequences than a wave has lanes, most of them short, empty rows
    between them; two runs give the same bits."""
    rng = np.random.default_rng(3 + dt)
    lens = (rng.integers(0, 90, 203) * (rng.random(203) < 0.8)).tolist()
    lens[100], lens[7] = 3777, 1200
    c = Cache(rng, dt, 16, 2, 64, 64, lens)
    q = rng.standard_normal((203, 1, 8, 64)).astype(np.float32)
    got = c.attend(q, 0.125)
    check(got, c.ref(q, 0.125), lens, 1)
    assert bits_equal(got, c.attend(q, 0.125))


def test_thousands_of_sequences(hip):
    """Most of them empty or of a few tokens, two long."""
    n_seq = 2060
    rng = np.random.default_rng(n_seq)
    lens = rng.integers(0, 5, n_seq).tolist()
    lens[3], lens[n_seq - 1] = 2500, 1700
    c = Cache(rng, 1, 16, 8, 64, 64, lens)
    q = rng.standard_normal((n_seq, 1, 8, 64)).astype(np.float32)
    got = c.attend(q, 0.125)
    check(got, c.ref(q, 0.125), lens, 1)
    assert bits_equal(got, c.attend(q, 0.125))


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
def test_pages_given_up_and_bad_pages(hip, dt):
    """Pages between the sinks and the window need no entry; ids outside the pool
    inside the visible part hide their keys and are reported."""
    rng = np.random.default_rng(11 + dt)
    lens = [2000, 700]
    c = Cache(rng, dt, 16, 8, 128, 128, lens)
    q = rng.standard_normal((2, 1, 32, 128)).astype(np.float32)
    table, bad = c.table.copy(), DA.from_numpy(np.zeros(1, np.int32))
    table[0, 1:(2000 - 300) // 16] = -1
    want = c.ref(q, 0.09, 300, 4)
    check(c.attend(q, 0.09, 300, 4, table=table, bad=bad), want, lens, 1)
    assert bad.numpy()[0] == 0
    for pg in (-1, c.n_pages, -2**31, 2**31 - 1):
        bad.copy_from(np.zeros(1, np.int32))
        t = table.copy()
        t[0, 120] = t[1, 0] = pg
        got = c.attend(q, 0.09, 300, 4, table=t, bad=bad)
        hidden = lambda s, j: j // 16 == (120 if s == 0 else 0)
        check(got, c.ref(q, 0.09, 300, 4, hidden=hidden), lens, 1)
        assert bad.numpy()[0] == 1
    # a length past the table is taken as the table's end
    got = c.attend(q, 0.09, lens=np.asarray([2**31 - 1, -5], np.int32))
    full = c.table.shape[1] * 16
    assert full == 2000
    check(got[:1], c.ref(q, 0.09)[:1], lens[:1], 1)
    assert not got[1].any()


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_ranges_of_scores_and_values(hip, D, dt):
    """Large scores that rise late (every sum is rescaled) and value scales from
    2^-60 to 2^60 along the sequence."""
    rng = np.random.default_rng(D + dt)
    n = 1500
    c = Cache(rng, dt, 16, 2, D, D, [n])
    pos = np.arange(n)
    mul = np.exp2(np.linspace(-60, 60, n)).astype(np.float32)
    k = (rng.standard_normal((n, 2, D)) * np.linspace(0.1, 6, n)[:, None, None]).astype(np.float32)
    v = rng.standard_normal((n, 2, D)).astype(np.float32) * mul[:, None, None]
    T, L = DA.from_numpy(c.table), DA.from_numpy(np.asarray([n], np.int32))
    ops.paged_kv_write(c.pool, 0, DA.from_numpy(k[None]), DA.from_numpy(v[None]), T, L, 1, n_q=n)
    if dt:
        (kc, ks), (vc, vs) = R.quantise(k, dt), R.quantise(v, dt)
        k, v = (a.astype(np.float64) * b[..., None].astype(np.float64) for a, b in ((kc, ks), (vc, vs)))
    c.K, c.V = [k.astype(np.float64)], [v.astype(np.float64)]
    q = rng.standard_normal((1, 1, 8, D)).astype(np.float32)
    for cut in (n, 900, 40):
        lens = np.asarray([cut], np.int32)
        got, want = c.attend(q, D ** -0.5, lens=lens), c.ref(q, D ** -0.5, lens=lens)
        # scores up to 6 * 5 sigma round by 2^-24 of themselves: 30 * 6e-8 * a few
        check(got, want, [cut], 1)


@pytest.mark.parametrize("dt", [0, 1], ids=["fp32", "int8"])
def test_plan_follows_growing_sequences(hip, dt):
    """A step recorded once: the lengths change between replays, with eager work
    in between; each replay equals the eager call bit for bit."""
    rng = np.random.default_rng(21)
    lens = [1500, 40, 700]
    c = Cache(rng, dt, 16, 8, 128, 128, lens)
    q = rng.standard_normal((3, 1, 32, 128)).astype(np.float32)
    out, dq, T = DA.empty(q.shape), DA.from_numpy(q), DA.from_numpy(c.table)
    L = DA.from_numpy(np.zeros(3, np.int32))
    plan = Plan()
    with plan:
        ops.paged_attention(c.pool, 0, dq, out, T, L, 3, 32, 0.09)
    stream = Stream()
    for now in ([1, 1, 0], [17, 40, 16], [1500, 33, 700], [2, 39, 699], [900, 0, 5]):
        ops.write_i32(L, list(enumerate(now)), stream)
        plan.launch(stream)
        stream.synchronize()
        got = out.numpy()
        lens = np.asarray(now, np.int32)
        check(got, c.ref(q, 0.09, lens=lens), now, 1)
        assert bits_equal(got, c.attend(q, 0.09, lens=lens))
    plan.destroy()
    stream.destroy()


def test_offsets_past_32_bits(hip):
    """Pages and a layer beyond 2^32 bytes of the pool."""
    rng = np.random.default_rng(5)
    page, HK, D, n_pages = 64, 8, 128, 10000           # 256 KB a page and side
    pool = paged.KvPool.empty(0, n_pages, page, HK, D, n_layers=2)
    assert pool.k.nbytes > 1 << 32
    n = 300
    table = np.asarray([[9999, 3, 9000, 9998, 0]], np.int32)
    T, L = DA.from_numpy(table), DA.from_numpy(np.asarray([n], np.int32))
    k, v = (rng.standard_normal((1, n, HK, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((1, 1, 32, D)).astype(np.float32)
    ko, vo, out = DA.empty(k.shape), DA.empty(v.shape), DA.empty(q.shape)
    for layer in (1, 0):
        ops.paged_kv_write(pool, layer, DA.from_numpy(k + layer), DA.from_numpy(v + layer), T, L,
                           1, n_q=n)
    ops.kv_pages_copy(pool, [9999, 9998], [4, 9997])
    T = DA.from_numpy(np.asarray([[4, 3, 9000, 9997, 0]], np.int32))
    for layer in (0, 1):
        ops.paged_kv_read(pool, layer, ko, vo, T, L, 1, n_q=n)
        assert bits_equal(ko.numpy(), k + layer) and bits_equal(vo.numpy(), v + layer)
        ops.paged_attention(pool, layer, DA.from_numpy(q), out, T, L, 1, 32, 0.09)
        want = R.attention(q[0], (k + layer)[0], (v + layer)[0], np.ones((1, n), bool), 0.09)
        assert rel_to_scale(out.numpy()[0], want) <= RTOL


# ----------------------------------------------------------------------- rows
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("HK,D,DV,page,lens,nq", [
    (8, 128, 128, 16, [40, 1, 0, 17], 1), (2, 64, 64, 32, [5, 300, 0], 7), (4, 256, 256, 64, [200], 190),
    (3, 80, 48, 16, [33, 2], 4), (1, 8, 4, 256, [1000], 999), (2, 20, 100, 128, [3], 1)])
def test_rows_written_and_read(hip, dt, HK, D, DV, page, lens, nq):
    """Codes, scales and values bit for bit, all else in the pool as it was."""
    rng = np.random.default_rng([dt, D, nq])
    c = Cache(rng, dt, page, HK, D, DV, lens, n_layers=2, layer=1)
    S = len(lens)
    k = rng.standard_normal((S, nq, HK, D)).astype(np.float32)
    v = (rng.standard_normal((S, nq, HK, DV)) * 1e-3).astype(np.float32)
    k[0, 0, 0] = 0                       # a zero vector: scale 1
    v[-1, -1, -1] *= np.float32(1e-36)   # subnormal values
    k[-1, -1, 0, :2] = (-3e38, 3e38)
    T, L = DA.from_numpy(c.table), DA.from_numpy(c.lens)
    ops.paged_kv_write(c.pool, 1, DA.from_numpy(k), DA.from_numpy(v), T, L, S, n_q=nq)
    want_raw, want_sc = [a.copy() for a in c.raw], [None if a is None else a.copy() for a in c.scales]
    back = [np.zeros_like(k), np.zeros_like(v)]
    for side, x in enumerate((k, v)):
        for s, n in enumerate(lens):
            for t in range(max(0, nq - n), nq):
                pos = n - nq + t
                pg, off = c.table[s, pos // page], pos % page
                if dt == 0:
                    want_raw[side][1, pg, :, off] = x[s, t]
                    back[side][s, t] = x[s, t]
                else:
                    code, sc = R.quantise(x[s, t], dt)
                    want_raw[side][1, pg, :, off] = R.pack(code, dt)
                    want_sc[side][1, pg, :, off] = sc
                    back[side][s, t] = code.astype(np.float32) * sc[:, None]
    for a, w in ((c.pool.k, want_raw[0]), (c.pool.v, want_raw[1]), (c.pool.k_scale, want_sc[0]),
                 (c.pool.v_scale, want_sc[1])):
        if w is not None:
            assert np.array_equal(a.numpy().view(np.uint8), w.view(np.uint8))
    ko, vo = DA.from_numpy(np.full_like(k, 9)), DA.from_numpy(np.full_like(v, 9))
    ops.paged_kv_read(c.pool, 1, ko, vo, T, L, S, n_q=nq)
    assert np.array_equal(ko.numpy(), back[0]) and np.array_equal(vo.numpy(), back[1])


def test_rows_match_the_contiguous_slot(hip):
    """The codes and scales are kv_write's, halves and clipping included."""
    rng = np.random.default_rng(8)
    n, HK, D = 64, 2, 128
    x = np.round(rng.standard_normal((1, n, HK, D)) * 200).astype(np.float32) / 2
    x[0, :, :, 0] = 127.0
    for dt in (ops.KV_INT8, ops.KV_INT4):
        pool = paged.KvPool.empty(dt, 1, 64, HK, D)
        T, L = DA.from_numpy(np.zeros((1, 1), np.int32)), DA.from_numpy(np.asarray([n], np.int32))
        dx = DA.from_numpy(x)
        ops.paged_kv_write(pool, 0, dx, dx, T, L, 1, n_q=n)
        slot = DA.empty(n * HK * ops.kv_vec_bytes(dt, D), np.uint8)
        sc = DA.empty(n * HK)
        ops.kv_write(dt, dx, n, HK, D, slot, sc, 0, n)
        assert np.array_equal(pool.k.numpy().reshape(HK, n, -1).transpose(1, 0, 2).reshape(-1),
                              slot.numpy())
        assert bits_equal(pool.v_scale.numpy().reshape(HK, n).T, sc.numpy().reshape(n, HK))


def test_rows_of_bad_pages(hip):
    rng = np.random.default_rng(9)
    c = Cache(rng, 1, 16, 2, 64, 64, [40, 40])
    k = rng.standard_normal((2, 40, 2, 64)).astype(np.float32)
    table = c.table.copy()
    table[0, 1], table[1, 2] = c.n_pages, -7
    bad = DA.from_numpy(np.zeros(1, np.int32))
    T, L, dk = DA.from_numpy(table), DA.from_numpy(c.lens), DA.from_numpy(k)
    ops.paged_kv_write(c.pool, 0, dk, dk, T, L, 2, n_q=40, bad=bad)
    assert bad.numpy()[0] == 1
    raw = c.pool.k.numpy()
    for s, col in ((0, 1), (1, 2)):      # what those rows' own pages hold is untouched
        assert np.array_equal(raw[0, c.table[s, col]], c.raw[0][0, c.table[s, col]])
    bad.copy_from(np.zeros(1, np.int32))
    out = DA.from_numpy(np.full_like(k, 9))
    ops.paged_kv_read(c.pool, 0, out, out, T, L, 2, n_q=40, bad=bad)
    got = out.numpy()
    assert bad.numpy()[0] == 1 and not got[0, 16:32].any() and not got[1, 32:].any()
    assert got[0, :16].any() and got[1, :32].any()


# ---------------------------------------------------------------------- pages
@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("page,HK,D,DV,layers,n", [(16, 8, 128, 128, 3, 300), (256, 1, 64, 64, 1, 1),
                                                   (32, 3, 80, 48, 2, 257), (16, 1, 4, 4, 5, 9)])
def test_pages_copied(hip, dt, page, HK, D, DV, layers, n):
    """Bit for bit, in every layer and plane; a source may be named often; more
    pairs than one launch takes."""
    rng = np.random.default_rng([dt, page, n])
    n_pages = 2 * n + 5
    perm = rng.permutation(n_pages).astype(np.int32)
    src, dst = perm[:n].copy(), perm[n:2 * n]
    src[: n // 3] = src[0]
    shape = (layers, n_pages, HK, page)
    kind = np.float32 if dt == 0 else np.uint8
    host = [rng.integers(0, 256, (*shape, ops.kv_vec_bytes(dt, d))).astype(np.uint8) for d in (D, DV)]
    host += [rng.integers(0, 256, (*shape, 4)).astype(np.uint8) for _ in range(2 if dt else 0)]
    dev = [DA.from_numpy(a.view(kind)) for a in host[:2]]
    dev += [DA.from_numpy(a.view(np.float32)) for a in host[2:]]
    pool = paged.KvPool(dt, dev[0], dev[1], n_pages, page, HK, D, DV, layers, *dev[2:])
    ops.kv_pages_copy(pool, src, dst)
    for a, d in zip(host, dev):
        a[:, dst] = a[:, src]
        assert np.array_equal(d.numpy().view(np.uint8).reshape(a.shape), a)


@pytest.mark.parametrize("dt,window,sinks", [(0, 0, 0), (1, 0, 0), (2, 0, 0), (1, 64, 4), (0, 50, 20)])
def test_serving_run(hip, dt, window, sinks):
    """The operators together, as a server uses them, two layers: prompts of
    different lengths, decode steps of some of the slots, a fork that diverges,
    pages given up behind the window, a rejected guess, a sequence that ends, a
    compaction, on one stream of its own; every step's rows against attention in
    64 bits over the tokens that each sequence was given."""
    rng = np.random.default_rng([dt, window])
    H, HK, D, layers = 8, 2, 64, 2
    pool = paged.KvPool.empty(dt, 60, 16, HK, D, n_layers=layers)
    kv = paged.PagedKV(pool, 5, 20)
    stream = Stream()
    K, V = {}, {}                        # slot -> per layer list of stored rows

    def stored(x):
        if dt == 0:
            return x.astype(np.float64)
        c, s = R.quantise(x, dt)
        return c.astype(np.float64) * s[..., None].astype(np.float64)

    def step(slots, n, table, lens, first, rows):
        """n new tokens of each slot; the call covers rows first .. first + rows - 1"""
        for l in range(layers):
            q, k, v = (rng.standard_normal((rows, n, h, D)).astype(np.float32) for h in (H, HK, HK))
            out = DA.empty(q.shape)
            ops.paged_kv_write(pool, l, DA.from_numpy(k), DA.from_numpy(v), table, lens, rows,
                               n_q=n, stream=stream)
            ops.paged_attention(pool, l, DA.from_numpy(q), out, table, lens, rows, H, 0.125, n_q=n,
                                window=window, sinks=sinks, stream=stream)
            stream.synchronize()
            got = out.numpy()
            for r in range(rows):
                s = first + r
                if s not in slots:
                    assert not got[r].any()
                    continue
                K[s][l].extend(stored(k[r]))
                V[s][l].extend(stored(v[r]))
                m = len(K[s][l])
                assert m == kv.length(s)
                keep = R.seen(np.arange(m - n, m), np.arange(m), window, sinks)
                want = R.attention(q[r], np.asarray(K[s][l]), np.asarray(V[s][l]), keep, 0.125)
                assert rel_to_scale(got[r], want) <= RTOL, (s, l, m)

    def prompt(n):
        s = kv.add()
        K[s], V[s] = [[] for _ in range(layers)], [[] for _ in range(layers)]
        kv.append([s], n, stream)
        step([s], n, *kv.rows(s), s, 1)
        return s

    def decode(slots, n=1):
        kv.append(slots, n, stream)
        step(slots, n, kv.table, kv.step, 0, 5)

    a, b = prompt(130), prompt(7)
    decode([a, b])
    c = kv.fork(a, stream)
    K[c], V[c] = [list(x) for x in K[a]], [list(x) for x in V[a]]
    for _ in range(3):
        decode([a, b, c])                # the fork's last page is copied once
    decode([c])
    if window:
        assert kv.trim(a, window, sinks, stream) > 0
    decode([a, b], 3)
    kv.truncate(a, kv.length(a) - 2, stream)      # two of three guesses rejected
    for x in (K, V):
        for l in range(layers):
            del x[a][l][-2:]
    decode([a, c])
    kv.free(b, stream)
    del K[b], V[b]
    d = prompt(33)
    moved = kv.compact(stream)
    decode([a, c, d])
    kv.free(a, stream)
    assert kv.compact(stream) + moved > 0
    for _ in range(2):
        decode([c, d])
    kv.free(c, stream)
    kv.free(d, stream)
    assert kv.free_pages == 60
    stream.synchronize()
    assert not kv.lens.numpy().any() and (kv.table.numpy() == -1).all()
    stream.destroy()


@pytest.mark.parametrize("dt", [0, 1], ids=["fp32", "int8"])
def test_lengths_past_the_table(hip, dt):
    """A length that the table has no room for is cut to the room, and said so."""
    rng = np.random.default_rng([70, dt])
    c = Cache(rng, dt, 16, 2, 64, 64, [64, 30])
    q = rng.standard_normal((2, 1, 4, 64)).astype(np.float32)
    bad = DA.from_numpy(np.zeros(1, np.int32))
    table = c.table[:, :4].copy()
    want = c.attend(q, 0.1, table=table, bad=bad)
    assert bad.numpy()[0] == 0
    got = c.attend(q, 0.1, table=table, lens=np.asarray([100, 30], np.int32), bad=bad)
    assert bad.numpy()[0] == 1 and bits_equal(got, want)


# widths between those of the matrix operands, K and V of two, whole pieces and not
WIDTHS = [(80, 80), (96, 96), (112, 112), (160, 160), (192, 192), (192, 128), (64, 128), (128, 64),
          (8, 8), (16, 240), (240, 16), (40, 104), (48, 48), (72, 100), (252, 4), (56, 256),
          (12, 20), (250, 250), (2, 6)]


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("D,DV", WIDTHS, ids=[f"{a}-{b}" for a, b in WIDTHS])
def test_widths(hip, D, DV, dt):
    """Other widths: what lies behind a vector (unused rows are NaN, or NaN scales)
    and behind a query's does not count."""
    if dt == 0 and (D % 4 or DV % 4):
        pytest.skip("fp32 rows are whole 16-byte pieces")
    rng = np.random.default_rng([D, DV, dt])
    lens = [700, 0, 1, 33, 5]
    c = Cache(rng, dt, 16, 3, D, DV, lens)
    for nq, window, sinks in ((1, 0, 0), (3, 40, 4)):
        q = rng.standard_normal((len(lens), nq, 15, D)).astype(np.float32)
        check(c.attend(q, 0.1, window, sinks), c.ref(q, 0.1, window, sinks), lens, nq)


def shifted(a, by=1):
    """a on the device, `by` elements behind a 16-byte boundary"""
    a = np.ascontiguousarray(a)
    buf = DA.empty(a.size + by, a.dtype)
    buf.copy_from(np.concatenate([np.zeros(by, a.dtype), a.reshape(-1)]))
    return buf.view(a.shape, offset_bytes=by * a.itemsize)


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("D,DV", [(128, 128), (64, 32), (256, 256)])
def test_rows_that_are_not_aligned(hip, D, DV, dt):
    """Queries, outputs and new rows at any 4-byte address."""
    rng = np.random.default_rng([D, dt, 71])
    H, HK, lens, nq = 8, 2, [300, 2, 17], 2
    c = Cache(rng, dt, 16, HK, D, DV, lens)
    q = rng.standard_normal((3, nq, H, D)).astype(np.float32)
    T, L = DA.from_numpy(c.table), DA.from_numpy(c.lens)
    want = c.ref(q, 0.1, 100, 4)
    for dq, out in ((shifted(q), DA.empty((3, nq, H, DV))),
                    (DA.from_numpy(q), shifted(np.ones((3, nq, H, DV), np.float32), 3)),
                    (shifted(q, 2), shifted(np.ones((3, nq, H, DV), np.float32)))):
        ops.paged_attention(c.pool, 0, dq, out, T, L, 3, H, 0.1, n_q=nq, window=100, sinks=4)
        check(out.numpy(), want, lens, nq)
    k = rng.standard_normal((3, nq, HK, D)).astype(np.float32)
    v = rng.standard_normal((3, nq, HK, DV)).astype(np.float32)
    rows = []
    for move in (DA.from_numpy, shifted):
        ops.paged_kv_write(c.pool, 0, move(k), move(v), T, L, 3, n_q=nq)
        ko, vo = move(np.full_like(k, 9)), move(np.full_like(v, 9))
        ops.paged_kv_read(c.pool, 0, ko, vo, T, L, 3, n_q=nq)
        rows.append((ko.numpy(), vo.numpy()))
        ops.paged_kv_write(c.pool, 0, DA.from_numpy(0 * k), DA.from_numpy(0 * v), T, L, 3, n_q=nq)
    assert bits_equal(rows[0][0], rows[1][0]) and bits_equal(rows[0][1], rows[1][1])
    assert rows[0][0].any()


@pytest.mark.parametrize("dt", [0, 1, 2], ids=["fp32", "int8", "int4"])
@pytest.mark.parametrize("H,HK,D,page,lens,nq,window,sinks", [
    (32, 8, 128, 16, [300, 900, 100, 0], 300, 64, 4), (8, 2, 64, 64, [3000, 700], 130, 33, 70),
    (2, 1, 64, 16, [3000], 20, 1000, 4), (16, 2, 256, 32, [2600, 40], 37, 1500, 0),
    (24, 1, 128, 16, [1200], 9, 500, 16), (6, 2, 48, 16, [800, 90], 50, 100, 3),
    (32, 8, 64, 16, [1500, 200], 200, 0, 0)])
def test_prompts(hip, H, HK, D, page, lens, nq, window, sinks, dt):
    """Many new tokens at once, windows that most of them do not share."""
    rng = np.random.default_rng([H, D, nq, dt])
    c = Cache(rng, dt, page, HK, D, D, lens)
    q = rng.standard_normal((len(lens), nq, H, D)).astype(np.float32)
    check(c.attend(q, 0.1, window, sinks), c.ref(q, 0.1, window, sinks), lens, nq)
