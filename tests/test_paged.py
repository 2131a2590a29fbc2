"""CPU: the arithmetic of the paged kernels' work (paged_sched.hpp, compiled as
plain C++), the bookkeeping of PagedKV against a plain model of pages, and the
refusals of the paged operators. Nothing here touches a GPU."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from aero_amd import _lib, ops, paged
from aero_amd.device import DeviceArray

SCHED = r"""
#include "paged_sched.hpp"
using namespace aero;
extern "C" {
int tiles(long long lo, long long hi, long long n_kv, int window, int sinks, int shift, int* out,
          int* place, int* column) {
    const KeyTiles t = key_tiles(lo, hi, n_kv, window, sinks);
    for (int x = 0; x < t.n; ++x) {
        out[x] = t.at(x);
        place[x] = t.page_place(x, shift);
        column[x] = t.column(place[x], shift);
    }
    return t.n;
}
int units(int n, int u) { return item_units(n, u); }
int chunks(int u, int total, int target) { return item_chunks(u, total, target); }
int begin(int c, int n, int u) { return chunk_begin(c, n, u); }
}
"""


@pytest.fixture(scope="module")
def sched(tmp_path_factory):
    d = tmp_path_factory.mktemp("sched")
    (d / "s.cpp").write_text(SCHED)
    so = d / "s.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "aero_amd", "csrc"), str(d / "s.cpp"), "-o", str(so)],
                   check=True)
    L = ctypes.CDLL(str(so))
    i64, i32p = ctypes.c_int64, ctypes.POINTER(ctypes.c_int32)
    L.tiles.argtypes = [i64, i64, i64, ctypes.c_int, ctypes.c_int, ctypes.c_int] + [i32p] * 3
    return L


def test_key_tiles_are_those_of_the_seen_keys(sched):
    """Every tile with a key that some position sees is in the list, once and in
    order; tiles between the sinks and the window are not; page places have no
    gaps and name the tile's own column."""
    rng = random.Random(1)
    out, place, col = ((ctypes.c_int32 * 400)() for _ in range(3))
    for _ in range(4000):
        n_kv = rng.choice((1, 15, 16, 17, 33, 100, 640, rng.randint(1, 2000)))
        window = rng.choice((0, 0, 1, 7, 16, 64, rng.randint(1, 1500)))
        sinks = rng.choice((0, 1, 4, 16, 17, 40, 3000)) if window else 0
        lo = rng.randint(-3, n_kv + 5)
        hi = lo + rng.choice((0, 0, 1, 5, 40))
        shift = rng.choice((0, 1, 2, 4))
        n = sched.tiles(lo, hi, n_kv, window, sinks, shift, out, place, col)
        got = list(out[:n])
        need = {j // 16 for p in range(lo, hi + 1) for j in range(min(p + 1, n_kv))
                if not window or p - j < window or j < sinks}
        assert need <= set(got) and got == sorted(set(got))
        assert all(16 * t < n_kv for t in got)
        # no tile without a key that the list's rule covers
        first = max(0, lo - window + 1) if window else 0
        assert all(16 * t + 15 >= min(first, hi + 1, n_kv) or 16 * t < sinks for t in got)
        assert list(col[:n]) == [t >> shift for t in got]
        if n:
            assert place[0] == 0 and all(b - a in (0, 1) for a, b in zip(place[:n], place[1:n]))


def test_chunks_cover_every_unit_once(sched):
    """An item's chunks are its units, none empty, none longer than the share of a
    chunk; all items' chunks fit the grid and the room for parts."""
    rng = random.Random(2)
    assert [sched.units(n, 8) for n in (0, 1, 8, 9)] == [1, 1, 1, 2]
    for _ in range(400):
        items = [rng.choice((1, 2, rng.randint(1, 40), rng.randint(1, 3000)))
                 for _ in range(rng.randint(1, 60))]
        total, target = sum(items), rng.choice((1, 5, 256, 768))
        n = [sched.chunks(u, total, target) for u in items]
        assert sum(n) <= target + len(items) and sum(x for x in n if x > 1) <= 2 * target
        for u, c in zip(items, n):
            cuts = [sched.begin(i, c, u) for i in range(c + 1)]
            assert cuts[0] == 0 and cuts[-1] == u
            assert all(0 < b - a <= -(-total // target) for a, b in zip(cuts, cuts[1:]))
    big = 2**31 - 1
    n = sched.chunks(big, big, 768)
    assert n <= 769 and sched.begin(n, n, big) == big and sched.begin(1, n, big) > 0


def test_kv_pool_struct_layout(tmp_path):
    """aero_kv_pool_t as the C compiler lays it out equals its ctypes mirror."""
    fields = [f for f, _ in _lib.KvPool._fields_]
    (tmp_path / "l.c").write_text(
        '#include <stddef.h>\n#include <stdio.h>\n#include "aero_hip.h"\nint main(void) {\n'
        + "".join(f'  printf("%zu\\n", offsetof(aero_kv_pool_t, {f}));\n' for f in fields)
        + '  printf("%zu\\n", sizeof(aero_kv_pool_t));\n  return 0;\n}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o",
                    str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [getattr(_lib.KvPool, f).offset for f in fields] + [ctypes.sizeof(_lib.KvPool)]


# -------------------------------------------------------------------- PagedKV
def fake(shape, dtype=np.float32):
    return DeviceArray(shape, dtype, _ptr=0x10000, _owner=False)


def fake_pool(n_pages=40, page=16, layers=2, dt=ops.KV_F32):
    vecs = layers * n_pages * 2 * page
    scales = {} if dt == 0 else {"k_scale": fake(vecs), "v_scale": fake(vecs)}
    kind = np.float32 if dt == 0 else np.uint8
    n = vecs * 64 // (2 if dt == 2 else 1)
    return paged.KvPool(dt, fake(n, kind), fake(n, kind), n_pages, page, 2, 64, n_layers=layers,
                        **scales)


class Model:
    """The device side as plain arrays: pages hold (sequence name, position)."""

    def __init__(self, monkeypatch, pool, max_seqs, max_pages):
        self.pages = {}                      # (page, offset) -> token
        monkeypatch.setattr(paged.DeviceArray, "empty",
                            classmethod(lambda cls, s, dt=np.float32: fake(s, dt)))
        monkeypatch.setattr(paged.DeviceArray, "copy_from", lambda a, x: None)
        monkeypatch.setattr(ops, "kv_pages_copy", self.copy)
        monkeypatch.setattr(ops, "write_i32", self.edit)
        n = max_seqs * max_pages
        self.dev = np.zeros(n + 2 * max_seqs, np.int64)
        self.dev[:n] = -1
        self.pool, self.n, self.mp, self.ms = pool, n, max_pages, max_seqs

    def copy(self, pool, src, dst, stream=None):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        for a, b in zip(src, dst):
            for o in range(pool.page):
                if (a, o) in self.pages:
                    self.pages[b, o] = self.pages[a, o]

    def edit(self, a, items, stream=None):
        at = [i for i, _ in items]
        assert at == sorted(set(at))
        for i, x in items:
            self.dev[i] = x

    def token(self, s, pos):
        page = self.dev[s * self.mp + pos // self.pool.page]
        return None if page < 0 else self.pages.get((int(page), pos % self.pool.page))

    def write(self, s, pos, value):
        page = int(self.dev[s * self.mp + pos // self.pool.page])
        assert page >= 0
        self.pages[page, pos % self.pool.page] = value


@pytest.mark.parametrize("seed", range(6))
def test_paged_kv_against_a_plain_model(monkeypatch, seed):
    """Random appends, forks, trims, truncations, frees and compactions: every
    sequence keeps its own tokens, pages are never shared by writers, none leaks."""
    rng = random.Random(seed)
    pool = fake_pool()
    m = Model(monkeypatch, pool, 6, 12)
    kv = paged.PagedKV(pool, 6, 12)
    truth, lost, wins, name = {}, {}, {}, 0
    for step in range(400):
        what = rng.choice(("add", "append", "append", "append", "fork", "trim", "cut", "free",
                           "compact"))
        if what == "add" and len(truth) < 6:
            s = kv.add()
            truth[s], lost[s], wins[s] = [], 0, 1 << 30
        elif what == "append" and truth:
            slots = rng.sample(sorted(truth), rng.randint(1, len(truth)))
            n = rng.choice((1, 1, 2, 16, 30))
            before = (m.dev.copy(), kv.free_pages)
            try:
                kv.append(slots, n)
            except (paged.OutOfPages, ValueError):
                assert np.array_equal(before[0], m.dev) and before[1] == kv.free_pages
                continue
            for s in slots:
                for _ in range(n):
                    m.write(s, len(truth[s]), name)
                    truth[s].append(name)
                    name += 1
            for s in range(6):
                assert m.dev[m.n + 6 + s] == (len(truth[s]) if s in slots else 0)
        elif what == "fork" and truth and len(truth) < 6:
            s = rng.choice(sorted(truth))
            d = kv.fork(s)
            truth[d], lost[d], wins[d] = list(truth[s]), lost[s], wins[s]
        elif what == "trim" and truth:
            s, w, k = rng.choice(sorted(truth)), rng.choice((5, 20, 40)), rng.choice((0, 4, 16, 20))
            first = truth[s][:k]
            kv.trim(s, w, k)
            wins[s] = w
            lost[s] = max(lost[s], len(truth[s]) - w)
            if lost[s] > 0:     # what neither this nor a later token sees may be gone
                truth[s] = [t if i < 0 or i >= lost[s] or m.token(s, i) == t else None
                            for i, t in enumerate(truth[s])]
                assert truth[s][:k] == first
        elif what == "cut" and truth:
            s = rng.choice(sorted(truth))
            n = rng.randint(lost[s] if lost[s] > 0 else 0, len(truth[s]))
            # (what the newest token left would see has to be there)
            if all(m.token(s, i) is not None for i in range(max(0, n - wins[s]), n)):
                kv.truncate(s, n)
                del truth[s][n:]
                lost[s] = min(lost[s], n)
            else:
                with pytest.raises(ValueError):
                    kv.truncate(s, n)
        elif what == "free" and truth:
            s = rng.choice(sorted(truth))
            kv.free(s)
            del truth[s], lost[s], wins[s]
        elif what == "compact":
            kv.compact()
            used = {p for s in truth for p in kv.pages(s) if p >= 0}
            assert used == set(range(kv.used_pages))
        for s, want in truth.items():
            assert kv.length(s) == len(want) == m.dev[m.n + s]
            for i, t in enumerate(want):
                assert t is None or m.token(s, i) == t, (step, what, s, i)
        used = {p for s in truth for p in kv.pages(s) if p >= 0}
        assert kv.used_pages == len(used) and kv.free_pages == pool.n_pages - len(used)
        for s in range(6):
            if s not in truth:
                assert m.dev[m.n + s] == 0 and (m.dev[s * 12:(s + 1) * 12] == -1).all()


def test_truncate_after_trim(monkeypatch):
    """Cut back to where the window is still whole, and to the sinks alone; not
    into pages given up."""
    pool = fake_pool()
    Model(monkeypatch, pool, 2, 12)
    kv = paged.PagedKV(pool, 2, 12)
    a = kv.add()
    kv.append([a], 160)
    kv.trim(a, 40, 4)                    # tokens 16 .. 111 gone
    assert kv.pages(a)[1:7] == [-1] * 6 and min(kv.pages(a)[7:]) >= 0
    b = kv.fork(a)
    for s in (a, b):
        with pytest.raises(ValueError):
            kv.truncate(s, 151)
        kv.truncate(s, 152)
    kv.truncate(b, 16)
    kv.append([b], 1)
    kv.free(a)
    a = kv.add()                         # a new sequence in the slot
    kv.append([a], 60)
    kv.truncate(a, 1)


def test_trim_with_more_sinks_later(monkeypatch):
    """First tokens that a trim without sinks gave up stay given up, and show as such;
    the window decides what may be cut back."""
    pool = fake_pool()
    Model(monkeypatch, pool, 2, 12)
    kv = paged.PagedKV(pool, 2, 12)
    a = kv.add()
    kv.append([a], 100)
    assert kv.trim(a, 40) == 3 and kv.pages(a)[:3] == [-1] * 3
    assert kv.trim(a, 40, 16) == 0 and kv.pages(a)[:3] == [-1] * 3
    kv.append([a], 30)
    assert kv.trim(a, 40, 16) == 2 and kv.pages(a)[:5] == [-1] * 5
    kv.truncate(a, 120)
    with pytest.raises(ValueError):
        kv.truncate(a, 119)
    assert kv.pages(a)[0] == -1


def test_paged_kv_refusals(monkeypatch):
    pool = fake_pool(n_pages=4)
    m = Model(monkeypatch, pool, 2, 3)
    kv = paged.PagedKV(pool, 2, 3)
    a = kv.add()
    for bad in (lambda: kv.append([a, a]), lambda: kv.append([1]), lambda: kv.append([a], 0),
                lambda: kv.append([a], 49), lambda: kv.truncate(a, 1), lambda: kv.trim(a, 0),
                lambda: kv.length(7), lambda: kv.rows(1, 2), lambda: kv.free(1)):
        with pytest.raises(ValueError):
            bad()
    b = kv.add()
    with pytest.raises(ValueError):
        kv.add()
    kv.append([a, b], 20)
    with pytest.raises(paged.OutOfPages):
        kv.append([a], 20)
    assert kv.length(a) == 20
    monkeypatch.setattr(paged, "recording_plan", lambda: object())
    with pytest.raises(RuntimeError):
        kv.append([a])
    with pytest.raises(RuntimeError):
        kv.compact()


def held(kv):
    """What a PagedKV says it holds."""
    return (kv.free_pages, {s: (kv.length(s), kv.pages(s)) for s in range(kv.max_seqs)
                            if s in kv._live})


@pytest.mark.parametrize("seed", range(4))
def test_a_launch_that_fails_changes_nothing(monkeypatch, seed):
    """Page copies and table writes that fail, the latter after part of their
    entries: the call raises, all is as before it, and the next call that succeeds
    leaves on the device what it should hold, no sequence's tokens lost."""
    rng = random.Random(seed)
    pool = fake_pool()
    m = Model(monkeypatch, pool, 5, 12)
    kv = paged.PagedKV(pool, 5, 12)
    truth, name, failed = {}, 0, 0
    fail = {"copy": False, "edit": False}

    def copy(pool, src, dst, stream=None):
        if fail["copy"]:
            raise _lib.AeroHipError("kv_pages_copy")
        m.copy(pool, src, dst)

    def edit(a, items, stream=None):
        if fail["edit"]:
            m.edit(a, items[:rng.randint(0, len(items))])
            raise _lib.AeroHipError("write_i32")
        m.edit(a, items)

    monkeypatch.setattr(ops, "kv_pages_copy", copy)
    monkeypatch.setattr(ops, "write_i32", edit)
    for step in range(500):
        fail["copy"], fail["edit"] = rng.random() < 0.3, rng.random() < 0.2
        what = rng.choice(("add", "append", "append", "append", "fork", "trim", "cut", "free",
                           "compact"))
        if what == "add":
            if len(truth) < 5:
                truth[kv.add()] = []
            continue
        if what != "compact" and not truth:
            continue
        s = rng.choice(sorted(truth)) if truth else None
        before = held(kv)
        try:
            if what == "append":
                slots = rng.sample(sorted(truth), rng.randint(1, len(truth)))
                n = rng.choice((1, 9, 20))
                kv.append(slots, n)
                for t in slots:
                    for _ in range(n):
                        m.write(t, len(truth[t]), name)
                        truth[t].append(name)
                        name += 1
            elif what == "fork":
                d = kv.fork(s)
                truth[d] = list(truth[s])
            elif what == "trim":        # (no window is longer than this one)
                kv.trim(s, 150, 16)
                gone = max(0, len(truth[s]) - 150) // 16 * 16
                truth[s][16:gone] = [None] * max(0, gone - 16)
            elif what == "cut":
                n = rng.randint(max(0, len(truth[s]) - 5), len(truth[s]))
                kv.truncate(s, n)
                del truth[s][n:]
            elif what == "free":
                kv.free(s)
                del truth[s]
            else:
                kv.compact()
        except _lib.AeroHipError:
            failed += 1
            assert held(kv) == before, (step, what)
            continue
        except (paged.OutOfPages, ValueError):
            assert held(kv) == before
            continue
        assert np.array_equal(m.dev, kv._host), (step, what)
        for t in range(5):
            row = kv.pages(t) if t in truth else []
            assert m.dev[t * 12:(t + 1) * 12].tolist() == row + [-1] * (12 - len(row)), (step, what)
            assert m.dev[m.n + t] == len(truth.get(t, []))
        for t, want in truth.items():
            for i, x in enumerate(want):
                assert x is None or m.token(t, i) == x, (step, what, t, i)
        used = {p for t in truth for p in kv.pages(t) if p >= 0}
        assert kv.used_pages == len(used)
    assert failed > 20          # (the run did meet failures)


# ------------------------------------------------------------------- refusals
def c_pool(**k):
    d = dict(kv_dt=1, page=16, n_layers=2, n_pages=8, n_head_kv=2, head_dim=64, value_dim=64,
             k=0x1000, v=0x2000, k_scale=0x3000, v_scale=0x4000)
    d.update(k)
    return _lib.KvPool(**d)


@pytest.mark.parametrize("bad", [
    dict(kv_dt=3), dict(kv_dt=-1), dict(page=8), dict(page=24), dict(page=512), dict(n_layers=0),
    dict(n_pages=0), dict(n_head_kv=0), dict(head_dim=0), dict(head_dim=260), dict(value_dim=257),
    dict(kv_dt=0, head_dim=66), dict(kv_dt=2, value_dim=63), dict(k=None), dict(v=0x2004),
    dict(k_scale=None), dict(v_scale=0x4008)])
def test_bad_pools_are_refused(bad):
    L, p = _lib.load(), c_pool(**bad)
    r = ctypes.byref(p)
    idx = np.zeros(1, np.int32)
    ip = idx.ctypes.data
    assert L.aero_hip_paged_attention_workspace(r, 1, 1, 4, 4) == (
        -1)
    assert L.aero_hip_paged_attention(r, 0, 16, 16, 16, 4, 16, 1, 1, 4, 1.0, 0, 0, None, 16,
                                      1 << 30, None) == 0
    assert "paged_attention" in _lib.last_error()
    assert L.aero_hip_paged_kv_write(r, 0, 16, 16, 16, 4, 16, 1, 1, None, None) == 0
    assert L.aero_hip_paged_kv_read(r, 0, 16, 16, 16, 4, 16, 1, 1, None, None) == 0
    assert L.aero_hip_kv_pages_copy(r, ip, ip, 1, None) == 0
    assert "kv_pages_copy" in _lib.last_error()


def test_bad_calls_are_refused():
    L, p = _lib.load(), c_pool()
    r = ctypes.byref(p)
    need = L.aero_hip_paged_attention_workspace(r, 3, 1, 4, 400)
    assert need > 0
    ok = dict(layer=0, q=16, out=16, table=16, max_pages=400, lens=16, n_seq=3, n_q=1, n_head=4,
              scale=1.0, window=0, sinks=0, bad=None, ws=16, ws_bytes=need)
    for k in (dict(layer=2), dict(layer=-1), dict(q=None), dict(out=None), dict(table=None),
              dict(lens=None), dict(ws=None), dict(ws=24), dict(ws_bytes=need - 1),
              dict(n_head=3), dict(n_head=0), dict(n_q=0), dict(n_seq=-1), dict(max_pages=0),
              dict(max_pages=1 << 28), dict(window=-1), dict(sinks=-1), dict(n_seq=1 << 31)):
        a = {**ok, **k}
        assert L.aero_hip_paged_attention(r, *a.values(), None) == 0, k
        assert "paged_attention" in _lib.last_error()
    assert L.aero_hip_paged_attention(None, *ok.values(), None) == 0
    rows = dict(layer=0, k=16, v=16, table=16, max_pages=4, lens=16, n_seq=1, n_q=1, bad=None)
    for f, name in ((L.aero_hip_paged_kv_write, "paged_kv_write"),
                    (L.aero_hip_paged_kv_read, "paged_kv_read")):
        for k in (dict(layer=2), dict(k=None), dict(v=None), dict(table=None), dict(lens=None),
                  dict(n_q=0), dict(n_seq=-1), dict(max_pages=0), dict(n_seq=1 << 31)):
            assert f(r, *{**rows, **k}.values(), None) == 0, k
            assert name in _lib.last_error()
        assert f(r, *{**rows, "n_seq": 0}.values(), None) == 1      # nothing to do

    def copy(src, dst):
        a, b = np.asarray(src, np.int32), np.asarray(dst, np.int32)
        return L.aero_hip_kv_pages_copy(r, a.ctypes.data, b.ctypes.data, a.size, None)

    for src, dst, word in (([0], [8], "outside"), ([-1], [1], "outside"), ([8], [1], "outside"),
                           ([0, 1], [5, 5], "twice"), ([0, 1], [1, 2], "a source and"),
                           ([3], [3], "a source and"), ([0] * 9, list(range(9)), "bad list")):
        assert copy(src, dst) == 0 and word in _lib.last_error(), (src, dst)
    assert copy([], []) == 1

    def write(at, n_base=10):
        a, b = np.asarray(at, np.int64), np.zeros(len(at), np.int32)
        return L.aero_hip_write_i32(16, n_base, a.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)),
                                    b.ctypes.data_as(_lib.ip), a.size, None)

    for at in ([10], [-1], [3, 3], [4, 2], [0, 1 << 40]):
        assert write(at) == 0 and "write_i32" in _lib.last_error()
    assert write([]) == 1

    s = dict(q=16, kv_dt=1, k=16, ks=16, v=16, vs=16, out=16, n_q=1, n_head=4, n_head_kv=2,
             head_dim=64, value_dim=64, scale=1.0, qpos=None, kpos=None, n_kv=4000, window=1000,
             sinks=4, ws=16, wsb=1 << 30)
    for k in (dict(q=None), dict(k=None), dict(vs=None), dict(out=None), dict(n_q=0),
              dict(n_head=3), dict(head_dim=257), dict(value_dim=0), dict(n_kv=0),
              dict(n_kv=1 << 30), dict(kv_dt=3), dict(kv_dt=0, head_dim=66),
              dict(kv_dt=2, value_dim=63), dict(sinks=-1), dict(kv_dt=0, k=20), dict(ws=None),
              dict(ws=24), dict(wsb=16)):
        assert L.aero_hip_attention_sinks(*{**s, **k}.values(), None) == 0, k
        assert "attention" in _lib.last_error()
    assert L.aero_hip_attention_sinks_workspace(1, 1, 4, 3, 64, 64, 100, 10, 4) == -1


def test_op_wrappers_check_on_the_host():
    pool = fake_pool(dt=ops.KV_INT8)
    t, n = fake((4, 5), np.int32), fake(4, np.int32)
    q = fake((4, 1, 4, 64))
    with pytest.raises(ValueError):
        ops.paged_attention(pool, 0, fake(100), q, t, n, 4, 4, 1.0)
    with pytest.raises(ValueError):
        ops.paged_attention(pool, 0, q, q, fake((3, 5), np.int32), n, 4, 4, 1.0)
    with pytest.raises(TypeError):
        ops.paged_attention(pool, 0, q, q, fake((4, 5)), n, 4, 4, 1.0)
    with pytest.raises(ValueError):
        ops.paged_attention(pool, 0, q, q, fake(20, np.int32), n, 4, 4, 1.0)
    with pytest.raises(ValueError):
        ops.paged_kv_write(pool, 0, fake(4 * 2 * 64 - 1), fake(4 * 2 * 64), t, n, 4)
    with pytest.raises(ValueError):
        ops.paged_kv_read(pool, 0, fake(4 * 2 * 64), fake(4 * 2 * 64), t, fake(3, np.int32), 4)
    for src, dst in (([0], [1, 2]), ([1 << 40], [1])):
        with pytest.raises(ValueError):
            ops.kv_pages_copy(pool, src, dst)
    with pytest.raises(TypeError):
        ops.kv_pages_copy(pool, [0.5], [1])
    for k in (dict(kv_dt=5), dict(page=20), dict(n_pages=0), dict(n_pages=1000)):
        with pytest.raises(ValueError):
            paged.KvPool(**{**dict(kv_dt=0, k=fake(40 * 2 * 16 * 64), v=fake(40 * 2 * 16 * 64),
                                   n_pages=40, page=16, n_head_kv=2, head_dim=64), **k})
    with pytest.raises(ValueError):
        paged.KvPool(1, fake(40960, np.uint8), fake(40960, np.uint8), 20, 16, 2, 64)


@pytest.mark.parametrize("k", [dict(window=1 << 32), dict(window=(1 << 32) + 5),
                               dict(window=1 << 31), dict(window=64, sinks=1 << 32),
                               dict(window=64, sinks=(1 << 32) + 4)], ids=str)
def test_windows_past_32_bits_are_refused(k):
    """A C int would take their low 32 bits: another window, or none."""
    pool = fake_pool(dt=ops.KV_INT8)
    t, n, q = fake((4, 5), np.int32), fake(4, np.int32), fake((4, 1, 4, 64))
    with pytest.raises(ValueError):
        ops.paged_attention(pool, 0, q, q, t, n, 4, 4, 1.0, **k)
    with pytest.raises(ValueError):
        ops.attention(q, q, q, q, 1, 4, 2, 64, 64, 4, 1.0, **{"sinks": 4, **k})
