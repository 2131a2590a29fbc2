"""A paged KV cache for several sequences: the pool in HBM (KvPool) and its
bookkeeping (PagedKV) for ops.paged_kv_write / paged_attention / paged_kv_read.

The reference keeps one contiguous slot a sequence (src/kv.cpp:30-133); here
sequences share a pool of fixed pages, so they grow, fork (sharing pages until
one of them writes), drop what their window has left behind and end without
moving each other.

    pool = KvPool.empty(ops.KV_INT8, n_pages=4096, page=16, n_head_kv=8,
                        head_dim=128, n_layers=32)
    kv = PagedKV(pool, max_seqs=64, max_pages=512)
    a = kv.add()
    kv.append([a], T)                      # room for a prompt of T tokens
    table, lens = kv.rows(a)               # one sequence's rows
    for l in range(32):
        ops.paged_kv_write(pool, l, k, v, table, lens, 1, n_q=T)
    b = kv.fork(a)                         # shares a's pages
    kv.append([a, b])                      # one token each: the shared last page is copied
    for l in range(32):
        ops.paged_kv_write(pool, l, k, v, kv.table, kv.step, kv.max_seqs)
        ops.paged_attention(pool, l, q, out, kv.table, kv.step, kv.max_seqs, 32, scale)
"""
from __future__ import annotations

import contextlib
import ctypes
import heapq

import numpy as np

from . import _lib, ops
from .device import DeviceArray, Stream, recording_plan


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than the call needs. Nothing was changed."""


class KvPool:
    """The pages of a cache: k [n_layers, n_pages, n_head_kv, page, head_dim] in
    kv_dt (ops.KV_*), v the same of value_dim, k_scale / v_scale [n_layers,
    n_pages, n_head_kv, page] fp32 for the integer types, DeviceArrays that the
    pool keeps alive. page: tokens a page, a power of two from 16 to 256."""

    def __init__(self, kv_dt: int, k: DeviceArray, v: DeviceArray, n_pages: int, page: int,
                 n_head_kv: int, head_dim: int, value_dim: int | None = None, n_layers: int = 1,
                 k_scale: DeviceArray | None = None, v_scale: DeviceArray | None = None):
        value_dim = head_dim if value_dim is None else value_dim
        if kv_dt not in (ops.KV_F32, ops.KV_INT8, ops.KV_INT4):
            raise ValueError(f"kv dtype {kv_dt}")
        if page < 16 or page > 256 or page & (page - 1):
            raise ValueError(f"page of {page} tokens: a power of two from 16 to 256")
        if min(n_pages, n_head_kv, head_dim, value_dim, n_layers) <= 0:
            raise ValueError("KvPool: sizes must be positive")
        vecs = n_layers * n_pages * n_head_kv * page
        for a, dim, name in ((k, head_dim, "k"), (v, value_dim, "v")):
            if not isinstance(a, DeviceArray):
                raise TypeError(f"{name}: expected a DeviceArray, got {type(a).__name__}")
            need = vecs * ops.kv_vec_bytes(kv_dt, dim)
            if a.nbytes < need:
                raise ValueError(f"{name}: {a.nbytes} bytes, needs {need}")
        if kv_dt != ops.KV_F32:
            if k_scale is None or v_scale is None:
                raise ValueError("integer pages need k_scale and v_scale")
            ops._need(k_scale, vecs, np.float32, "k_scale")
            ops._need(v_scale, vecs, np.float32, "v_scale")
        else:
            k_scale = v_scale = None
        self.kv_dt, self.k, self.v, self.k_scale, self.v_scale = kv_dt, k, v, k_scale, v_scale
        self.n_pages, self.page, self.n_head_kv = int(n_pages), int(page), int(n_head_kv)
        self.head_dim, self.value_dim = int(head_dim), int(value_dim)
        self.n_layers = int(n_layers)
        self.struct = _lib.KvPool(kv_dt, page, n_layers, n_pages, n_head_kv, head_dim, value_dim,
                                  k.ptr, v.ptr, None if k_scale is None else k_scale.ptr,
                                  None if v_scale is None else v_scale.ptr)
        self.ref = ctypes.byref(self.struct)

    @classmethod
    def empty(cls, kv_dt: int, n_pages: int, page: int, n_head_kv: int, head_dim: int,
              value_dim: int | None = None, n_layers: int = 1) -> "KvPool":
        """A pool in new device memory (its contents undefined)."""
        value_dim = head_dim if value_dim is None else value_dim
        vecs = n_layers * n_pages * n_head_kv * page
        kind = np.float32 if kv_dt == ops.KV_F32 else np.uint8

        def side(dim):
            return DeviceArray.empty(vecs * ops.kv_vec_bytes(kv_dt, dim) // np.dtype(kind).itemsize,
                                     kind)

        scales = (None, None) if kv_dt == ops.KV_F32 else (DeviceArray.empty(vecs),
                                                           DeviceArray.empty(vecs))
        return cls(kv_dt, side(head_dim), side(value_dim), n_pages, page, n_head_kv, head_dim,
                   value_dim, n_layers, *scales)


class PagedKV:
    """Which page holds what: up to max_seqs sequences of up to max_pages pages.

    Device arrays, changed in stream order by the methods: `table` [max_seqs,
    max_pages] (-1: no page), `lens` [max_seqs] (0: a free slot) and `step`
    [max_seqs], the lengths of the sequences that the last append() named and 0
    elsewhere: with it as a call's lens, the other slots are padding rows.

    One thread and one stream at a time: a page that is given up may be handed
    out again by the next call, which only the stream's order protects. The
    methods change state by the call and are refused while a plan records.

    A method that raises has changed nothing here. Where it was a launch that
    failed, the device arrays may hold part of the change until the next append,
    fork, truncate, trim, free or compact that does not, which writes what they
    should hold."""

    def __init__(self, pool: KvPool, max_seqs: int, max_pages: int):
        if max_seqs <= 0 or max_pages <= 0 or max_pages * pool.page > 1 << 30:
            raise ValueError(f"PagedKV: {max_seqs} sequences of {max_pages} pages")
        self.pool, self.max_seqs, self.max_pages = pool, int(max_seqs), int(max_pages)
        n = max_seqs * max_pages
        self._dev = DeviceArray.empty(n + 2 * max_seqs, np.int32)
        host = np.zeros(n + 2 * max_seqs, np.int32)
        host[:n] = -1
        self._dev.copy_from(host)
        self.table = self._dev.view((max_seqs, max_pages))
        self.lens = self._dev.view((max_seqs,), offset_bytes=4 * n)
        self.step = self._dev.view((max_seqs,), offset_bytes=4 * (n + max_seqs))
        self._host = host                      # what the device will hold
        self._refs = np.zeros(pool.n_pages, np.int64)
        self._free = list(range(pool.n_pages))   # a heap: the lowest page first
        self._live: set[int] = set()
        self._window: dict[int, int] = {}      # of the slots that trim has been at
        self._edits: dict[int, int] = {}
        self._undo: list[tuple] = []           # (array, place, value) before a change

    # ------------------------------------------------------------ what there is
    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def used_pages(self) -> int:
        return self.pool.n_pages - len(self._free)

    def length(self, slot: int) -> int:
        return int(self._host[self._lens_at(self._slot(slot))])

    def pages(self, slot: int) -> list[int]:
        """The slot's table row up to its last page (-1: given up by trim)."""
        s = self._slot(slot)
        return self._row(s)[: -(-self.length(s) // self.pool.page)].tolist()

    def rows(self, first: int, n: int = 1):
        """(table, lens) views of slots first .. first + n - 1."""
        if first < 0 or n <= 0 or first + n > self.max_seqs:
            raise ValueError(f"slots {first} .. {first + n - 1} of {self.max_seqs}")
        return (self.table.view((n, self.max_pages), offset_bytes=4 * first * self.max_pages),
                self.lens.view((n,), offset_bytes=4 * first))

    # ---------------------------------------------------------------- sequences
    def add(self) -> int:
        """A free slot (the lowest), empty."""
        self._check()
        for s in range(self.max_seqs):
            if s not in self._live:
                self._live.add(s)
                return s
        raise ValueError(f"all {self.max_seqs} slots are taken")

    def append(self, slots, n: int = 1, stream: Stream | None = None) -> None:
        """Room for n new tokens of each slot: lens grow by n, pages are taken, and
        a page shared with another sequence that the new tokens would write is
        copied first. All or nothing (OutOfPages, ValueError)."""
        self._check()
        slots = [self._slot(s) for s in slots]
        if n <= 0 or len(set(slots)) != len(slots):
            raise ValueError("append: n must be positive and no slot named twice")
        page, refs = self.pool.page, {}
        copies, news, need = [], [], 0
        for s in slots:
            have = self.length(s)
            if have + n > self.max_pages * page:
                raise ValueError(f"slot {s}: {have} + {n} tokens are more than {self.max_pages} "
                                 f"pages of {page}")
            old = -(-have // page)
            if have % page:
                p = int(self._row(s)[old - 1])
                r = refs.get(p, int(self._refs[p]))
                if r > 1:
                    refs[p] = r - 1
                    copies.append((s, old - 1, p))
                    need += 1
            more = -(-(have + n) // page) - old
            news.append((s, old, more, have + n))
            need += more
        if need > len(self._free):
            raise OutOfPages(f"append needs {need} pages, {len(self._free)} are free")
        with self._change(stream):
            pairs = []
            for s, col, p in copies:
                new = self._take()
                self._drop(p)
                self._set(s * self.max_pages + col, new)
                pairs.append((p, new))
            step = [0] * self.max_seqs
            for s, old, more, length in news:
                for c in range(old, old + more):
                    self._set(s * self.max_pages + c, self._take())
                self._set(self._lens_at(s), length)
                step[s] = length
            for s, length in enumerate(step, self._lens_at(self.max_seqs)):
                self._set(s, length)
            if pairs:
                ops.kv_pages_copy(self.pool, [a for a, _ in pairs], [b for _, b in pairs], stream)

    def fork(self, slot: int, stream: Stream | None = None) -> int:
        """A new slot with the same tokens, in the same pages."""
        s = self._slot(slot)
        d = self.add()
        row, n = self._row(s), self.length(s)
        try:
            with self._change(stream):
                for c in range(-(-n // self.pool.page)):
                    p = int(row[c])
                    if p >= 0:
                        self._ref(p, 1)
                    self._set(d * self.max_pages + c, p)
                self._set(self._lens_at(d), n)
        except BaseException:
            self._live.discard(d)
            raise
        if s in self._window:
            self._window[d] = self._window[s]
        return d

    def truncate(self, slot: int, n: int, stream: Stream | None = None) -> None:
        """Keep the slot's first n tokens (a rejected guess, a shorter prompt).
        Refused where trim has given up a page in the last trim's window of the
        newest of them: trim with a window that is longer by what may be taken back."""
        self._check()
        s = self._slot(slot)
        have = self.length(s)
        if n < 0 or n > have:
            raise ValueError(f"slot {s} holds {have} tokens, not {n}")
        page = self.pool.page
        seen = self._row(s)[max(0, n - self._window.get(s, n)) // page: -(-n // page)]
        if (seen < 0).any():
            raise ValueError(f"slot {s}: pages that token {n - 1} sees were given up by trim")
        with self._change(stream):
            for c in range(-(-n // page), -(-have // page)):
                self._clear(s, c)
            self._set(self._lens_at(s), n)
            self._set(self._lens_at(s) + self.max_seqs, 0)

    def trim(self, slot: int, window: int, sinks: int = 0, stream: Stream | None = None) -> int:
        """Give up the pages that neither the newest token nor a later one sees
        under `window` and `sinks`; the number given up. What one call gives up stays
        so: a later call with more sinks or a longer window does not bring it back
        (pages() has -1 there, attention does not see those keys and sets its `bad`)."""
        self._check()
        s = self._slot(slot)
        if window <= 0 or sinks < 0:
            raise ValueError(f"trim: window {window}, sinks {sinks}")
        page, gone = self.pool.page, 0
        with self._change(stream):
            for c in range(-(-sinks // page), max(0, self.length(s) - window) // page):
                if self._row(s)[c] >= 0:
                    self._clear(s, c)
                    gone += 1
        self._window[s] = int(window)
        return gone

    def free(self, slot: int, stream: Stream | None = None) -> None:
        """End a sequence: its slot and the pages that no other one shares."""
        self.truncate(slot, 0, stream)
        self._live.discard(int(slot))
        self._window.pop(int(slot), None)

    def compact(self, stream: Stream | None = None) -> int:
        """Move the pages in use to the front of the pool (in every layer), so
        that pages used_pages .. n_pages - 1 are free; the number moved."""
        self._check()
        used = self.used_pages
        holes = [p for p in sorted(self._free) if p < used]
        tail = [p for p in range(used, self.pool.n_pages) if self._refs[p] > 0]
        to = dict(zip(tail, holes))
        with self._change(stream):
            if tail:
                ops.kv_pages_copy(self.pool, tail, holes, stream)
            for a, b in to.items():
                self._ref(b, int(self._refs[a]))
                self._ref(a, -int(self._refs[a]))
            self._free = list(range(used, self.pool.n_pages))
            for s in self._live:
                row = self._row(s)
                for c in range(-(-self.length(s) // self.pool.page)):
                    p = int(row[c])
                    if p in to:
                        self._set(s * self.max_pages + c, to[p])
        return len(tail)

    # ------------------------------------------------------------------ helpers
    def _check(self) -> None:
        if recording_plan() is not None:
            raise RuntimeError("a PagedKV changes by the call and cannot be recorded in a plan")

    def _slot(self, slot: int) -> int:
        s = int(slot)
        if s not in self._live:
            raise ValueError(f"slot {slot} is not in use")
        return s

    def _lens_at(self, s: int) -> int:
        return self.max_seqs * self.max_pages + s

    def _row(self, s: int) -> np.ndarray:
        return self._host[s * self.max_pages: (s + 1) * self.max_pages]

    @contextlib.contextmanager
    def _change(self, stream: Stream | None):
        """A change of tables, lengths and pages, written to the device at its end;
        taken back where something raises (its edits, of which the device may have
        some, then become those that write the old values)."""
        try:
            yield
            if self._edits:
                ops.write_i32(self._dev, sorted(self._edits.items()), stream)
        except BaseException:
            for a, at, value in reversed(self._undo):
                a[at] = value
            self._free = np.flatnonzero(self._refs == 0).tolist()   # (ascending: a heap)
            self._edits = {at: int(self._host[at]) for at in self._edits}
            raise
        else:
            self._edits.clear()
        finally:
            self._undo.clear()

    def _ref(self, p: int, by: int) -> None:
        self._undo.append((self._refs, p, int(self._refs[p])))
        self._refs[p] += by

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._ref(p, 1)
        return p

    def _drop(self, p: int) -> None:
        self._ref(p, -1)
        if self._refs[p] == 0:
            heapq.heappush(self._free, p)

    def _clear(self, s: int, c: int) -> None:
        p = int(self._row(s)[c])
        if p >= 0:
            self._drop(p)
        self._set(s * self.max_pages + c, -1)

    def _set(self, at: int, value: int) -> None:
        if self._host[at] != value:
            self._undo.append((self._host, at, int(self._host[at])))
            self._host[at] = value
            self._edits[at] = value
