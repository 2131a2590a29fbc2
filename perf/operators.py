"""What a program that serves several sequences has the framework do with its
key-value caches: attention of new tokens over a paged cache, attention with a
sliding window and first tokens that stay visible, rows written into pages and
read back, pages copied for forks and compaction.

Layouts: a pool holds K [layers][pages][kv heads][page][dim], V the same, and for
integer caches one fp32 scale a vector [layers][pages][kv heads][page]; a table
row lists a sequence's pages, lens counts its tokens, the new ones included. A
contiguous cache is [n_kv][kv heads][dim].

Cache types: 0 fp32, 1 int8 (scale amax / 127), 2 int4 (amax / 7, two codes a
byte, the low nibble first).
"""
import math

import numpy as np
import torch

own = False

GEOMETRIES = ((14, 2, 64), (32, 8, 64), (32, 8, 128), (64, 8, 128), (8, 4, 256), (16, 2, 256))


def listed():
    return [
        # one chat on a small model a few hundred tokens in: the shortest call,
        # where each launch and memory round trip counts
        dict(name="paged_chat", kind="paged", heads=14, kv_heads=2, dim=64, dt=1, page=16, seqs=1,
             n_q=1, max_len=333, window=0, sinks=0),
        # a serving batch: 48 rows of very different lengths, the last a padding
        # row of no tokens, int8 pages of 16 tokens
        dict(name="paged_batch_int8", kind="paged", heads=32, kv_heads=8, dim=128, dt=1, page=16,
             seqs=48, n_q=1, max_len=8192, window=0, sinks=0),
        # a few long documents at full precision: the largest read
        dict(name="paged_long_fp32", kind="paged", heads=64, kv_heads=8, dim=128, dt=0, page=64,
             seqs=4, n_q=1, max_len=50001, window=0, sinks=0),
        # a sliding-window layer of head dim 256, 3 tokens a step (a speculative
        # step), pages behind the window never read
        dict(name="paged_window_d256", kind="paged", heads=8, kv_heads=4, dim=256, dt=1, page=32,
             seqs=64, n_q=3, max_len=6000, window=1024, sinks=4),
        # a prompt through a windowed layer with sinks
        dict(name="sinks_prompt", kind="sinks", heads=32, kv_heads=8, dim=128, dt=0, n_q=2048,
             n_kv=2048, window=512, sinks=4, ring=False),
        # an odd piece of a long prompt after cached tokens, small heads
        dict(name="sinks_piece_d64", kind="sinks", heads=14, kv_heads=2, dim=64, dt=0, n_q=1001,
             n_kv=9001, window=1024, sinks=16, ring=False),
        # one token over a long int8 cache of which the window and the sinks count
        dict(name="sinks_decode_int8", kind="sinks", heads=32, kv_heads=8, dim=128, dt=1, n_q=1,
             n_kv=32768, window=4096, sinks=4, ring=False),
        # one token over a bounded cache: the sinks, then a ring of the window
        dict(name="sinks_ring_fp32", kind="sinks", heads=8, kv_heads=4, dim=256, dt=0, n_q=1,
             n_kv=2052, window=2048, sinks=4, ring=True),
        # a prompt's keys and values into fp32 pages
        dict(name="write_prompt_fp32", kind="rows", kv_heads=8, dim=128, dt=0, page=64, seqs=1,
             n_q=1999, max_len=2500),
        # a serving step's new rows quantised into their pages, and read back
        dict(name="write_read_int8", kind="rows", kv_heads=8, dim=128, dt=1, page=16, seqs=64,
             n_q=4, max_len=3000),
        # sixteen forks: the pages that parent and child would both write, in
        # every layer
        dict(name="pages_fork_int8", kind="pages", layers=32, kv_heads=8, dim=128, dt=1, page=16,
             n_pages=400, moves=16, what="fork"),
        # a pool made dense again: pages behind the last used place into holes
        dict(name="pages_compact_fp32", kind="pages", layers=16, kv_heads=8, dim=128, dt=0,
             page=64, n_pages=160, moves=61, what="compact"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(("paged", "paged", "paged", "sinks", "sinks", "sinks", "rows", "pages"))
    h, hk, d = rng.choice(GEOMETRIES)
    dt = rng.choice((0, 1, 1, 2))
    page = rng.choice((16, 16, 32, 64, 128))
    if kind == "paged":
        window = rng.choice((0, 0, _log(rng, 64, 4096)))
        return dict(kind=kind, heads=h, kv_heads=hk, dim=d, dt=dt, page=page,
                    seqs=_log(rng, 1, 128), n_q=rng.choice((1, 1, 1, 2, 3, 5)),
                    max_len=_log(rng, 16, 50000), window=window,
                    sinks=rng.choice((0, 1, 4, 16)) if window else 0)
    if kind == "sinks":
        window, sinks = _log(rng, 64, 4096), rng.choice((1, 4, 4, 16, 64))
        if rng.random() < 0.5:
            if rng.random() < 0.5:
                return dict(kind=kind, heads=h, kv_heads=hk, dim=d, dt=dt, n_q=1,
                            n_kv=window + sinks, window=window, sinks=sinks, ring=True)
            return dict(kind=kind, heads=h, kv_heads=hk, dim=d, dt=dt, n_q=rng.choice((1, 1, 4)),
                        n_kv=_log(rng, 64, 32768), window=window, sinks=sinks, ring=False)
        n_q = _log(rng, 24, 2048)
        return dict(kind=kind, heads=h, kv_heads=hk, dim=d, dt=rng.choice((0, 0, dt)), n_q=n_q,
                    n_kv=n_q + rng.choice((0, 0, _log(rng, 16, 8192))), window=window, sinks=sinks,
                    ring=False)
    if kind == "rows":
        n_q = rng.choice((1, 1, 4, _log(rng, 16, 2048)))
        seqs = _log(rng, 1, 128) if n_q <= 4 else rng.choice((1, 2, 4))
        return dict(kind=kind, kv_heads=hk, dim=d, dt=dt, page=page, seqs=seqs, n_q=n_q,
                    max_len=n_q + _log(rng, 1, 3000))
    n_pages = _log(rng, 40, 400)
    return dict(kind=kind, layers=_log(rng, 1, 32), kv_heads=hk, dim=d, dt=dt, page=page,
                n_pages=n_pages, moves=rng.randint(1, n_pages // 3),
                what=rng.choice(("fork", "compact")))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _state_bytes(case):
    """About what a state and the plain form's gathered copies take."""
    k = case["kind"]
    if k == "paged":
        return case["seqs"] * case["max_len"] * case["kv_heads"] * case["dim"] * 16
    if k == "sinks":
        return case["heads"] * case["n_q"] * case["n_kv"] * 8
    if k == "rows":
        return case["seqs"] * case["max_len"] * case["kv_heads"] * case["dim"] * 8
    return case["layers"] * case["n_pages"] * _page_bytes(case)


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= top and _state_bytes(c) <= 12e9:
            return c


# --------------------------------------------------------------------- sizes
def _vec(dt, dim):
    return {0: 4 * dim, 1: dim, 2: dim // 2}[dt]


def _page_bytes(case):
    """Bytes of one page in one layer: K, V and the scales."""
    n = case["kv_heads"] * case["page"]
    return 2 * n * (_vec(case["dt"], case["dim"]) + (4 if case["dt"] else 0))


def _lens(case):
    """The rows' lengths: the first the longest, the others spread towards
    short ones; from eight rows on the last is padding (no tokens)."""
    n, lo, hi = case["seqs"], case["n_q"], case["max_len"]
    lens = [max(lo, int(hi * ((i * 0.6180339887 + 0.999) % 1) ** 2)) for i in range(n)]
    lens[0] = max(lo, hi)
    if n >= 8:
        lens[-1] = 0
    return lens


def _visible(p, window, sinks):
    """Keys that a query at position p sees in a cache that holds them all."""
    if window <= 0 or p + 1 <= window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def _reach(p0, p1, window, sinks):
    """Keys that some query of positions p0 .. p1 sees."""
    if window <= 0:
        return p1 + 1
    first = max(0, p0 - window + 1)
    return p1 + 1 - first + min(sinks, first)


def work(case):
    k = case["kind"]
    if k in ("paged", "sinks"):
        h, hk, d, nq, w, s = (case[x] for x in ("heads", "kv_heads", "dim", "n_q", "window",
                                               "sinks"))
        key = 2 * hk * (_vec(case["dt"], d) + (4 if case["dt"] else 0))
        if k == "paged":
            lens = [n for n in _lens(case) if n >= nq]
            rows, table = case["seqs"], sum(-(-n // case["page"]) for n in lens) * 4
        else:
            lens, rows, table = [case["n_kv"]], 1, 4 * nq
        pairs = sum(_visible(n - nq + t, w, s) for n in lens for t in range(nq))
        keys = sum(_reach(n - nq, n - 1, w, s) for n in lens)
        return {"bytes": keys * key + 2 * rows * nq * h * d * 4 + table, "flops": 4 * h * d * pairs}
    if k == "rows":
        n = sum(min(x, case["n_q"]) for x in _lens(case)) * case["kv_heads"]
        vec = _vec(case["dt"], case["dim"]) + (4 if case["dt"] else 0)
        once = 2 * n * (4 * case["dim"] + vec)
        return {"bytes": once * (2 if case["dt"] else 1), "flops": 2 * n * case["dim"]}
    return {"bytes": 2 * case["moves"] * case["layers"] * _page_bytes(case), "flops": 0}


# -------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 41)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _quantise(x, dt):
    """(codes, scales) of vectors along the last axis; (x, None) in fp32. The
    scale and the quotient are fp32, halves go away from zero."""
    if dt == 0:
        return x, None
    top = 127.0 if dt == 1 else 7.0
    amax = x.abs().amax(-1)
    scale = torch.where(amax > 0, amax / top, torch.ones_like(amax))
    r = x / scale[..., None]
    t = torch.trunc(r)
    c = (t + torch.sign(r) * ((r - t).abs() >= 0.5)).clamp(-top, top)
    if dt == 1:
        return c.to(torch.int8), scale
    c = c.to(torch.int32) & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), scale


def _values(codes, scale, dt):
    """The fp32 values that stored vectors stand for."""
    if dt == 0:
        return codes
    if dt == 2:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int32)
        codes = (c ^ 8) - 8
    return codes.to(torch.float32) * scale[..., None]


def _cache(g, dt, *shape):
    return _quantise(_randn(g, *shape), dt)


def _pages(case, g, lens):
    """A table over a shuffled pool with a few pages to spare, -1 where a row
    has no page."""
    need = [-(-n // case["page"]) for n in lens]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return n_pages, table


def prepare(case, seed):
    g, k = _gen(seed), case["kind"]
    s = {"case": case}
    hk, d, dt = case["kv_heads"], case["dim"], case["dt"]
    if k == "paged":
        lens = _lens(case)
        n_pages, s["table"] = _pages(case, g, lens)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        shape = (1, n_pages, hk, case["page"], d)
        s["k"], s["ks"] = _cache(g, dt, *shape)
        s["v"], s["vs"] = _cache(g, dt, *shape)
        s["q"] = _randn(g, case["seqs"], case["n_q"], case["heads"], d)
        s["out"] = torch.zeros_like(s["q"])
    elif k == "sinks":
        n_q, n_kv = case["n_q"], case["n_kv"]
        s["k"], s["ks"] = _cache(g, dt, n_kv, hk, d)
        s["v"], s["vs"] = _cache(g, dt, n_kv, hk, d)
        s["q"] = _randn(g, n_q, case["heads"], d)
        s["out"] = torch.zeros_like(s["q"])
        slots = torch.arange(n_kv, dtype=torch.int32, device="cuda")
        last = n_kv - 1
        s["kpos"] = None
        if case["ring"]:       # sinks in the first slots, a ring of the window behind them
            ring, sinks = n_kv - case["sinks"], case["sinks"]
            last += 2 * ring + int(seed) % ring
            newest = last - (last - sinks - (slots - sinks)) % ring
            s["kpos"] = torch.where(slots < sinks, slots, newest).to(torch.int32)
        s["qpos"] = torch.arange(last - n_q + 1, last + 1, dtype=torch.int32, device="cuda")
    elif k == "rows":
        lens = _lens(case)
        n_pages, s["table"] = _pages(case, g, lens)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        shape = (1, n_pages, hk, case["page"], d)
        s["k"], s["ks"] = _cache(g, dt, *shape)
        s["v"], s["vs"] = _cache(g, dt, *shape)
        s["k_new"] = _randn(g, case["seqs"], case["n_q"], hk, d)
        s["v_new"] = _randn(g, case["seqs"], case["n_q"], hk, d)
        s["k_out"], s["v_out"] = torch.zeros_like(s["k_new"]), torch.zeros_like(s["v_new"])
    else:
        shape = (case["layers"], case["n_pages"], hk, case["page"], d)
        s["k"], s["ks"] = _cache(g, dt, *shape)
        s["v"], s["vs"] = _cache(g, dt, *shape)
        n, m = case["n_pages"], case["moves"]
        if case["what"] == "fork":      # any used page to any free one
            p = torch.randperm(n, generator=g, device="cuda")
            src, dst = p[:m], p[m:2 * m]
        else:                           # the last pages into holes below them
            src = torch.arange(n - m, n, device="cuda")
            dst = torch.randperm(n - m, generator=g, device="cuda")[:m].sort().values
        s["src"], s["dst"] = src, dst
        s["src_host"] = src.cpu().numpy().astype(np.int32)
        s["dst_host"] = dst.cpu().numpy().astype(np.int32)
    return s


# ------------------------------------------------------------- the plain form
def _softmax_rows(scores, keep):
    """exp(s - max) over the kept keys, and its sum (1 where nothing is kept)."""
    s = torch.where(keep, scores, torch.full_like(scores, -math.inf))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    z = e.sum(-1, keepdim=True)
    return e, torch.where(z > 0, z, torch.ones_like(z))


def _keep(qpos, kpos, window, sinks):
    """qpos [..., Q, 1], kpos [..., 1, J] -> [..., Q, J]"""
    keep = kpos <= qpos
    if window > 0:
        keep = keep & ((qpos - kpos < window) | (kpos < sinks))
    return keep


def _paged(s):
    c = s["case"]
    S, nq, h, hk, d = c["seqs"], c["n_q"], c["heads"], c["kv_heads"], c["dim"]
    at = s["table"].clamp(min=0).long()

    def rows(x, scale):       # [S, hk, keys, d]
        x = _values(x[0][at], None if scale is None else scale[0][at], c["dt"])
        return x.permute(0, 2, 1, 3, 4).reshape(S, hk, -1, d)

    K, V = rows(s["k"], s["ks"]), rows(s["v"], s["vs"])
    q = s["q"].reshape(S, nq, hk, h // hk, d).permute(0, 2, 1, 3, 4)
    scores = (q.reshape(S, hk, -1, d) @ K.transpose(-1, -2)) * d ** -0.5
    j = torch.arange(K.shape[2], device="cuda")
    p = s["lens"].long()[:, None] - nq + torch.arange(nq, device="cuda")
    keep = _keep(p[:, :, None], j, c["window"], c["sinks"]) & (p >= 0)[:, :, None]
    keep = keep[:, None, :, None, :].expand(S, hk, nq, h // hk, -1).reshape(scores.shape)
    e, z = _softmax_rows(scores, keep)
    out = ((e @ V) / z).reshape(S, hk, nq, h // hk, d)
    return out.permute(0, 2, 1, 3, 4).reshape(S, nq, h, d)


def _sinks(s):
    c = s["case"]
    nq, h, hk, d = c["n_q"], c["heads"], c["kv_heads"], c["dim"]
    K = _values(s["k"], s["ks"], c["dt"]).permute(1, 0, 2)
    V = _values(s["v"], s["vs"], c["dt"]).permute(1, 0, 2)
    q = s["q"].reshape(nq, hk, h // hk, d).permute(1, 0, 2, 3).reshape(hk, -1, d)
    scores = (q @ K.transpose(-1, -2)) * d ** -0.5
    kpos = torch.arange(c["n_kv"], device="cuda") if s["kpos"] is None else s["kpos"].long()
    keep = _keep(s["qpos"].long()[:, None], kpos, c["window"], c["sinks"])
    keep = keep[None, :, None, :].expand(hk, nq, h // hk, -1).reshape(scores.shape)
    e, z = _softmax_rows(scores, keep)
    out = ((e @ V) / z).reshape(hk, nq, h // hk, d)
    return out.permute(1, 0, 2, 3).reshape(nq, h, d)


def _rows(s):
    c = s["case"]
    nq, page = c["n_q"], c["page"]
    p = s["lens"].long()[:, None] - nq + torch.arange(nq, device="cuda")
    has = p >= 0
    row = torch.arange(c["seqs"], device="cuda")[:, None].expand_as(p)[has]
    at = s["table"][row, p[has] // page].long()
    off = p[has] % page
    outs = []
    for new, pool, scales in (("k_new", "k", "ks"), ("v_new", "v", "vs")):
        codes, scale = _quantise(s[new][has], c["dt"])
        s[pool][0, at, :, off] = codes
        if scale is None:
            outs.append(s[pool])
            continue
        s[scales][0, at, :, off] = scale
        back = torch.zeros_like(s[new])
        back[has] = _values(s[pool][0, at, :, off], s[scales][0, at, :, off], c["dt"])
        outs.append(back)
    return tuple(outs)


def _copied(s):
    pools = [s[x] for x in ("k", "v", "ks", "vs") if s[x] is not None]
    for x in pools:
        x[:, s["dst"]] = x[:, s["src"]]
    return tuple(pools)


# -------------------------------------------------------- the framework's calls
def _handles(s):
    """What a program holds beside its buffers: the pool's description, arrays
    over the buffers and, for single tokens, the recorded step."""
    from aero_amd import ops
    from aero_amd.device import DeviceArray, Plan
    from aero_amd.paged import KvPool

    def array(t):
        if t is None:
            return None
        kind = {torch.float32: np.float32, torch.int32: np.int32, torch.int8: np.int8,
                torch.uint8: np.uint8}[t.dtype]
        return DeviceArray(tuple(t.shape), kind, _ptr=t.data_ptr(), _owner=False, _base=t)

    c = s["case"]
    a = {x: array(t) for x, t in s.items() if isinstance(t, torch.Tensor) and
         t.dtype != torch.int64}
    if c["kind"] != "sinks":
        a["pool"] = KvPool(c["dt"], a["k"], a["v"], s["k"].shape[1], c["page"], c["kv_heads"],
                           c["dim"], n_layers=s["k"].shape[0], k_scale=a.get("ks"),
                           v_scale=a.get("vs"))

    def step():
        if c["kind"] == "paged":
            ops.paged_attention(a["pool"], 0, a["q"], a["out"], a["table"], a["lens"], c["seqs"],
                                c["heads"], c["dim"] ** -0.5, n_q=c["n_q"], window=c["window"],
                                sinks=c["sinks"])
        elif c["kind"] == "sinks":
            ops.attention(a["q"], a["k"], a["v"], a["out"], c["n_q"], c["heads"], c["kv_heads"],
                          c["dim"], c["dim"], c["n_kv"], c["dim"] ** -0.5, qpos=a["qpos"],
                          kpos=a.get("kpos"), window=c["window"], kv_dt=c["dt"],
                          k_scale=a.get("ks"), v_scale=a.get("vs"), sinks=c["sinks"])
        elif c["kind"] == "rows":
            ops.paged_kv_write(a["pool"], 0, a["k_new"], a["v_new"], a["table"], a["lens"],
                               c["seqs"], n_q=c["n_q"])
            if c["dt"]:
                ops.paged_kv_read(a["pool"], 0, a["k_out"], a["v_out"], a["table"], a["lens"],
                                  c["seqs"], n_q=c["n_q"])
        else:
            ops.kv_pages_copy(a["pool"], s["src_host"], s["dst_host"])

    if c.get("n_q") == 1:       # a serving step is recorded once and replayed
        plan = Plan()
        with plan:
            step()
        return plan.launch
    return step


def _call(s):
    if "step" not in s:
        s["step"] = _handles(s)
    s["step"]()
    k = s["case"]["kind"]
    if k in ("paged", "sinks"):
        return s["out"]
    if k == "rows":
        return (s["k_out"], s["v_out"]) if s["case"]["dt"] else (s["k"], s["v"])
    return tuple(s[x] for x in ("k", "v", "ks", "vs") if s[x] is not None)


def run(s):
    if own:
        return _call(s)
    return {"paged": _paged, "sinks": _sinks, "rows": _rows, "pages": _copied}[s["case"]["kind"]](s)


# ------------------------------------------------------------- in 64 bits
def _double(codes, scale, dt):
    if dt == 0:
        return codes.double()
    if dt == 2:
        b = codes.long()
        both = torch.cat([(b % 16)[..., None], (b // 16)[..., None]], -1).reshape(*b.shape[:-1], -1)
        codes = torch.where(both > 7, both - 16, both)
    return codes.double() * scale.double()[..., None]


def _attend64(q, K, V, seen, scale):
    """One query row set [r, d] over K, V [keys, d], seen [keys]."""
    at = torch.nonzero(seen)[:, 0]
    if at.numel() == 0:
        return torch.zeros(q.shape[0], V.shape[1], dtype=torch.float64, device="cuda")
    w = torch.softmax(torch.mm(q.double(), K[at].t().contiguous()) * scale, 1)
    return torch.mm(w, V[at])


def exact(case, seed):
    k = case["kind"]
    if k == "pages":
        return None
    s = prepare(case, seed)
    if k == "rows":
        nq, page, outs = case["n_q"], case["page"], []
        top = {0: 0, 1: 127, 2: 7}[case["dt"]]
        lens, table = s["lens"].tolist(), s["table"].tolist()
        for new, pool in (("k_new", "k"), ("v_new", "v")):
            x = s[new].double()
            if top:     # the scale and the quotient are defined in fp32
                a = x.abs().amax(-1, keepdim=True)
                sc = torch.where(a > 0, (a / top).float().double(), torch.ones_like(a))
                r = (x / sc).float().double()
                c = torch.floor(r.abs() + 0.5).clamp(max=top) * torch.sign(r)
                y = c * sc
                for i, n in enumerate(lens):
                    y[i, :max(0, nq - n)] = 0
            else:
                y = s[pool].double()
                for i, n in enumerate(lens):
                    for u in range(max(0, n - nq), n):
                        y[0, table[i][u // page], :, u % page] = x[i, u - n + nq]
            outs.append(y)
        return tuple(outs)
    h, hk, d, nq = case["heads"], case["kv_heads"], case["dim"], case["n_q"]
    rep, scale, w, sinks = h // hk, d ** -0.5, case["window"], case["sinks"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    if k == "paged":
        lens, table = s["lens"].tolist(), s["table"]
        for i, n in enumerate(lens):
            if n == 0:
                continue
            at = table[i, :-(-n // case["page"])].long()

            def flat(x, sc):
                x = _double(x[0, at], None if sc is None else sc[0, at], case["dt"])
                return x.transpose(0, 1).reshape(hk, -1, d)[:, :n]

            K, V = flat(s["k"], s["ks"]), flat(s["v"], s["vs"])
            j = torch.arange(n, device="cuda")
            for t in range(max(0, nq - n), nq):
                p = n - nq + t
                seen = (j <= p) & ((j > p - w) | (j < sinks)) if w else j <= p
                for a in range(hk):
                    out[i, t, a * rep:(a + 1) * rep] = _attend64(
                        s["q"][i, t, a * rep:(a + 1) * rep], K[a], V[a], seen, scale)
        return out
    K, V = _double(s["k"], s["ks"], case["dt"]), _double(s["v"], s["vs"], case["dt"])
    j = s["kpos"].long() if s["kpos"] is not None else torch.arange(case["n_kv"], device="cuda")
    for a in range(hk):
        Ka, Va = K[:, a].t().contiguous(), V[:, a].contiguous()
        for t in range(0, nq, 256):
            p = s["qpos"][t:t + 256].long()[:, None]
            hide = (j > p) | ((j <= p - w) & (j >= sinks))
            x = torch.matmul(s["q"][t:t + 256, a * rep:(a + 1) * rep].double(), Ka) * scale
            x = torch.softmax(x.masked_fill(hide[:, None, :], -math.inf), -1)
            out[t:t + 256, a * rep:(a + 1) * rep] = torch.matmul(x, Va)
    return out
