"""What a program that runs a model in microscaled numbers has the framework do:
rows quantised in blocks of 32 values that share a power of two, the norms and
activations of a layer with such an output, and the product of such rows with
4-bit weights.

Formats: 0, 8 bits: whole numbers -127 .. 127 in units of 2^-6 of the scale; 1,
4 bits: a sign, two bits of exponent and one of mantissa (0 .5 1 1.5 2 3 4 6), two
codes a byte, the low nibble first. A scale is a byte s that stands for 2^(s-127),
one for each 32 values of a row, 255 for a block that holds NaN or an infinity. It
is the smallest under which the block's largest value does not pass the format's
largest (127/64, 6), and not below 4 in 8 bits; a value goes to the nearest code,
halves to the even one. Norms and activations are rounded to fp32 once, then
quantised.
"""
import math

import numpy as np
import torch

own = False

INT8, FP4 = 0, 1
#: (least scale byte, exponent of the largest value, its mantissa's bits in fp32)
_TOP = ((4, 0, 0x7E0000), (0, 2, 0x400000))
EPS = 1e-5


def listed():
    return [
        # a weight matrix to 4 bits when a model is loaded, read back to look at
        dict(name="quantize_weight_fp4", kind="quantize", fmt=FP4, rows=4096, cols=14336),
        # a decode batch's attention outputs, before the output projection
        dict(name="quantize_batch_int8", kind="quantize", fmt=INT8, rows=64, cols=8192),
        # the shortest call: one token of a small model, residual and norm
        dict(name="norm_token_int8", kind="norm", fmt=INT8, rows=1, cols=896, add=True, unit=False),
        # a long prompt on a large model: the largest stream
        dict(name="norm_long_int8", kind="norm", fmt=INT8, rows=16384, cols=8192, add=True,
             unit=False),
        # an odd batch through a (1 + w) norm to 4 bits, no residual
        dict(name="norm_odd_fp4", kind="norm", fmt=FP4, rows=333, cols=2560, add=False, unit=True),
        # SwiGLU of a prompt, gate and up side by side as one product leaves them
        dict(name="act_prompt_int8", kind="act", fmt=INT8, act="silu", rows=512, cols=14336),
        # GeGLU of an odd prompt, to 4 bits
        dict(name="act_gelu_fp4", kind="act", fmt=FP4, act="gelu_tanh", rows=2047, cols=10240),
        # one token of a small model: latency
        dict(name="product_token_int8", kind="product", fmt=INT8, tokens=1, rows=9728, cols=896),
        # a decode batch over a large matrix: the weights' bytes
        dict(name="product_batch_int8", kind="product", fmt=INT8, tokens=64, rows=28672, cols=8192),
        # the down projection of a prompt: a long sum, few tiles
        dict(name="product_down_int8", kind="product", fmt=INT8, tokens=512, rows=4096, cols=14336),
        # gate and up of a long prompt in one product: the largest
        dict(name="product_prompt_int8", kind="product", fmt=INT8, tokens=2048, rows=28672,
             cols=4096),
        # both sides in 4 bits, an odd number of tokens
        dict(name="product_odd_fp4", kind="product", fmt=FP4, tokens=333, rows=2560, cols=10240),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(("quantize", "norm", "act", "product", "product", "product"))
    fmt = rng.choice((INT8, INT8, FP4))
    cols = 32 * _log(rng, 2, 448)
    if kind == "quantize":
        return dict(kind=kind, fmt=fmt, rows=_log(rng, 1, 16384), cols=cols)
    if kind == "norm":
        return dict(kind=kind, fmt=fmt, rows=_log(rng, 1, 16384), cols=32 * _log(rng, 2, 256),
                    add=rng.random() < 0.6, unit=rng.random() < 0.3)
    if kind == "act":
        return dict(kind=kind, fmt=fmt, act=rng.choice(("silu", "gelu_tanh", "gelu")),
                    rows=_log(rng, 1, 4096), cols=cols)
    return dict(kind=kind, fmt=fmt, tokens=rng.choice((1, _log(rng, 1, 128), _log(rng, 1, 2048))),
                rows=_log(rng, 16, 28672), cols=cols)


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 300)


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= top:
            return c


def _held(fmt, rows, cols):
    """Bytes of rows in a format, scales included."""
    return rows * (cols // (2 if fmt == FP4 else 1) + cols // 32)


def work(case):
    k, fmt, rows, cols = (case[x] for x in ("kind", "fmt", "rows", "cols"))
    if k == "product":
        t = case["tokens"]
        return {"bytes": _held(fmt, t, cols) + _held(FP4, rows, cols) + 4 * t * rows,
                "flops": 2 * t * rows * cols}
    n = rows * cols
    read = {"quantize": 4 * n, "norm": 4 * n + 4 * cols, "act": 8 * n}[k]
    if k == "norm" and case["add"]:
        read += 8 * n              # the other term, and the sum written
    back = 4 * n if fmt == FP4 else 0                   # 4-bit rows are read back as values
    ops = {"quantize": 4, "norm": 8, "act": 12}[k]
    return {"bytes": read + _held(fmt, rows, cols) + back, "flops": ops * n}


# -------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 77)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(g, rows, cols):
    """Activations: a spread of sizes from channel to channel, a few of them large."""
    size = torch.exp(0.5 * _randn(g, cols))
    size[torch.randint(0, cols, (max(1, cols // 256),), generator=g, device="cuda")] *= 30
    return _randn(g, rows, cols).mul_(size)


def prepare(case, seed):
    g, k, fmt, rows, cols = _gen(seed), *(case[x] for x in ("kind", "fmt", "rows", "cols"))
    s = {"case": case}
    if k == "product":
        t = case["tokens"]
        s["codes"], s["scales"] = _stored(*_quantised(_rows(g, t, cols), fmt), fmt)
        w = _randn(g, rows, cols).mul_(cols ** -0.5)
        s["w_codes"], s["w_scales"] = _stored(*_quantised(w, FP4), FP4)
        s["y"] = torch.zeros(t, rows, device="cuda")
        return s
    if k == "act":
        s["both"] = _randn(g, rows, 2 * cols).mul_(2)
    else:
        s["x"] = _rows(g, rows, cols)
    if k == "norm":
        s["w"] = _randn(g, cols).mul_(0.1).add_(0 if case["unit"] else 1)
        if case["add"]:
            s["d"] = _rows(g, rows, cols)
            s["x_out"] = torch.zeros_like(s["x"])
    held = (rows, cols // 2) if fmt == FP4 else (rows, cols)
    s["codes"] = torch.zeros(held, dtype=torch.uint8 if fmt == FP4 else torch.int8, device="cuda")
    s["scales"] = torch.zeros((rows, cols // 32), dtype=torch.uint8, device="cuda")
    if fmt == FP4:
        s["values"] = torch.zeros((rows, cols), device="cuda")
    return s


# ------------------------------------------------------------- the plain form
def _pow2(e):
    """2^e in 64 bits, e whole."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantised(h, fmt):
    """(whole codes of 8 bits or the values of 4-bit ones, scale bytes) of fp32 rows."""
    low, top, mantissa = _TOP[fmt]
    h = h.reshape(h.shape[0], -1, 32)
    bits = h.abs().amax(-1).view(torch.int32)
    k = bits >> 23
    s = (k - top + ((bits & 0x7FFFFF) > mantissa)).clamp(low, 254)
    s = torch.where(torch.isfinite(h).all(-1), s, torch.full_like(s, 255))
    q = h.double() * _pow2(127 - s)[..., None]
    q = torch.where((s == 255)[..., None], torch.zeros_like(q), q)
    if fmt == INT8:
        return torch.round(q * 64).clamp(-127, 127), s.to(torch.uint8)
    a = q.abs()
    r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a),
                                                               torch.round(a / 2) * 2))
    return torch.copysign(r.clamp(max=6), q), s.to(torch.uint8)


def _stored(q, s, fmt):
    """Codes as they lie in memory."""
    if fmt == INT8:
        return q.to(torch.int8).flatten(1), s
    a = q.abs()
    c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    c = (c | (torch.signbit(q).to(torch.uint8) << 3)).flatten(1)
    return c[:, 0::2] | (c[:, 1::2] << 4), s


def _values(codes, s, fmt):
    """fp32 rows of what codes and scales stand for."""
    if fmt == FP4:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).to(torch.int32)
        m = c & 7
        v = torch.where(m < 4, m, torch.where(m < 6, 2 * m - 4, 4 * m - 16)).float() * 0.5
        v = torch.where(c > 7, -v, v)
    else:
        v = codes.float() / 64
    scale = _pow2(s.int() - 127).float()
    scale = torch.where(s == 255, torch.full_like(scale, math.nan), scale)
    return (v.reshape(*s.shape, 32) * scale[..., None]).flatten(1)


def _product(s):
    x = _values(s["codes"], s["scales"], s["case"]["fmt"])
    return x @ _values(s["w_codes"], s["w_scales"], FP4).t()


def _act64(v, kind):
    if kind == "silu":
        return v / (1 + torch.exp(-v))
    if kind == "gelu_tanh":
        return v / (1 + torch.exp(-2 * 0.7978845608028654 * (v + 0.044715 * v * v * v)))
    a = (v * 0.7071067811865476).abs()
    t = 1 / (1 + 0.3275911 * a)
    p = ((((1.061405429 * t - 1.453152027) * t + 1.421413741) * t - 0.284496736) * t
         + 0.254829592) * t
    p = p * torch.exp(-a * a)
    return 0.5 * v * torch.where(v < 0, p, 2 - p)


def _plain(s):
    c = s["case"]
    outs = ()
    if c["kind"] == "product":
        return _product(s)
    if c["kind"] == "quantize":
        h = s["x"]
    elif c["kind"] == "norm":
        h = s["x"]
        if c["add"]:
            h = h + s["d"]
            outs = (h,)
        v = h.double()
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
        h = (v * (s["w"].double() + (1 if c["unit"] else 0))).float()
    else:
        gate, up = s["both"].double().chunk(2, -1)
        h = (_act64(gate, c["act"]) * up).float()
    q, scales = _quantised(h, c["fmt"])
    if c["fmt"] == FP4:
        return (*outs, (q * _pow2(scales.int() - 127)[..., None]).float().flatten(1))
    return (*outs, q.to(torch.int8).flatten(1), scales.view(torch.float8_e8m0fnu))


# -------------------------------------------------------- the framework's calls
def _handles(s):
    """What a program holds beside its buffers: arrays over them, the weights laid
    out for the product and, for single tokens, the recorded step."""
    from aero_amd import mx, ops
    from aero_amd.device import DeviceArray, Plan

    def array(t):
        kind = {torch.float32: np.float32, torch.int8: np.int8, torch.uint8: np.uint8}[t.dtype]
        return DeviceArray(tuple(t.shape), kind, _ptr=t.data_ptr(), _owner=False, _base=t)

    c = s["case"]
    a = {x: array(t) for x, t in s.items() if isinstance(t, torch.Tensor)}
    fmt, rows, cols = c["fmt"], c["rows"], c["cols"]
    if c["kind"] == "product":
        weight = mx.MxWeight(a["w_codes"], a["w_scales"], rows, cols)

    def step():
        if c["kind"] == "product":
            ops.mx_matmul(fmt, a["codes"], a["scales"], weight, a["y"], c["tokens"])
            return
        if c["kind"] == "quantize":
            ops.mx_quantize(fmt, a["x"], a["codes"], a["scales"], rows, cols)
        elif c["kind"] == "norm":
            ops.rmsnorm_mx(fmt, a["x"], a["w"], a["codes"], a["scales"], rows, cols, EPS,
                           unit_offset=c["unit"], d=a.get("d"), x_out=a.get("x_out"))
        else:
            ops.act_mul_mx(fmt, c["act"], a["both"], a["both"].view(offset_bytes=4 * cols,
                           shape=2 * rows * cols - cols), a["codes"], a["scales"], rows, cols,
                           ld=2 * cols)
        if fmt == FP4:
            ops.mx_dequant(fmt, a["codes"], a["scales"], a["values"], rows, cols)

    if (c["tokens"] if c["kind"] == "product" else rows) == 1:   # a step that is replayed
        plan = Plan()
        with plan:
            step()
        return plan.launch
    return step


def _call(s):
    if "step" not in s:
        s["step"] = _handles(s)
    s["step"]()
    if s["case"]["kind"] == "product":
        return s["y"]
    outs = (s["x_out"],) if "x_out" in s else ()
    if s["case"]["fmt"] == FP4:
        return (*outs, s["values"])
    return (*outs, s["codes"], s["scales"].view(torch.float8_e8m0fnu))


def run(s):
    return _call(s) if own else _plain(s)


# ------------------------------------------------------------- in 64 bits
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_rows(h, fmt):
    """(codes, scales) as values in 64 bits of rows in 64 bits that are fp32 numbers."""
    h = h.reshape(h.shape[0], -1, 32)
    m, e = torch.frexp(h.abs().amax(-1))
    if fmt == INT8:
        e = torch.where(m > 127 / 128, e, e - 1).clamp(min=4 - 127)
    else:
        e = torch.where(m > 0.75, e - 2, e - 3).clamp(min=-127)
    e = torch.where(m == 0, torch.full_like(e, (4 if fmt == INT8 else 0) - 127), e)
    q = torch.ldexp(h, -e[..., None])
    if fmt == INT8:
        n = torch.floor(q * 64)
        over = q * 64 - n
        n = n + ((over > 0.5) | ((over == 0.5) & (torch.remainder(n, 2) == 1)))
        return n, torch.ldexp(torch.ones_like(h[..., 0]), e)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=h.device)
    a, r = q.abs(), torch.zeros_like(q)
    for i in range(7):               # past the middle of two grid values, or at it to an even code
        middle = (grid[i] + grid[i + 1]) / 2
        r = torch.where((a > middle) | ((a == middle) & (i % 2 == 1)), grid[i + 1], r)
    return torch.where(q < 0, -r, r), torch.ldexp(torch.ones_like(h[..., 0]), e)


def exact(case, seed):
    s, k, fmt = prepare(case, seed), case["kind"], case["fmt"]
    if k == "product":
        def wide(codes, scales, f):
            if f == FP4:
                grid = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float64,
                                    device="cuda")
                codes = torch.cat([grid[(codes % 16).long()][..., None],
                                   grid[(codes // 16).long()][..., None]], -1).flatten(1)
            else:
                codes = codes.double() / 64
            e = scales.int()[..., None] - 127
            return torch.ldexp(codes.reshape(*scales.shape, 32), e).flatten(1)

        x = wide(s["codes"], s["scales"], fmt)
        return torch.cat([torch.mm(x, wide(s["w_codes"][i:i + 4096], s["w_scales"][i:i + 4096],
                                           FP4).t()) for i in range(0, case["rows"], 4096)], 1)
    outs, parts, step = [], [], max(1, (1 << 25) // case["cols"])
    for i in range(0, case["rows"], step):
        if k == "act":
            gate, up = s["both"][i:i + step].double().split(case["cols"], 1)
            if case["act"] == "silu":
                h = gate * torch.sigmoid(gate) * up
            elif case["act"] == "gelu_tanh":
                z = math.sqrt(2 / math.pi) * gate * (1 + 0.044715 * gate * gate)
                h = gate * torch.sigmoid(2 * z) * up
            else:
                z = gate.abs() * math.sqrt(0.5)
                t = torch.reciprocal(1 + 0.3275911 * z)
                tail = torch.zeros_like(t)
                for c in (1.061405429, -1.453152027, 1.421413741, -0.284496736, 0.254829592):
                    tail = (tail + c) * t
                tail = tail * torch.exp(-z * z)
                h = torch.where(gate > 0, gate - gate * tail / 2, gate * tail / 2) * up
        else:
            h = s["x"][i:i + step].double()
            if "d" in s:
                h = (h + s["d"][i:i + step].double()).float().double()
                outs.append(h)
            if k == "norm":
                w = s["w"].double() + (1.0 if case["unit"] else 0.0)
                h = h / torch.sqrt(torch.sum(h ** 2, 1, keepdim=True) / case["cols"] + EPS) * w
        q, scale = _exact_rows(h.float().double(), fmt)
        parts.append(((q * scale[..., None]).flatten(1),) if fmt == FP4 else (q.flatten(1), scale))
    outs = (torch.cat(outs),) if outs else ()
    return (*outs, *(torch.cat(p) for p in zip(*parts)))
