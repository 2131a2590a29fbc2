"""GPU: microscaled rows (ops.mx_quantize, mx_dequant, rmsnorm_mx, act_mul_mx) and their
product with 4-bit weights (ops.mx_matmul, mx.MxWeight) against plain 64-bit forms
(tests/mx_ref.py).

Rows: codes and scales equal, the residual sums and the values read back bit for bit. The
norms and activations are 64-bit expressions rounded to fp32 once, so both sides round the
same number but where it lies within some 2^-50 of a border of two fp32 numbers.

Product: its terms are exact, each of a sum's additions rounds to fp32. A step of 64
columns adds 8 groups of 8 products and the running sum, twice for 8-bit rows (a code's
halves): 9 K / 32 additions, each off by up to 2^-23 of the running sum, which grows to
the result's size; as independent errors sqrt(9 K / 32) 2^-24 of the result, in the norm.
No element further than 2^-20 of the sum of its terms' magnitudes."""
import numpy as np
import pytest

import mx_ref as R
from conftest import bits_equal
from aero_amd import _lib, mx, ops
from aero_amd.device import DeviceArray as DA, Plan, Stream, synchronize, tune_set

pytestmark = pytest.mark.gpu

INT8, FP4 = ops.MX_INT8, ops.MX_FP4
FMTS = [INT8, FP4]


def held(fmt, rows, cols, fill=0x5A):
    codes = np.full((rows, ops.mx_row_bytes(fmt, cols)), fill, np.int8 if fmt == INT8 else np.uint8)
    return DA.from_numpy(codes), DA.from_numpy(np.full((rows, cols // 32), fill, np.uint8))


def same(dc, ds, want):
    assert np.array_equal(ds.numpy(), want[1])
    assert np.array_equal(dc.numpy(), want[0])


def awkward(rng, rows, cols):
    """Rows of many sizes with zeros, subnormals, the largest numbers, ties and blocks whose
    largest value is at, just below and just above a scale's border."""
    x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-140, 120, (rows, 1)))).astype(np.float32)
    b = x.reshape(-1, 32)
    n = len(b)
    for i in range(0, n, 3):
        kind = (i // 3) % 8
        e = np.float32(2.0) ** np.float32(rng.integers(-100, 100))
        if kind == 0:
            b[i] = 0
            b[i, 1::2] = -0.0
        elif kind == 1:
            b[i] = (rng.integers(-9, 10, 32) * 2.0 ** -149).astype(np.float32)
        elif kind == 2:
            b[i, rng.integers(32)] = np.finfo(np.float32).max
        elif kind == 3:      # every tie of 8 bits below the largest code
            b[i] = (rng.integers(-126, 126, 32) + 0.5) / 64 * e
            b[i, 0] = 127 / 64 * e
        elif kind == 4:      # and of 4 bits
            b[i] = rng.choice([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, -.25, -5.0, 6.0], 32) * e
            b[i, 0] = 6 * e
        elif kind == 5:
            b[i, 3] = np.nextafter(np.float32(np.abs(b[i]).max()) * 0 + np.float32(127 / 64) * e, np.float32(np.inf))
        elif kind == 6:
            b[i] = b[i] * 0 + np.nextafter(np.float32(6) * e, np.float32(np.inf))
        else:
            b[i] = b[i] * 0 - np.nextafter(np.float32(6) * e, np.float32(0))
    return b.reshape(rows, cols)


SIZES = [(1, 32), (3, 64), (1, 896), (37, 96), (130, 2560), (5, 14336)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantise(hip, fmt, rows, cols):
    x = awkward(np.random.default_rng(rows + cols), rows, cols)
    dc, ds = held(fmt, rows, cols)
    ops.mx_quantize(fmt, DA.from_numpy(x), dc, ds, rows, cols)
    same(dc, ds, R.quantise(x, fmt))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantise_not_finite(hip, fmt):
    x = np.random.default_rng(1).standard_normal((6, 96)).astype(np.float32)
    x[0, 5], x[1, 40], x[2, 95], x[3, 32:64] = np.nan, np.inf, -np.inf, np.nan
    dc, ds = held(fmt, 6, 96)
    ops.mx_quantize(fmt, DA.from_numpy(x), dc, ds, 6, 96)
    want = R.quantise(x, fmt)
    assert (want[1] == 255).sum() == 4
    same(dc, ds, want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("off,ld", [(0, 96), (0, 100), (1, 97), (3, 203), (2, 96)])
def test_quantise_strides_and_addresses(hip, fmt, off, ld):
    rows, cols = 19, 96
    rng = np.random.default_rng(ld)
    flat = rng.standard_normal(off + rows * ld).astype(np.float32)
    x = np.stack([flat[off + r * ld:off + r * ld + cols] for r in range(rows)])
    d = DA.from_numpy(flat[:off + (rows - 1) * ld + cols])
    dc, ds = held(fmt, rows + 1, cols)
    ops.mx_quantize(fmt, d.view(shape=d.size - off, offset_bytes=4 * off), dc, ds, rows, cols, ld=ld)
    want = R.quantise(x, fmt)
    assert np.array_equal(dc.numpy()[:rows], want[0]) and np.array_equal(ds.numpy()[:rows], want[1])
    assert (dc.numpy()[rows] == 0x5A).all() and (ds.numpy()[rows] == 0x5A).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("off", [0, 1])
def test_dequant_every_code_and_scale(hip, fmt, off):
    """Every code under every scale byte, also where the value is an fp32 subnormal, past
    the largest fp32 number (an infinity, as rounding gives) or NaN."""
    per = 256 if fmt == INT8 else 32
    codes = np.tile(np.arange(256, dtype=np.uint8).view(np.int8), (256, 1)) if fmt == INT8 else \
        np.tile(R.pack(np.arange(32)[None] % 16, FP4), (256, 1))
    s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], per // 32, 1)
    out = DA.from_numpy(np.full(256 * per + 8, 7, np.float32))
    ops.mx_dequant(fmt, DA.from_numpy(codes), DA.from_numpy(s),
                   out.view(shape=256 * per, offset_bytes=4 * off), 256, per)
    with np.errstate(over="ignore"):
        want = R.values(codes, s, fmt).astype(np.float32)
    got = out.numpy()
    body = got[off:off + 256 * per].reshape(256, per)
    assert np.array_equal(np.isnan(body), np.isnan(want))
    assert bits_equal(np.nan_to_num(body, nan=1), np.nan_to_num(want, nan=1)) or \
        np.array_equal(body[~np.isnan(body)], want[~np.isnan(want)])
    assert (got[:off] == 7).all() and (got[off + 256 * per:] == 7).all()


NORMS = [(1, 32), (1, 896), (5, 224), (333, 2560), (9, 512), (64, 4096), (3, 8192), (2, 14336),
         (3, 16384), (2, 16416), (2, 28672), (2, 32800)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("add", ["none", "x", "d", "apart"])
@pytest.mark.parametrize("rows,cols", NORMS)
def test_norm(hip, fmt, add, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal(cols))).astype(np.float32)
    d = rng.standard_normal((rows, cols)).astype(np.float32)
    unit = cols % 512 == 0
    w = None if rows == 2 else (rng.standard_normal(cols) * 0.1 + (not unit)).astype(np.float32)
    dx, dd = DA.from_numpy(x), DA.from_numpy(d)
    out = {"none": None, "x": dx, "d": dd, "apart": DA.empty((rows, cols))}[add]
    dc, ds = held(fmt, rows, cols)
    ops.rmsnorm_mx(fmt, dx, None if w is None else DA.from_numpy(w), dc, ds, rows, cols, 1e-5,
                   unit_offset=unit, d=None if add == "none" else dd, x_out=out)
    total = x if add == "none" else x + d
    same(dc, ds, R.quantise(R.norm(total, w, 1e-5, unit), fmt))
    if out is not None:
        assert bits_equal(out.numpy(), total)
    for arr, host in ((dx, x), (dd, d)):
        if arr is not out:
            assert bits_equal(arr.numpy(), host)


@pytest.mark.parametrize("fmt", FMTS)
def test_norm_awkward_rows(hip, fmt):
    """Zero rows, rows whose squares pass fp32's range, NaN and infinities; odd addresses."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((8, 160)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e30)
    x[2] *= np.float32(1e-30)
    x[3, 7] = np.inf
    x[4, 9] = np.nan
    x[5, 0] = np.float32(3e38)
    w = rng.standard_normal(160).astype(np.float32)
    want = R.quantise(R.norm(x, w, 1e-6, False), fmt)
    assert (want[1][4] == 255).all() and (want[1][3] == 255).sum() == 1
    for off in (0, 1):
        dx = DA.from_numpy(np.concatenate([np.zeros(off, np.float32), x.reshape(-1)]))
        dw = DA.from_numpy(np.concatenate([np.zeros(off, np.float32), w]))
        dc, ds = held(fmt, 8, 160)
        ops.rmsnorm_mx(fmt, dx.view(shape=1280, offset_bytes=4 * off),
                       dw.view(shape=160, offset_bytes=4 * off), dc, ds, 8, 160, 1e-6)
        same(dc, ds, want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "identity", "sigmoid"])
@pytest.mark.parametrize("rows,cols,layout", [(1, 4864, "halves"), (33, 96, "halves"), (7, 320, "own"),
                                              (5, 64, "odd"), (130, 1024, "own")])
def test_act(hip, fmt, kind, rows, cols, layout):
    rng = np.random.default_rng(cols)
    g, u = ((rng.standard_normal((rows, cols)) * 3).astype(np.float32) for _ in range(2))
    g[0, :32] = np.linspace(-200, 200, 32)
    g[0, 32:64] = -30 - np.arange(32)                 # a block of tails only
    with np.errstate(over="ignore"):
        want = R.quantise((R.act(kind, g) * u).astype(np.float32), fmt)
    dc, ds = held(fmt, rows, cols)
    if layout == "own":
        ops.act_mul_mx(fmt, kind, DA.from_numpy(g), DA.from_numpy(u), dc, ds, rows, cols)
    else:
        gap = 0 if layout == "halves" else 3
        both = DA.from_numpy(np.concatenate([g, u, np.full((rows, gap), np.nan, np.float32)], 1))
        ld = 2 * cols + gap
        ops.act_mul_mx(fmt, kind, both, both.view(shape=both.size - cols, offset_bytes=4 * cols), dc,
                       ds, rows, cols, ld=ld)
    same(dc, ds, want)
    if kind != "identity":
        ops.act_mul_mx(fmt, kind, DA.from_numpy(g), None, dc, ds, rows, cols)
        with np.errstate(over="ignore"):
            same(dc, ds, R.quantise(R.act(kind, g).astype(np.float32), fmt))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "sigmoid"])
def test_act_next_to_borders(hip, fmt, kind):
    """Values that lie within a few fp32 steps of a border between two codes, or of the scale:
    `up` is such a border over the activation, moved by up to 40 steps either way. Tails, tiny
    blocks and zeros too."""
    rng = np.random.default_rng(21)
    rows, cols = 64, 1024
    g = (rng.standard_normal((rows, cols)) * 4).astype(np.float32)
    a = R.act(kind, g)
    if fmt == INT8:
        border = (rng.integers(-126, 126, (rows, cols)) + 0.5) / 64
    else:
        border = rng.choice([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0], (rows, cols))
    border[:, ::32] = R.TOP[fmt]
    border *= np.exp2(np.repeat(rng.integers(-90, 90, (rows, cols // 32)), 32, 1))
    border[-8:] *= 2.0 ** -140
    u = border / np.where(a == 0, 1, a) * (1 + rng.integers(-40, 41, (rows, cols)) * 2.0 ** -24)
    u = np.clip(u, -3e38, 3e38).astype(np.float32)
    u[5], u[6, ::2] = 0, -0.0
    g[7] = np.float32(-90)
    with np.errstate(over="ignore", under="ignore"):
        want = R.quantise((R.act(kind, g) * u).astype(np.float32), fmt)
    dc, ds = held(fmt, rows, cols)
    ops.act_mul_mx(fmt, kind, DA.from_numpy(g), DA.from_numpy(u), dc, ds, rows, cols)
    same(dc, ds, want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", "sigmoid"])
def test_act_of_subnormals_times_large(hip, fmt, kind):
    """act(gate) below fp32's normal numbers, of which fp32 would keep a few bits or none,
    brought back by `up`."""
    rng = np.random.default_rng(22)
    rows, cols = 16, 256
    g = (rng.integers(-9, 10, (rows, cols)) * 2.0 ** -149).astype(np.float32)
    g[4:8] = (rng.standard_normal((4, cols)) * 2.0 ** -130).astype(np.float32)
    g[8:12, ::3] = (rng.standard_normal((4, 86)) * 2.0 ** -110).astype(np.float32)
    g[12:] = np.where(rng.random((4, cols)) < .03, np.float32(2.0 ** -149), np.float32(0))
    u = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(20, 120, (rows, 1)))).astype(np.float32)
    want = R.quantise((R.act(kind, g) * u).astype(np.float32), fmt)
    dc, ds = held(fmt, rows, cols)
    ops.act_mul_mx(fmt, kind, DA.from_numpy(g), DA.from_numpy(u), dc, ds, rows, cols)
    same(dc, ds, want)


def test_act_not_finite(hip):
    g = np.random.default_rng(2).standard_normal((4, 64)).astype(np.float32)
    u = np.ones_like(g)
    g[0, 3], g[1, 40], u[2, 5], u[3, 60] = np.nan, np.inf, np.nan, np.float32(3e38)
    g[3, 60] = 100                                     # 3e40: past fp32
    dc, ds = held(INT8, 4, 64)
    ops.act_mul_mx(INT8, "silu", DA.from_numpy(g), DA.from_numpy(u), dc, ds, 4, 64)
    with np.errstate(over="ignore", invalid="ignore"):
        want = R.quantise((R.act("silu", g) * u).astype(np.float32), INT8)
    assert (want[1] == 255).sum() == 4
    same(dc, ds, want)


# ------------------------------------------------------------------ product
def operands(rng, fmt, T, N, K, spread=0):
    """(x codes, x scales, W codes, W scales) of rows of different sizes."""
    x = rng.standard_normal((T, K)) * np.exp2(rng.integers(-spread, spread + 1, (T, 1)))
    x[:, ::97] *= 20
    w = rng.standard_normal((N, K)) * 0.02
    return (*R.quantise(x.astype(np.float32), fmt), *R.quantise(w.astype(np.float32), FP4))


def product(fmt, xc, xs, wc, ws, stream=None, guard=64):
    T, N, K = xc.shape[0], wc.shape[0], 32 * xs.shape[1]
    weight = mx.MxWeight(DA.from_numpy(wc), DA.from_numpy(ws), N, K)
    y = DA.from_numpy(np.full(T * N + guard, 7.0, np.float32))
    ops.mx_matmul(fmt, DA.from_numpy(xc), DA.from_numpy(xs), weight, y, T, stream=stream)
    synchronize()
    y = y.numpy()
    assert (y[T * N:] == 7).all()
    return y[:T * N].reshape(T, N)


def near(got, xc, xs, wc, ws, fmt):
    K = 32 * xs.shape[1]
    x, w = R.values(xc, xs, fmt), R.values(wc, ws, FP4)
    want = x @ w.T
    assert (np.abs(got - want) <= 2.0 ** -20 * (np.abs(x) @ np.abs(w).T) + 2.0 ** -149).all()
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= np.sqrt(9 * K / 32) * 2.0 ** -24, off


PRODUCTS = [(1, 1, 32), (1, 9728, 896), (1, 100, 64), (2, 33, 96), (3, 4096, 160), (5, 50, 992),
            (16, 257, 512), (17, 31, 2560), (31, 64, 128), (32, 96, 4096), (33, 130, 224),
            (64, 1000, 1024), (65, 129, 352), (100, 3, 4864), (127, 255, 736), (128, 256, 256),
            (129, 257, 288), (200, 513, 1056), (256, 512, 2048), (300, 1021, 928), (512, 640, 4096),
            (513, 300, 544), (1000, 100, 1120), (9, 12300, 160),
            (20, 12290, 96), (24, 6200, 1760), (18, 20490, 64)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,N,K", PRODUCTS)
def test_product(hip, fmt, T, N, K):
    print(f"product fmt={fmt} T={T} N={N} K={K}", flush=True)
    a = operands(np.random.default_rng(T + N + K), fmt, T, N, K, spread=2)
    near(product(fmt, *a), *a, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("tiles", range(6))
@pytest.mark.parametrize("T,N,K", [(33, 300, 32), (97, 261, 96), (130, 270, 160), (300, 513, 1632)])
def test_product_on_every_tile(hip, fmt, tiles, T, N, K):
    """Each size of tile, with one stage, fewer stages than buffers and more."""
    print(f"product fmt={fmt} tiles={tiles} T={T} N={N} K={K}", flush=True)
    a = operands(np.random.default_rng(tiles + T), fmt, T, N, K, spread=2)
    tune_set("mx_tiles", tiles)
    try:
        near(product(fmt, *a), *a, fmt)
    finally:
        tune_set("mx_tiles", None)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T", [1, 40, 200])
def test_product_any_codes_and_scales(hip, fmt, T):
    """Random bytes for codes (-128 and both zeros among them), scales over 40 binades."""
    rng = np.random.default_rng(T)
    N, K = 70, 480
    xc = rng.integers(0, 256, (T, ops.mx_row_bytes(fmt, K))).astype(np.uint8)
    xc = xc.view(np.int8) if fmt == INT8 else xc
    xs, ws = (rng.integers(107, 147, (n, K // 32)).astype(np.uint8) for n in (T, N))
    wc = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
    got = product(fmt, xc, xs, wc, ws)
    x, w = R.values(xc, xs, fmt), R.values(wc, ws, FP4)
    assert (np.abs(got - x @ w.T) <= 2.0 ** -20 * (np.abs(x) @ np.abs(w).T)).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T", [3, 140])
def test_product_of_not_finite_blocks(hip, fmt, T):
    """A NaN block makes its token's, or its weight row's, results NaN and no others; scales
    at both ends of their range meet."""
    rng = np.random.default_rng(9)
    N, K = 40, 224
    xc, xs, wc, ws = operands(rng, fmt, T, N, K)
    xs[1, 3], ws[7, 6] = 255, 255
    got = product(fmt, xc, xs, wc, ws)
    nan = np.isnan(got)
    assert nan[1].all() and nan[:, 7].all()
    keep = np.ones((T, N), bool)
    keep[1], keep[:, 7] = False, False
    assert not nan[keep].any()
    xs[1, 3], ws[7, 6] = 127, 127
    xs[:], ws[:] = 250, 4      # 2^123 * 2^-123
    got = product(fmt, xc, xs, wc, ws)
    x, w = R.values(xc, xs, fmt), R.values(wc, ws, FP4)
    assert (np.abs(got - x @ w.T) <= 2.0 ** -20 * (np.abs(x) @ np.abs(w).T)).all()


def test_product_of_nothing(hip):
    w = mx.MxWeight.from_rows(DA.from_numpy(np.ones((4, 32), np.float32)), 4, 32)
    y = DA.from_numpy(np.full(4, 7, np.float32))
    ops.mx_matmul(INT8, *held(INT8, 1, 32), w, y, 0)
    assert (y.numpy() == 7).all()


def test_product_rows_at_odd_addresses(hip):
    """y anywhere on 4 bytes."""
    rng = np.random.default_rng(4)
    for T in (2, 130):
        a = operands(rng, INT8, T, 64, 256)
        w = mx.MxWeight(DA.from_numpy(a[2]), DA.from_numpy(a[3]), 64, 256)
        flat = DA.from_numpy(np.full(T * 64 + 9, 7, np.float32))
        ops.mx_matmul(INT8, DA.from_numpy(a[0]), DA.from_numpy(a[1]), w,
                      flat.view(shape=T * 64, offset_bytes=4), T)
        got = flat.numpy()
        near(got[1:1 + T * 64].reshape(T, 64), *a, INT8)
        assert got[0] == 7 and (got[1 + T * 64:] == 7).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_same_call_same_bits(hip, fmt):
    """The same call twice: the same bits."""
    a = operands(np.random.default_rng(8), fmt, 150, 300, 1056)
    assert bits_equal(product(fmt, *a), product(fmt, *a))


# ------------------------------------------------------------ as they are used
def test_feed_forward_in_a_plan(hip):
    """Residual and norm to 8 bits, gate and up in one product, the activation to 8 bits, the
    down projection, recorded once and replayed on new inputs on a stream; each step against
    its formula on the inputs that it had."""
    rng = np.random.default_rng(11)
    T, C, F = 70, 256, 416
    wg, wd = ((rng.standard_normal((n, k)) * k ** -0.5).astype(np.float32)
              for n, k in ((2 * F, C), (C, F)))
    nw = rng.standard_normal(C).astype(np.float32)
    w1 = mx.MxWeight.from_rows(DA.from_numpy(wg), 2 * F, C)
    w2 = mx.MxWeight.from_rows(DA.from_numpy(wd), C, F)
    x, d, y = DA.empty((T, C)), DA.empty((T, C)), DA.empty((T, C))
    both, dw = DA.empty((T, 2 * F)), DA.from_numpy(nw)
    hc, hs = held(INT8, T, C)
    ac, as_ = held(INT8, T, F)
    up = both.view(shape=both.size - F, offset_bytes=4 * F)
    plan = Plan()
    with plan:
        ops.rmsnorm_mx(INT8, x, dw, hc, hs, T, C, 1e-5, d=d)
        ops.mx_matmul(INT8, hc, hs, w1, both, T)
        ops.act_mul_mx(INT8, "silu", both, up, ac, as_, T, F, ld=2 * F)
        ops.mx_matmul(INT8, ac, as_, w2, y, T)
    stream = Stream()
    for step in range(3):
        hx, hd = (rng.standard_normal((T, C)).astype(np.float32) * (step + 1) for _ in range(2))
        x.copy_from(hx)
        d.copy_from(hd)
        plan.launch(stream)
        stream.synchronize()
        assert bits_equal(x.numpy(), hx + hd)
        same(hc, hs, R.quantise(R.norm(hx + hd, nw, 1e-5, False), INT8))
        near(both.numpy(), hc.numpy(), hs.numpy(), *R.quantise(wg, FP4), INT8)
        g, u = both.numpy()[:, :F], both.numpy()[:, F:]
        same(ac, as_, R.quantise((R.act("silu", g) * u).astype(np.float32), INT8))
        near(y.numpy(), ac.numpy(), as_.numpy(), *R.quantise(wd, FP4), INT8)
    stream.destroy()


def test_on_a_stream_of_its_own(hip):
    """Every op on another stream than the null one, in order behind one another."""
    rng = np.random.default_rng(15)
    T, C, N = 40, 288, 70
    x, d = (rng.standard_normal((T, C)).astype(np.float32) for _ in range(2))
    wr = rng.standard_normal((N, C)).astype(np.float32)
    weight = mx.MxWeight.from_rows(DA.from_numpy(wr), N, C)
    dx, dd, y, back = DA.from_numpy(x), DA.from_numpy(d), DA.empty((T, N)), DA.empty((T, C))
    c, s = held(INT8, T, C)
    q, qs = held(FP4, T, C)
    a, as_ = held(INT8, T, C)
    stream = Stream()
    ops.rmsnorm_mx(INT8, dx, None, c, s, T, C, 1e-5, d=dd, stream=stream)
    ops.mx_matmul(INT8, c, s, weight, y, T, stream=stream)
    ops.mx_dequant(INT8, c, s, back, T, C, stream=stream)
    ops.mx_quantize(FP4, back, q, qs, T, C, stream=stream)
    ops.act_mul_mx(INT8, "silu", back, dx, a, as_, T, C, stream=stream)
    stream.synchronize()
    stream.destroy()
    want = R.quantise(R.norm(x + d, None, 1e-5, False), INT8)
    same(c, s, want)
    near(y.numpy(), *want, *R.quantise(wr, FP4), INT8)
    values = R.values(*want, INT8).astype(np.float32)
    assert bits_equal(back.numpy(), values)
    same(q, qs, R.quantise(values, FP4))
    same(a, as_, R.quantise((R.act("silu", values) * (x + d)).astype(np.float32), INT8))


def test_weights_are_not_laid_out_in_a_plan(hip):
    codes, scales = held(FP4, 4, 32)
    x = DA.from_numpy(np.ones((4, 32), np.float32))
    plan = Plan()
    with plan:
        with pytest.raises(RuntimeError):
            mx.MxWeight(codes, scales, 4, 32)
        with pytest.raises(RuntimeError):
            mx.MxWeight.from_rows(x, 4, 32)
    assert len(plan) == 0


def test_plan_holds_the_weights(hip):
    """The weights of a recorded product stay while the plan does."""
    a = operands(np.random.default_rng(14), INT8, 3, 64, 128)
    weight = mx.MxWeight(DA.from_numpy(a[2]), DA.from_numpy(a[3]), 64, 128)
    xc, xs, y = DA.from_numpy(a[0]), DA.from_numpy(a[1]), DA.empty((3, 64))
    plan = Plan()
    with plan:
        ops.mx_matmul(INT8, xc, xs, weight, y, 3)
    del weight
    others = [DA.from_numpy(np.full(64 * 128, 255, np.uint8)) for _ in range(8)]
    plan.launch()
    synchronize()
    near(y.numpy(), *a, INT8)
    del others


def test_plan_keeps_its_workspace(hip):
    """A plan recorded before a larger call has its own workspace, and gives the same bits."""
    a = operands(np.random.default_rng(12), INT8, 130, 200, 512)
    weight = mx.MxWeight(DA.from_numpy(a[2]), DA.from_numpy(a[3]), 200, 512)
    xc, xs, y = DA.from_numpy(a[0]), DA.from_numpy(a[1]), DA.empty((130, 200))
    plan = Plan()
    with plan:
        ops.mx_matmul(INT8, xc, xs, weight, y, 130)
    plan.launch()
    synchronize()
    first = y.numpy()
    near(first, *a, INT8)
    b = operands(np.random.default_rng(13), INT8, 700, 64, 4096)
    near(product(INT8, *b), *b, INT8)
    for _ in range(2):
        y.copy_from(np.zeros((130, 200), np.float32))
        plan.launch()
        synchronize()
        assert bits_equal(y.numpy(), first)


# ------------------------------------------- products at the ends of fp32's range
def whole(rng, fmt, T, N, K, unit):
    """Random codes whose scales make every product a whole number of 2^unit: (operands,
    sums in those units). The sums stay below 2^24, so that every partial sum is exact in
    fp32 wherever 2^unit and the result are in its range, subnormal or not."""
    xc = rng.integers(0, 256, (T, ops.mx_row_bytes(fmt, K))).astype(np.uint8)
    xc = xc.view(np.int8) if fmt == INT8 else xc
    wc = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
    one = np.full((T, K // 32), 127, np.uint8), np.full((N, K // 32), 127, np.uint8)
    low = 2.0 ** (-7 if fmt == INT8 else -2)          # 1/64 or 1/2, times 1/2
    x, w = R.values(xc, one[0], fmt), R.values(wc, one[1], FP4)
    sums = (x @ w.T) / low
    assert (np.abs(x) @ np.abs(w).T / low < 2 ** 24).all()
    total = 254 + unit + (7 if fmt == INT8 else 2)    # of the two scale bytes
    return xc, wc, sums, total


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,tiles", [(1, None), (13, None), (20, None), (32, None)] +
                         [(40, k) for k in range(6)])
@pytest.mark.parametrize("unit,x_scale", [(-149, 4), (-149, 60), (-149, 100), (-143, 30), (-135, 50),
                                          (100, 247), (100, 248), (100, 249), (100, 254),
                                          (0, 249), (20, 254)])
def test_product_at_the_ends_of_the_range(hip, fmt, T, tiles, unit, x_scale):
    """Sums of whole numbers of 2^unit come out exact down to fp32's last subnormal bit and
    up to the largest scales, alike for every number of tokens."""
    print(f"ends fmt={fmt} T={T} tiles={tiles} unit={unit} x_scale={x_scale}", flush=True)
    N, K = 70, 352
    rng = np.random.default_rng(T + x_scale)
    xc, wc, sums, total = whole(rng, fmt, T, N, K, unit)
    xs, ws = np.full((T, K // 32), x_scale, np.uint8), np.full((N, K // 32), total - x_scale, np.uint8)
    assert 0 <= total - x_scale <= 254
    tune_set("mx_tiles", tiles)
    try:
        got = product(fmt, xc, xs, wc, ws)
    finally:
        tune_set("mx_tiles", None)
    assert bits_equal(got + np.float32(0), (sums * 2.0 ** unit).astype(np.float32) + np.float32(0))


@pytest.mark.parametrize("T,tiles", [(1, None), (13, None), (32, None)] + [(40, k) for k in range(6)])
def test_product_of_scales_far_apart(hip, T, tiles):
    """Blocks of one token at both ends of the scales, tokens that are NaN, tiny or large
    beside each other: 8-bit rows whose every block has a scale of its own."""
    print(f"far apart T={T} tiles={tiles}", flush=True)
    N, K = 40, 416
    rng = np.random.default_rng(T)
    xc = rng.integers(-128, 128, (T, K)).astype(np.int8)
    xs = rng.choice(np.array([4, 5, 120, 247, 248, 249, 252, 254], np.uint8), (T, K // 32))
    wc = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
    ws = rng.integers(0, 110, (N, K // 32)).astype(np.uint8)
    xs[T // 2, 7] = 255
    tune_set("mx_tiles", tiles)
    try:
        got = product(INT8, xc, xs, wc, ws)
    finally:
        tune_set("mx_tiles", None)
    ok = np.arange(T) != T // 2
    assert np.isnan(got[T // 2]).all() and not np.isnan(got[ok]).any()
    x, w = R.values(xc, xs, INT8)[ok], R.values(wc, ws, FP4)
    # the terms' own bound, and half a last bit for each addition of what is subnormal
    room = 2.0 ** -20 * (np.abs(x) @ np.abs(w).T) + 9 * K / 32 * 2.0 ** -150
    assert (np.abs(got[ok] - x @ w.T) <= room).all()


# ------------------------------------------------ every tile as calls come to it
def tiles_of(fmt, T, N, K):
    return _lib.lib().aero_hip_mx_matmul_tiles(fmt, N, K, T)


@pytest.mark.parametrize("fmt,tiles,T,N,K", [
    (INT8, 0, 1859, 9163, 704), (INT8, 0, 2047, 6003, 1056), (INT8, 1, 525, 6207, 3680),
    (INT8, 1, 263, 7397, 288), (INT8, 2, 835, 1637, 1376), (INT8, 4, 259, 3401, 4704),
    (INT8, 3, 1031, 897, 1984), (INT8, 4, 707, 815, 2880), (INT8, 4, 35, 9321, 672),
    (INT8, 4, 141, 4219, 2112), (FP4, 0, 2139, 9101, 1184), (FP4, 0, 2137, 2339, 2400),
    (FP4, 1, 453, 6511, 960), (FP4, 2, 131, 10657, 2496), (FP4, 3, 181, 3149, 4032),
    (FP4, 3, 33, 8393, 992), (FP4, 4, 65, 8653, 1984), (FP4, 5, 577, 3363, 6080)])
def test_product_on_the_tiles_of_its_size(hip, fmt, tiles, T, N, K):
    """Sizes that the rule itself sends to each size of tile: more workgroups than run at a
    time, more token tiles than lie side by side, long and ragged sums."""
    print(f"product fmt={fmt} tiles={tiles} T={T} N={N} K={K}", flush=True)
    assert tiles_of(fmt, T, N, K) == tiles
    a = operands(np.random.default_rng(T + N + K), fmt, T, N, K, spread=2)
    near(product(fmt, *a), *a, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("tiles", range(6))
@pytest.mark.parametrize("T,N,K", [(645, 265, 4128), (673, 530, 4256)])
def test_long_sums_on_every_tile(hip, fmt, tiles, T, N, K):
    print(f"long fmt={fmt} tiles={tiles} T={T} N={N} K={K}", flush=True)
    a = operands(np.random.default_rng(tiles + T), fmt, T, N, K, spread=2)
    tune_set("mx_tiles", tiles)
    try:
        near(product(fmt, *a), *a, fmt)
    finally:
        tune_set("mx_tiles", None)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("tiles", range(6))
def test_any_codes_on_every_tile(hip, fmt, tiles):
    """Random bytes for codes and scales, and NaN blocks: their token's, and their weight
    row's, results are NaN and no others."""
    print(f"codes fmt={fmt} tiles={tiles}", flush=True)
    rng = np.random.default_rng(tiles)
    T, N, K = 150, 290, 608
    xc = rng.integers(0, 256, (T, ops.mx_row_bytes(fmt, K))).astype(np.uint8)
    xc = xc.view(np.int8) if fmt == INT8 else xc
    xs, ws = (rng.integers(107, 147, (n, K // 32)).astype(np.uint8) for n in (T, N))
    wc = rng.integers(0, 256, (N, K // 2)).astype(np.uint8)
    xs[1, 3], xs[149, 18], ws[7, 6], ws[289, 0] = 255, 255, 255, 255
    tune_set("mx_tiles", tiles)
    try:
        got = product(fmt, xc, xs, wc, ws)
    finally:
        tune_set("mx_tiles", None)
    nan = np.zeros((T, N), bool)
    nan[[1, 149]], nan[:, [7, 289]] = True, True
    assert np.array_equal(np.isnan(got), nan)
    x, w = (np.nan_to_num(R.values(*a)) for a in ((xc, xs, fmt), (wc, ws, FP4)))
    ok = ~nan
    assert (np.abs(got - x @ w.T)[ok] <= (2.0 ** -20 * (np.abs(x) @ np.abs(w).T))[ok]).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_dequant_bit_for_bit(hip, fmt):
    """Every code under every scale byte, the sign of zeros too."""
    per = 256 if fmt == INT8 else 32
    codes = np.tile(np.arange(256, dtype=np.uint8).view(np.int8), (256, 1)) if fmt == INT8 else \
        np.tile(R.pack(np.arange(32)[None] % 16, FP4), (256, 1))
    s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], per // 32, 1)
    out = DA.empty((256, per))
    ops.mx_dequant(fmt, DA.from_numpy(codes), DA.from_numpy(s), out, 256, per)
    with np.errstate(over="ignore"):
        want = R.values(codes, s, fmt).astype(np.float32)
    got = out.numpy()
    assert np.isnan(got[255]).all() and not np.isnan(got[:255]).any()
    assert bits_equal(got[:255], want[:255])


@pytest.mark.parametrize("fmt", FMTS)
def test_norm_of_more_rows_than_a_launch_takes(hip, fmt):
    """2^26 + 3 rows of 32 values, 2^32 lanes and more: rows on both sides of what one launch
    takes, and the last."""
    rows, cols = (1 << 26) + 3, 32
    x = DA.empty((rows, cols))
    ops.fill_f32(x, 1.0)
    codes = DA.empty((rows, ops.mx_row_bytes(fmt, cols)), np.int8 if fmt == INT8 else np.uint8)
    scales = DA.empty((rows, 1), np.uint8)
    rng = np.random.default_rng(3)
    at = [0, (1 << 25) - 2, rows - 4]          # four rows each, none of them twice
    h = rng.standard_normal((len(at), 4, cols)).astype(np.float32)
    for r, v in zip(at, h):
        x.view(shape=(4, cols), offset_bytes=r * 4 * cols).copy_from(v)
    ops.rmsnorm_mx(fmt, x, None, codes, scales, rows, cols, 1e-5)
    synchronize()
    per = ops.mx_row_bytes(fmt, cols)
    for r, v in zip(at, h):
        same(codes.view(shape=(4, per), offset_bytes=r * per), scales.view(shape=(4, 1), offset_bytes=r),
             R.quantise(R.norm(v, None, 1e-5, False), fmt))


def test_dequant_of_more_values_than_a_launch_takes(hip):
    """2^33 values and some: 34 GB written in two launches."""
    cols = 1 << 13
    rows = (1 << 20) + 5
    codes, scales = DA.empty((rows, cols // 2), np.uint8), DA.empty((rows, cols // 32), np.uint8)
    out = DA.empty((rows, cols))
    rng = np.random.default_rng(4)
    at = [0, (1 << 20) - 2, rows - 2]
    for r in at:
        x = rng.standard_normal((2, cols)).astype(np.float32)
        c, s = R.quantise(x, FP4)
        codes.view(shape=c.shape, offset_bytes=r * c.shape[1]).copy_from(c)
        scales.view(shape=s.shape, offset_bytes=r * s.shape[1]).copy_from(s)
    ops.mx_dequant(FP4, codes, scales, out, rows, cols)
    synchronize()
    for r in at:
        c = codes.view(shape=(2, cols // 2), offset_bytes=r * (cols // 2)).numpy()
        s = scales.view(shape=(2, cols // 32), offset_bytes=r * (cols // 32)).numpy()
        got = out.view(shape=(2, cols), offset_bytes=r * 4 * cols).numpy()
        assert bits_equal(got, R.values(c, s, FP4).astype(np.float32))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,N,K", [(24, 4112, 4128), (32, 20500, 96), (17, 8230, 2080), (32, 100, 14336)])
def test_product_without_a_workspace(hip, fmt, T, N, K):
    """Calls of up to 32 tokens that the rule sends to tiles, on the few-token kernel."""
    print(f"no workspace fmt={fmt} T={T} N={N} K={K}", flush=True)
    assert 0 <= tiles_of(fmt, T, N, K) < 6 or K == 2080
    a = operands(np.random.default_rng(T + N + K), fmt, T, N, K, spread=2)
    d = [DA.from_numpy(v) for v in a]
    w = mx.MxWeight(d[2], d[3], N, K)
    y = DA.from_numpy(np.full(T * N + 64, 7.0, np.float32))
    _lib.check(_lib.lib().aero_hip_mx_matmul(fmt, d[0].ptr, d[1].ptr, w.buf.ptr, w.buf.nbytes, y.ptr, N, K, T,
                                             None, 0, None), "mx_matmul")
    synchronize()
    got = y.numpy()
    assert (got[T * N:] == 7).all()
    near(got[:T * N].reshape(T, N), *a, fmt)
