"""CPU: refusals of the microscaled ops and their host-side sizes; the plain forms that
the GPU tests compare with, on values worked out by hand."""
import numpy as np
import pytest

import mx_ref as R
from aero_amd import _lib, ops


def test_plain_forms_by_hand():
    x = np.zeros((1, 32), np.float32)
    x[0, :6] = [1.984375, -1, 0.0078125, 0.0234375, 3 / 128, -0.0078125]
    c, s = R.quantise(x, R.INT8)                       # 127/64 just fits 2^0; ties to even
    assert s[0, 0] == 127 and c[0, :6].tolist() == [127, -64, 0, 2, 2, 0]
    x[0, 0] = 2
    c, s = R.quantise(x, R.INT8)
    assert s[0, 0] == 128 and c[0, :2].tolist() == [64, -32]
    x[0, :4] = [6, -5, 0.25, 0.75]
    c, s = R.quantise(x, R.FP4)
    assert s[0, 0] == 127 and c[0, 0] == 7 | (0x8 | 6) << 4 and c[0, 1] == 0 | 2 << 4
    assert R.values(c, s, R.FP4)[0, :4].tolist() == [6, -4, 0, 1]
    x[0, 0] = 6.5
    assert R.quantise(x, R.FP4)[1][0, 0] == 128
    x[0, 1] = np.inf
    assert R.quantise(x, R.FP4)[1][0, 0] == 255 and np.isnan(R.values(*R.quantise(x, R.FP4), R.FP4)).all()


def test_sizes():
    L = _lib.load()
    assert ops.mx_row_bytes(ops.MX_INT8, 96) == 96 and ops.mx_row_bytes(ops.MX_FP4, 96) == 48
    for cols in (0, -32, 33, 16):
        with pytest.raises(ValueError):
            ops.mx_row_bytes(ops.MX_INT8, cols)
    with pytest.raises(ValueError):
        ops.mx_row_bytes(2, 32)
    assert L.aero_hip_mx_weight_bytes(1, 32) == 2176           # a tile of 32 rows, 128 columns
    assert L.aero_hip_mx_weight_bytes(33, 160) == 4 * 2176
    assert L.aero_hip_mx_weight_bytes(28672, 8192) == 28672 * 8192 * 17 // 32
    for sizes in ((0, 32), (1, 31), (1, 0), (-1, 32), (1, 1 << 25)):
        assert L.aero_hip_mx_weight_bytes(*sizes) == -1
    assert L.aero_hip_mx_matmul_workspace(2, 32, 32, 1) == -1
    assert L.aero_hip_mx_matmul_workspace(0, 32, 33, 1) == -1
    assert L.aero_hip_mx_matmul_workspace(0, 32, 32, -1) == -1
    assert L.aero_hip_mx_matmul_workspace(1, 32, 1 << 24, 1 << 60) == -1
    assert L.aero_hip_mx_matmul_workspace(0, 32, 32, 0) == 0
    assert L.aero_hip_mx_matmul_workspace(0, 32, 32, 32) == 0
    assert L.aero_hip_mx_matmul_workspace(0, 32, 160, 33) == 2 * 2 * (4 * 1536 + 128)
    assert L.aero_hip_mx_matmul_workspace(1, 32, 160, 33) == 2 * 2 * (2 * 1024 + 128)
    assert L.aero_hip_mx_matmul_workspace(0, 20480, 32, 17) == 4 * 1536 + 128


@pytest.mark.parametrize("call,args,reason", [
    ("mx_quantize", (2, 16, 32, 16, 16, 1, 32, None), "format"),
    ("mx_quantize", (0, 16, 32, 16, 16, 1, 31, None), "blocks"),
    ("mx_quantize", (0, 16, 32, 16, 16, 1, 0, None), "blocks"),
    ("mx_quantize", (0, 16, 32, 16, 16, -1, 32, None), "arguments"),
    ("mx_quantize", (0, None, 32, 16, 16, 1, 32, None), "input"),
    ("mx_quantize", (0, 18, 32, 16, 16, 1, 32, None), "input"),
    ("mx_quantize", (0, 16, 32, None, 16, 1, 32, None), "arguments"),
    ("mx_quantize", (0, 16, 32, 16, None, 1, 32, None), "arguments"),
    ("mx_quantize", (0, 16, 32, 18, 16, 1, 32, None), "4 bytes"),
    ("mx_quantize", (0, 16, 31, 16, 16, 1, 32, None), "apart"),
    ("mx_dequant", (5, 16, 16, 16, 1, 32, None), "format"),
    ("mx_dequant", (0, 16, 16, None, 1, 32, None), "input"),
    ("mx_dequant", (0, 16, 16, 16, 1, 48, None), "blocks"),
    ("rmsnorm_mx", (0, 16, 16, None, 16, 16, 16, 1, 32, 1e-5, 0, None), "together"),
    ("rmsnorm_mx", (0, 16, None, 16, 16, 16, 16, 1, 32, 1e-5, 0, None), "together"),
    ("rmsnorm_mx", (0, 16, None, None, 17, 16, 16, 1, 32, 1e-5, 0, None), "input"),
    ("rmsnorm_mx", (0, 16, None, None, 16, 16, 16, 1, 32, 1e-5, 2, None), "flags"),
    ("rmsnorm_mx", (0, 16, None, None, 16, 16, 16, 1, 40, 1e-5, 0, None), "blocks"),
    ("act_mul_mx", (0, 9, 16, 16, 32, 16, 16, 1, 32, None), "kind"),
    ("act_mul_mx", (0, 3, 16, None, 32, 16, 16, 1, 32, None), "identity"),
    ("act_mul_mx", (0, 0, None, 16, 32, 16, 16, 1, 32, None), "input"),
    ("act_mul_mx", (0, 0, 16, 16, 16, 16, 16, 1, 32, None), "apart"),
    ("mx_pack", (16, 16, 16, 2175, 1, 32, None), "bytes"),
    ("mx_pack", (16, 16, 24, 4096, 1, 32, None), "bytes"),
    ("mx_pack", (16, 16, None, 4096, 1, 32, None), "bytes"),
    ("mx_pack", (16, 16, 16, 4096, 0, 32, None), "rows"),
    ("mx_matmul", (0, 16, 16, 16, 2175, 16, 1, 32, 1, None, 0, None), "take"),
    ("mx_matmul", (0, 20, 16, 16, 2176, 16, 1, 32, 1, None, 0, None), "16-byte"),
    ("mx_matmul", (0, 16, 16, 16, 2176, None, 1, 32, 1, None, 0, None), "y"),
    ("mx_matmul", (0, 16, 16, 16, 2176, 18, 1, 32, 1, None, 0, None), "y"),
    ("mx_matmul", (3, 16, 16, 16, 2176, 16, 1, 32, 1, None, 0, None), "format"),
    ("mx_matmul", (0, 16, 16, 16, 2176, 16, 1, 32, -1, None, 0, None), "arguments"),
    ("mx_matmul", (0, 16, 16, 24, 4096, 16, 1, 32, 1, None, 0, None), "take"),
    ("mx_matmul", (0, 16, 16, 16, 2176, 16, 1, 32, 33, None, 0, None), "workspace"),
    ("mx_matmul", (1, 16, 16, 16, 2176, 16, 1, 32, 33, 16, 2 * 2176 - 1, None), "workspace"),
    ("mx_matmul", (0, 16, 16, 16, 2176, 16, 1, 32, 33, 24, 1 << 20, None), "workspace"),
])
def test_refusals(call, args, reason):
    """Refused with a reason before anything is launched: no pointer here is memory."""
    L = _lib.load()
    assert getattr(L, "aero_hip_" + call)(*args) == 0
    assert reason in _lib.last_error(), _lib.last_error()


def test_nothing_to_do():
    L = _lib.load()
    assert L.aero_hip_mx_quantize(0, 16, 32, 16, 16, 0, 32, None) == 1
    assert L.aero_hip_mx_dequant(0, 16, 16, 16, 0, 32, None) == 1
    assert L.aero_hip_rmsnorm_mx(0, 16, None, None, None, 16, 16, 0, 32, 1e-5, 0, None) == 1
    assert L.aero_hip_act_mul_mx(0, 0, 16, None, 32, 16, 16, 0, 32, None) == 1
    assert L.aero_hip_mx_matmul(0, 16, 16, 16, 2176, 16, 1, 32, 0, None, 0, None) == 1


def test_arrays_are_checked():
    """Buffers too small or of another type are refused by the Python ops."""
    def arr(n, dtype):
        return ops.DeviceArray((n,), dtype, _ptr=16, _owner=False)

    x, c8, c4, s = arr(64, np.float32), arr(64, np.int8), arr(32, np.uint8), arr(2, np.uint8)
    with pytest.raises(TypeError):
        ops.mx_quantize(ops.MX_INT8, x, c4, s, 1, 64)
    with pytest.raises(TypeError):
        ops.mx_quantize(ops.MX_FP4, x, c8, s, 1, 64)
    with pytest.raises(ValueError):
        ops.mx_quantize(ops.MX_INT8, x, c8, s, 2, 64)
    with pytest.raises(ValueError):
        ops.mx_quantize(ops.MX_INT8, x, c8, s, 2, 32, ld=33)
    with pytest.raises(ValueError):
        ops.mx_dequant(ops.MX_FP4, c4, s, arr(63, np.float32), 1, 64)
    with pytest.raises(ValueError):
        ops.rmsnorm_mx(ops.MX_INT8, x, arr(32, np.float32), c8, s, 1, 64, 1e-5)
    with pytest.raises(ValueError):
        ops.rmsnorm_mx(ops.MX_INT8, x, None, c8, s, 1, 64, 1e-5, x_out=x)
    with pytest.raises(ValueError):
        ops.act_mul_mx(ops.MX_INT8, "silu", x, arr(63, np.float32), c8, s, 1, 64)
    with pytest.raises(KeyError):
        ops.act_mul_mx(ops.MX_INT8, "relu", x, x, c8, s, 1, 64)


@pytest.mark.parametrize("fmt,n_tok,n_rows,n_cols,few", [
    # us on the few-token kernel (which takes no workspace) and on tiles
    (0, 16, 1 << 20, 8192, True),
    (0, 17, 20000, 8192, False),          # 32.0, 19.7: a second round of workgroups
    (0, 32, 20000, 8192, False),          # 39.0, 23.1
    (1, 24, 18432, 4096, False),          # 16.5, 11.4
    (0, 24, 5120, 5120, False),           # 15.3, 11.0
    (0, 24, 10240, 4096, False),          # 16.2, 10.5
    (0, 32, 4096, 14336, False),          # 23.3, 19.0
    (0, 17, 4096, 14336, True),           # 16.9, 18.7
    (0, 24, 14336, 4096, False),          # 12.2, 11.3
    (1, 24, 14336, 4096, True),           # 9.4, 9.9
    (0, 32, 16384, 2048, True),           # 8.5, 9.9
    (0, 32, 4096, 4096, True),            # 8.6, 9.8
    (0, 32, 9728, 896, True),             # 6.1, 7.3
    (1, 32, 5120, 2560, True),            # 6.2, 6.4
    (0, 33, 32, 32, False),
])
def test_which_calls_are_few_tokens(fmt, n_tok, n_rows, n_cols, few):
    """The rule between the product's two ways, on a chip of 256 CUs, at sizes where the
    other one was measured to be slower."""
    assert (_lib.load().aero_hip_mx_matmul_workspace(fmt, n_rows, n_cols, n_tok) == 0) == few


@pytest.mark.parametrize("fmt,n_tok,n_rows,n_cols,tiles", [
    (0, 2048, 28672, 4096, 0), (1, 2048, 28672, 4096, 0), (0, 512, 6144, 4096, 1), (0, 512, 4096, 14336, 2),
    (1, 333, 2560, 10240, 3), (0, 70, 40000, 2048, 4), (1, 64, 4096, 4096, 5), (1, 128, 14336, 128, 5),
    (0, 1, 4096, 4096, 6), (0, 20, 4096, 4096, 6), (1, 0, 64, 64, 6),
    (0, 1, 4096, 4095, -1), (0, 1, 0, 64, -1), (2, 1, 64, 64, -1), (0, -1, 64, 64, -1)])
def test_which_tiles(fmt, n_tok, n_rows, n_cols, tiles):
    """What the rule takes on a chip of 256 CUs."""
    assert _lib.load().aero_hip_mx_matmul_tiles(fmt, n_rows, n_cols, n_tok) == tiles


def recorded(call):
    """Launches of a call that is recorded, not run: no pointer here is memory."""
    L = _lib.load()
    plan = L.aero_hip_plan_create()
    assert L.aero_hip_plan_begin(plan)
    try:
        call()
    finally:
        L.aero_hip_plan_end(plan)
        n = L.aero_hip_plan_size(plan)
        L.aero_hip_plan_destroy(plan)
    return n


def test_more_lanes_than_a_launch_takes():
    """A launch has fewer than 2^32 lanes; larger calls are several."""
    L = _lib.load()
    for rows, cols, n in ((1 << 25, 32, 1), ((1 << 25) + 1, 32, 2), (1 << 26, 32, 2), ((1 << 26) + 1, 512, 3),
                          (1 << 23, 1024, 1), ((1 << 23) + 1, 1024, 2), (1 << 21, 16384, 1), ((1 << 22) + 1, 16384, 3)):
        assert recorded(lambda: _lib.check(L.aero_hip_rmsnorm_mx(
            0, 16, None, None, None, 16, 16, rows, cols, 1e-5, 0, None), "norm")) == n
    for addr, rows, n in ((16, 1 << 25, 1), (20, 1 << 25, 4)):         # not at 16 bytes: 256 lanes a row
        assert recorded(lambda: _lib.check(L.aero_hip_rmsnorm_mx(
            1, addr, None, None, None, 16, 16, rows, 32, 1e-5, 0, None), "norm")) == n
    for rows, n in ((1 << 28, 1), ((1 << 28) + 1, 2), ((1 << 30) + 1, 5)):
        assert recorded(lambda: _lib.check(L.aero_hip_mx_dequant(0, 16, 16, 16, rows, 32, None), "dequant")) == n
        assert recorded(lambda: _lib.check(L.aero_hip_mx_quantize(1, 16, 32, 16, 16, rows, 32, None), "quantize")) == n
    for rows, cols, n in ((1 << 24, 4096, 1), ((1 << 24) + 1, 4096, 2), ((1 << 26) - 1, 4096, 4)):
        assert recorded(lambda: _lib.check(L.aero_hip_mx_pack(
            16, 16, 16, 1 << 60, rows, cols, None), "pack")) == n


@pytest.mark.parametrize("n_tok,n_rows,n", [(1, 1 << 27, 1),
                                           (16, (1 << 28) - 32, 1), (1, 1 << 28, 0), (20, 1 << 31, 2)])
def test_products_with_more_rows_than_a_launch_takes(n_tok, n_rows, n):
    L, ok = _lib.load(), []
    launches = recorded(lambda: ok.append(L.aero_hip_mx_matmul(
        0, 16, 16, 16, 1 << 60, 16, n_rows, 32, n_tok, 16, 1 << 60, None)))
    assert ok == [n > 0]
    assert launches == n if n else "too many" in _lib.last_error()


@pytest.mark.parametrize("n_tok,n_rows,n_cols,ws,launches", [
    (24, 5120, 5120, True, 2), (24, 5120, 5120, False, 1), (32, 40960, 8192, False, 1), (17, 64, 64, True, 1),
    (17, 64, 64, False, 1), (33, 64, 64, True, 2), (33, 64, 64, False, 0)])
def test_few_tokens_without_a_workspace(n_tok, n_rows, n_cols, ws, launches):
    """Up to 32 tokens need no workspace, whichever kernel the rule would take with one."""
    L, ok = _lib.load(), []
    n = recorded(lambda: ok.append(L.aero_hip_mx_matmul(
        0, 16, 16, 16, 1 << 60, 16, n_rows, n_cols, n_tok, 16 if ws else None, 1 << 60 if ws else 0, None)))
    assert ok == [launches > 0] and n == launches
    if not launches:
        assert "workspace" in _lib.last_error()
