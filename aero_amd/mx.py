"""Weights in 4-bit microscaled numbers, laid out for ops.mx_matmul.

    w = MxWeight.from_rows(fp32_rows, n_rows, n_cols)       # quantised here
    w = MxWeight(codes, scales, n_rows, n_cols)             # rows of ops.mx_quantize
    ops.rmsnorm_mx(ops.MX_INT8, x, norm_w, c, s, T, n_cols, eps, d=d)
    ops.mx_matmul(ops.MX_INT8, c, s, w, y, T)

The layout (32 rows, blocks of 32 columns, 16 bytes a row) is that of the product's
matrix steps; it is made once, and the rows it was made from may be freed.
"""
from __future__ import annotations

import numpy as np

from . import _lib, ops
from .device import DeviceArray, Stream, recording_plan, synchronize


class MxWeight:
    """n_rows rows of n_cols 4-bit microscaled values (17 bytes for 32 of them), rows and
    columns rounded up to 32 and 128 with zeros."""

    def __init__(self, codes: DeviceArray, scales: DeviceArray, n_rows: int, n_cols: int,
                 stream: Stream | None = None):
        ops._mx_rows(ops.MX_FP4, codes, scales, n_rows, n_cols)
        if recording_plan() is not None:
            raise RuntimeError("MxWeight: weights are laid out once, not in a plan")
        L = _lib.lib()
        nbytes = int(L.aero_hip_mx_weight_bytes(n_rows, n_cols))
        _lib.check(nbytes > 0, "MxWeight")
        self.n_rows, self.n_cols = int(n_rows), int(n_cols)
        self.buf = DeviceArray.empty(nbytes, np.uint8)
        _lib.check(L.aero_hip_mx_pack(codes.ptr, scales.ptr, self.buf.ptr, nbytes, self.n_rows,
                                      self.n_cols, ops._s(stream)), "MxWeight")

    @classmethod
    def from_rows(cls, x: DeviceArray, n_rows: int, n_cols: int) -> "MxWeight":
        """Quantised from fp32 rows (ops.mx_quantize); complete when this returns."""
        if recording_plan() is not None:
            raise RuntimeError("MxWeight: weights are laid out once, not in a plan")
        codes = DeviceArray.empty(n_rows * ops.mx_row_bytes(ops.MX_FP4, n_cols), np.uint8)
        scales = DeviceArray.empty(n_rows * (n_cols // 32), np.uint8)
        ops.mx_quantize(ops.MX_FP4, x, codes, scales, n_rows, n_cols)
        w = cls(codes, scales, n_rows, n_cols)
        synchronize()
        return w
