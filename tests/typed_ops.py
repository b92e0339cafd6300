# SPDX-License-Identifier: Unlicense
"""Buffers of typed rows for the tests of the typed operations of
ops_b200.h: float32 or bfloat16 values in strided rows inside a larger
buffer, whose other elements have to stay as they were."""

import numpy as np

import coreg
from test_tc_gemm_gpu import bf16_round

F32, BF16 = coreg.OPS_FP32, coreg.OPS_BF16
# Largest relative rounding of a value written in the type: half a step.
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
GUARD = 0x7B


def rounded(x, t):
    x = np.asarray(x, np.float32)
    return bf16_round(x) if t == BF16 else x


def to_bytes(x, t):
    x = rounded(x, t)
    if t == BF16:
        return (x.view(np.uint32) >> 16).astype(np.uint16).view(np.uint8)
    return np.ascontiguousarray(x).view(np.uint8)


def from_bytes(raw, t):
    if t == BF16:
        return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32)
    return raw.view(np.float32)


class Rows:
    """rows x cols elements of type t (or int8 with t None) at an element
    offset and pitch, the rest of the buffer filled with a guard byte."""

    def __init__(self, dev, rows, cols, t, values=None, off=0, ld=None, tail=7):
        self.dev, self.rows, self.cols, self.t = dev, rows, cols, t
        self.off, self.ld = off, cols if ld is None else ld
        self.es = {F32: 4, BF16: 2, None: 1}[t]
        self.n = off + max(rows - 1, 0) * self.ld + cols + tail
        raw = np.full(self.n * self.es, GUARD, np.uint8)
        self.buf = None
        self.inside = np.zeros(self.n, bool)
        for r in range(rows):
            self.inside[off + r * self.ld:off + r * self.ld + cols] = True
        if values is not None:
            v = np.ascontiguousarray(np.asarray(values).reshape(-1))
            v = v.astype(np.int8).view(np.uint8) if t is None else to_bytes(v, t)
            raw.reshape(self.n, self.es)[self.inside] = v.reshape(-1, self.es)
        self.buf = dev.upload(raw)

    @property
    def opnd(self):
        return coreg.Opnd(self.buf.handle, self.off, self.ld, 0, 0)

    @property
    def handle(self):
        return self.buf.handle

    def read(self):
        """The values; fails where anything around them was written."""
        raw = self.buf.read(np.uint8, self.n * self.es).reshape(self.n, self.es)
        coreg.check(self.dev.lib)
        assert (raw[~self.inside] == GUARD).all(), "written outside the rows"
        v = np.ascontiguousarray(raw[self.inside]).reshape(-1)
        v = v.view(np.int8) if self.t is None else from_bytes(v, self.t)
        return v.reshape(self.rows, self.cols)


def close(got, want, tol):
    """Elementwise |got - want| <= tol, NaN and infinities in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fin = np.isfinite(want)
    assert (np.isnan(got) == np.isnan(want)).all()
    assert (got[~fin & ~np.isnan(want)] == want[~fin & ~np.isnan(want)]).all()
    err = np.abs(got - want)[fin]
    tol = np.broadcast_to(tol, want.shape)[fin]
    bad = err > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.max(err / tol)} of the bound"
