# SPDX-License-Identifier: Unlicense
"""ops_gemm and ops_gemm_noalloc in bfloat16 mode into some columns of a wider
float32 matrix (GPU): rows 16-byte aligned whose last column ends anywhere,
every width of tile; the columns behind and the rows' ends stay as they were.

The operands are whole numbers, exact in bfloat16, and their sums in float32:
results are equal."""

import numpy as np
import pytest

import coreg
from coreg import Opnd
from typed_ops import F32, Rows

SHAPES = [
    # M, N, K, columns behind N
    (130, 1, 64, 3),
    (746, 6, 32, 2),
    (300, 15, 64, 1),
    (200, 17, 40, 7),
    (129, 31, 64, 5),
    (300, 50, 128, 2),
    (77, 130, 40, 6),
    (200, 141, 64, 3),
    (300, 253, 64, 3),
    (1000, 1003, 256, 1),
    (129, 4097, 64, 3),
    (3300, 2901, 256, 3),
    (3300, 2902, 256, 10),
    (300, 64, 64, 4),
]


@pytest.fixture(scope="module")
def dev16():
    d = coreg.Device(0, precision=coreg.OPS_BF16)
    yield d
    d.close()


@pytest.mark.gpu
@pytest.mark.parametrize("act", [coreg.ACT_NONE, coreg.ACT_RELU], ids=["none", "relu"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_columns_behind_are_left(dev16, shape, act):
    M, N, K, more = shape
    rng = np.random.default_rng(N)
    a, b = (rng.integers(-8, 9, (n, K)).astype(np.float32) for n in (M, N))
    bias, res = rng.integers(-9, 10, N), rng.integers(-99, 100, (M, N))
    want = a.astype(np.float64) @ b.T + bias
    want = (np.maximum(want, 0) if act == coreg.ACT_RELU else want) + res
    A, B, V = dev16.upload(a), dev16.upload(b), dev16.upload(bias.astype(np.float32))
    for fn in (dev16.lib.ops_gemm, dev16.lib.ops_gemm_noalloc):
        # A residual of its own, then in place.
        R = Rows(dev16, M, N, F32, res, off=4, ld=N + more)
        C = Rows(dev16, M, N, F32, np.full((M, N), 7), off=8, ld=N + more)
        for out, off in ((C, 8), (R, 4)):
            fn(dev16.ops_p, M, N, K, Opnd(A.handle, 0, K, 0, 0), Opnd(B.handle, 0, K, 0, 0), 1,
               Opnd(out.handle, off, N + more, 0, 0), 1, 1, V.handle, 0, R.handle, 4, 1.0, act, 0.0)
            assert (out.read() == want).all()
    assert dev16.lib.coreg_tc_status() == 0
