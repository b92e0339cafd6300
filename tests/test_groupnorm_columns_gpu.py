# SPDX-License-Identifier: Unlicense
"""ops_groupnorm_cl from some columns of a wider map into others of it: they
share no element, so it runs (GPU) wherever they lie in the rows; columns
that do share one are refused (CPU, with the checks before any CUDA call)."""

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from test_typed_ops_refusals import Host
from test_typed_ops_refusals import M as opnd
from typed_ops import F32

CASES = [
    # images, pixels, columns of a row, X's first, Y's first, rows between images
    (1, 300, 48, 0, 24, 0),
    (1, 300, 48, 24, 0, 0),
    (1, 300, 51, 1, 26, 0),
    (3, 130, 52, 4, 28, 0),
    (3, 130, 52, 28, 4, 2),
    (4, 1, 48, 0, 24, 0),
    (2, 9000, 48, 24, 0, 0),
]
C, GROUPS = 24, 3


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_columns_beside(dev, case):
    n, hw, ld, xc, yc, gap = case
    rng = np.random.default_rng(ld)
    rows = n * (hw + gap)
    m = rng.standard_normal((rows, ld)).astype(np.float32)
    B, work = dev.upload(m), dev.alloc(dev.lib.ops_groupnorm_cl_bytes(n, hw, C, GROUPS))
    X, Y = (coreg.Opnd(B.handle, c, ld, (hw + gap) * ld, 0) for c in (xc, yc))
    dev.lib.ops_groupnorm_cl(dev.ops_p, n, hw, C, GROUPS, X, F32, Y, F32, None, None, 1e-5, 0, 0.0,
                             work.handle)
    coreg.check(dev.lib)
    got = B.read().reshape(n, hw + gap, ld)
    m = m.reshape(n, hw + gap, ld)
    want = ref.groupnorm(m[:, :hw, xc:xc + C], GROUPS)
    assert np.abs(got[:, :hw, yc:yc + C] - want).max() <= 1e-4
    got[:, :hw, yc:yc + C] = m[:, :hw, yc:yc + C]
    assert (got == m).all()


def test_columns_that_meet_are_refused():
    h = Host()
    B, need = h.buf(), h.lib.ops_groupnorm_cl_bytes(2, 9, 12, 3)
    work = h.buf(need)

    def args(x, y, n=2, hw=9, xt=F32, yt=F32):
        return (n, hw, 12, 3, x, xt, y, yt, None, None, 1e-5, 0, 0.0, work)

    f = "ops_groupnorm_cl"
    # One column in common, either way round, and around the rows' end.
    h.refuses("overlaps", f, *args(opnd(B, 30, 0, 270), opnd(B, 30, 11, 270)))
    h.refuses("overlaps", f, *args(opnd(B, 30, 11, 270), opnd(B, 30, 0, 270)))
    h.refuses("overlaps", f, *args(opnd(B, 30, 0, 270), opnd(B, 30, 19, 270)))
    # Beside each other in a map, but not from map to map.
    h.refuses("overlaps", f, *args(opnd(B, 30, 0, 275), opnd(B, 30, 12, 275)))
    h.refuses("overlaps", f, *args(opnd(B, 30, 0, 270), opnd(B, 30, 12, 300 + 270 + 5)))
    # Rows of different lengths, types or counts of bytes.
    h.refuses("overlaps", f, *args(opnd(B, 30, 0, 270), opnd(B, 31, 12, 279)))
    h.refuses("overlaps", f, *args(opnd(B, 30, 0, 270), opnd(B, 30, 24, 270), yt=coreg.OPS_BF16))
    # Maps of one pixel that are closer together than their columns.
    h.refuses("overlaps", f, *args(opnd(B, 0, 0, 20), opnd(B, 0, 12, 20), hw=1))
