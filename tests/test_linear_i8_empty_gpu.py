# SPDX-License-Identifier: Unlicense
"""8-bit products and layers of depth 0 (GPU): act(bias) + R, whatever the
scales hold, which ops_quant_i8 leaves unwritten for rows without columns."""

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from typed_ops import BF16, F32, HALF_STEP, Rows, close, rounded


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["none", "relu", "silu"])
@pytest.mark.parametrize("M,N", [(1, 7), (2, 33), (5, 200), (8, 8), (9, 65), (300, 70)])
def test_depth_zero(dev, M, N, kind, t):
    rng = np.random.default_rng(M + N)
    bias, res = rng.standard_normal(N).astype(np.float32), rounded(rng.standard_normal((M, N)), t)
    junk = [dev.upload(np.full(max(M, N), v, np.float32)) for v in (np.nan, np.inf)]
    A, B = Rows(dev, M, 0, None, ld=16), Rows(dev, N, 0, None, ld=16)
    X, V = Rows(dev, max(M, N), 0, F32, ld=4), dev.upload(bias)
    R = Rows(dev, M, N, t, res, ld=N + 3)
    lib, o, act = dev.lib, dev.ops_p, ref.ACTS.index(kind)
    lib.ops_quant_i8(o, M, 0, X.opnd, F32, A.opnd, junk[0].handle, 0)
    lib.ops_quant_i8(o, N, 0, X.opnd, F32, B.opnd, junk[1].handle, 0)
    need = lib.ops_linear_i8_bytes(M, 0)
    work = dev.alloc(need) if need else None
    plain = ref.act(bias, kind)
    for b, r in ((V, R), (None, None), (V, None)):
        want = np.broadcast_to(plain if b else 0.0, (M, N)) + (res.astype(np.float64) if r else 0.0)
        mag = np.abs(bias) + np.abs(res)
        tol = 32 * 2.0 ** -24 * mag + HALF_STEP[t] * np.abs(want)
        for layer in (False, True):
            C = Rows(dev, M, N, t, np.full((M, N), 7), ld=N + 3)
            if layer:
                lib.ops_linear_i8(o, M, 0, N, X.opnd, F32, B.opnd, junk[1].handle, coreg.handle(b),
                                  C.opnd, t, r and r.handle, 0, act, 0.0, coreg.handle(work))
            else:
                lib.ops_gemm_i8(o, M, N, 0, A.opnd, junk[0].handle, B.opnd, junk[1].handle,
                                coreg.handle(b), C.opnd, t, r and r.handle, 0, act, 0.0)
            close(C.read(), want, tol)
