# SPDX-License-Identifier: Unlicense
"""The activations of the typed operations over the whole of float32 (GPU):
values that arrive as a bias (products with sums of zero, by the streaming
kernels, the tensor cores and at depth 0) and as a beta (maps of constant
groups), in all neighbourhoods of large and small ones.

Bounds, against 64 bits. SiLU and GELU-tanh: v / (1 + 2^z) with z up to 60 off
by at most 4 roundings of itself, 60 x 4 x 2^-24 ln 2 = 2^-16.6 of the result,
the quotient 4e-7 more: 2^-16. GELU: Phi is off by at most 1.5e-7, times |v|
and a rounding: 2e-7 |v|, to v = -14. Where z passes 60 (v below -41 for SiLU,
-13.8 for GELU, -7.5 for GELU-tanh) the result is below 60 2^-60 and the true
one too: 2^-54 absolute, whatever v is. ReLU and leaky: a rounding."""

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from test_groupnorm_gpu import Maps, call
from typed_ops import F32, Rows

SIZES = [0.0, 1e-30, 1e-3, 0.5, 1, 3, 5, 6.5, 7.4, 7.6, 9, 13.7, 13.9, 14.1, 20, 41, 41.5, 42, 50, 63.9,
         64.1, 88, 100, 127, 1e3, 1e6, 1e10, 1e20, 1e30, 3.4e38]


def values(n):
    v = np.float32(np.concatenate([SIZES, -np.float32(SIZES)]))
    return np.random.default_rng(n).choice(v, n).astype(np.float32)


def bound(v, want, kind):
    v = v.astype(np.float64)
    if kind in ("silu", "gelu_tanh"):
        return 2.0 ** -16 * np.abs(want) * (v < 0) + 2.0 ** -20 * np.abs(want) + 2.0 ** -54
    if kind == "gelu":
        return np.where(v > -14, 2e-7 * np.minimum(np.abs(v), 14), 0) + 2.0 ** -20 * np.abs(want) + 2.0 ** -54
    return 2.0 ** -24 * np.abs(want)


def check(got, v, kind):
    # (v^3 of the largest passes a double's range in no form: 1e115.)
    want = ref.act(v.astype(np.float64), kind)
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= bound(v, want, kind))
    assert not bad.any(), list(zip(np.broadcast_to(v, got.shape)[bad][:5], got[bad][:5]))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ref.ACTS)
@pytest.mark.parametrize("M,N,K", [(1, 501, 0), (40, 501, 0), (1, 501, 16), (5, 501, 16), (40, 501, 16),
                                   (300, 700, 128), (300, 700, 2048), (20, 500, 2048)])
def test_products(dev, kind, M, N, K):
    v = values(N)
    A, B = (Rows(dev, n, K, None, np.zeros((n, K)), ld=(K + 15) // 16 * 16 + 16) for n in (M, N))
    S, V, C = dev.upload(np.ones(max(M, N), np.float32)), dev.upload(v), Rows(dev, M, N, F32)
    dev.lib.ops_gemm_i8(dev.ops_p, M, N, K, A.opnd, S.handle, B.opnd, S.handle, V.handle, C.opnd,
                        F32, None, 0, ref.ACTS.index(kind), 0.1)
    check(C.read(), v, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ref.ACTS)
@pytest.mark.parametrize("hw,C,ld", [(40, 640, 640), (60001, 64, 64), (50, 630, 631), (9, 8200, 8201)])
def test_group_norms(dev, kind, hw, C, ld):
    v, x = values(C), np.full((1, hw, C), 3, np.float32)
    X, Y = Maps(dev, 1, hw, C, F32, x, ld=ld), Maps(dev, 1, hw, C, F32, x, ld=ld)
    check(call(dev, X, Y, 2, np.ones(C, np.float32), v, kind), v, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_nan_keeps_to_itself(dev, kind):
    v = np.float32([np.nan, -1e30, -50, np.nan, np.nan, 2, 3, np.nan, -1, 1])
    A, C = Rows(dev, 40, 0, None, np.zeros((40, 0)), ld=16), Rows(dev, 40, 10, F32)
    S, V = dev.upload(np.ones(40, np.float32)), dev.upload(v)
    dev.lib.ops_gemm_i8(dev.ops_p, 40, 10, 0, A.opnd, S.handle, A.opnd, S.handle, V.handle, C.opnd,
                        F32, None, 0, ref.ACTS.index(kind), 0.1)
    got = C.read()
    assert (np.isnan(got) == np.isnan(v)).all()
    fin = ~np.isnan(v)
    check(got[:, fin], v[fin], kind)
