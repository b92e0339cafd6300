# SPDX-License-Identifier: Unlicense
"""ops_groupnorm_cl against its plain form in 64 bits (GPU).

Bound: with z = (x - mean) / sigma (sigma^2 = var + eps) and A the largest
|x| / sigma of the group, the mean is off by at most 24 steps of 2^-24 of A
(in units of sigma: the sums of a thread are split so that no chain of
additions is longer than 16, then trees), the variance by 32 steps relative
plus twice the mean's error squared; x - mean, the scaling, gamma and beta
add 6 steps. So |y - want| <= |g| (40 A + 40 |z|) 2^-24 + 8 |b| 2^-24, with
the activation's (test_linear_i8_gpu.py's 32 steps of its argument) and the
store's half step."""

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from typed_ops import BF16, F32, HALF_STEP, Rows, close, rounded

TYPES = {"f32": F32, "bf16": BF16}


class Maps:
    """nimg maps of HW x C in one guarded buffer: images as runs of rows."""

    def __init__(self, dev, nimg, HW, C, t, values=None, off=0, ld=None, gap=0):
        self.ld = C if ld is None else ld
        self.nimg, self.HW, self.C = nimg, HW, C
        rows = nimg * HW + (nimg - 1) * gap
        self.pick = np.concatenate([np.arange(HW) + i * (HW + gap) for i in range(nimg)])
        v = None
        if values is not None:
            v = np.full((rows, C), 0.25, np.float32)
            v[self.pick] = values.reshape(-1, C)
        self.rows = Rows(dev, rows, C, t, v, off=off, ld=self.ld)
        self.v, self.t = v, t
        self.opnd = coreg.Opnd(self.rows.handle, off, self.ld, (HW + gap) * self.ld, 0)

    def read(self):
        got = self.rows.read()
        rest = np.ones(len(got), bool)
        rest[self.pick] = False
        if self.v is not None:
            assert (got[rest] == 0.25).all()
        return got[self.pick].reshape(self.nimg, self.HW, self.C)


def call(dev, X, Y, groups, g, b, kind="none", eps=1e-5):
    G = None if g is None else dev.upload(g)
    B = None if b is None else dev.upload(b)
    need = dev.lib.ops_groupnorm_cl_bytes(X.nimg, X.HW, X.C, groups)
    work = dev.alloc(need) if need else None
    dev.lib.ops_groupnorm_cl(dev.ops_p, X.nimg, X.HW, X.C, groups, X.opnd, X.t, Y.opnd, Y.t,
                             coreg.handle(G), coreg.handle(B), eps, ref.ACTS.index(kind), 0.1,
                             coreg.handle(work))
    out = Y.read()
    coreg.check(dev.lib)
    return out


def check(got, x, groups, g, b, kind, t, eps=1e-5):
    n, hw, C = x.shape
    v = x.astype(np.float64).reshape(n, hw, groups, -1)
    sigma = np.sqrt(v.var((1, 3), keepdims=True) + eps)
    A = np.broadcast_to(np.abs(v).max((1, 3), keepdims=True) / sigma, v.shape).reshape(x.shape)
    pre = ref.groupnorm(x, groups, g, b, eps)
    z = np.abs(ref.groupnorm(x, groups, None, None, eps))
    ga, ba = (1.0, 0.0) if g is None else (np.abs(g), np.abs(b))
    want = ref.act(pre, kind)
    tol = 2.0 ** -24 * (ga * 40 * (A + z) + 8 * ba) * 1.2 + HALF_STEP[t] * np.abs(want)
    if kind in ("gelu", "gelu_tanh", "silu"):
        tol = tol + 32 * 2.0 ** -24 * np.abs(pre)
    close(got, want, tol + 1e-37)


SHAPES = [
    # images, pixels, channels, groups, X (offset, pitch, gap), Y (offset, pitch, gap)
    (1, 1, 1, 1, (0, 1, 0), (0, 1, 0)),
    (1, 1, 64, 32, (0, 64, 0), (0, 64, 0)),
    (2, 7, 6, 3, (1, 7, 2), (2, 9, 1)),
    (1, 1225, 512, 32, (0, 512, 0), (0, 512, 0)),
    (3, 341, 120, 5, (0, 120, 0), (0, 120, 0)),
    (2, 4097, 64, 32, (0, 64, 0), (0, 64, 0)),
    (2, 1000, 64, 1, (0, 64, 0), (0, 64, 0)),
    (5, 300, 256, 8, (8, 264, 0), (0, 256, 0)),
    (1, 20000, 16, 16, (0, 16, 0), (0, 16, 0)),
    (1, 33, 1000, 10, (0, 1000, 0), (0, 1000, 0)),
    (2, 50, 2048, 32, (0, 2048, 0), (0, 2048, 0)),
    (1, 3001, 33, 11, (0, 33, 0), (0, 33, 0)),
    (9, 64, 96, 4, (4, 100, 3), (8, 104, 5)),
    (1, 17, 6000, 3, (0, 6000, 0), (0, 6000, 0)),
    (40, 5, 8, 2, (0, 8, 0), (0, 8, 0)),
    (2, 130000, 8, 4, (0, 8, 0), (0, 8, 0)),
    (1, 90001, 64, 16, (0, 64, 0), (0, 64, 0)),
    # Several images at a time over the whole grid, the last batch not full;
    # channels merged by four, two and none; rows in twos, fours and eights.
    (3, 60001, 32, 8, (0, 32, 0), (0, 32, 0)),
    (5, 30007, 64, 32, (0, 64, 2), (0, 64, 0)),
    (3, 50001, 36, 9, (0, 36, 0), (0, 36, 0)),
    (2, 70003, 34, 17, (0, 34, 0), (0, 34, 0)),
    (4, 9001, 204, 34, (0, 204, 0), (0, 204, 0)),
    (1, 40009, 63, 7, (0, 63, 0), (0, 63, 0)),
    (3, 5, 21, 7, (0, 21, 0), (0, 21, 0)),
    # Odd channel counts too wide for whole vectors; groups wider than a block.
    (1, 50, 1003, 17, (0, 1003, 0), (0, 1003, 0)),
    (2, 9, 9000, 2, (0, 9000, 0), (0, 9000, 0)),
]


def maps(rng, n, hw, C, t):
    x = rng.standard_normal((n, hw, C)) * np.exp(0.5 * rng.standard_normal(C))
    return rounded(x + 2 * rng.standard_normal(C), t)


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["f32-f32", "f32-bf16", "bf16-f32", "bf16-bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_groupnorm(dev, shape, types):
    n, hw, C, groups, (xo, xl, xg), (yo, yl, yg) = shape
    xt, yt = (TYPES[t] for t in types.split("-"))
    rng = np.random.default_rng(hw + C)
    x = maps(rng, n, hw, C, xt)
    g, b = (rng.standard_normal(C).astype(np.float32) for _ in range(2))
    X = Maps(dev, n, hw, C, xt, x, xo, xl, xg)
    Y = Maps(dev, n, hw, C, yt, np.zeros_like(x), yo, yl, yg)
    got = call(dev, X, Y, groups, g, b)
    check(got, x, groups, g, b, "none", yt)
    assert (X.read() == x).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ref.ACTS)
def test_groupnorm_activations_in_place(dev, kind, t):
    rng = np.random.default_rng(3)
    for n, hw, C, groups in ((2, 600, 96, 12), (1, 30000, 64, 8)):
        x = maps(rng, n, hw, C, TYPES[t])
        g, b = (rng.standard_normal(C).astype(np.float32) for _ in range(2))
        X = Maps(dev, n, hw, C, TYPES[t], x)
        check(call(dev, X, X, groups, g, b, kind), x, groups, g, b, kind, TYPES[t])
        # without gamma and beta
        X = Maps(dev, n, hw, C, TYPES[t], x)
        check(call(dev, X, X, groups, None, None, kind), x, groups, None, None, kind, TYPES[t])


@pytest.mark.gpu
@pytest.mark.parametrize("hw", [50, 5000, 200000])
def test_groupnorm_large_mean(dev, hw):
    """Values far from zero (mean 1000 sigma): the variance has to come from
    differences; and a constant group gives beta."""
    rng = np.random.default_rng(hw)
    x = (1000 + rng.standard_normal((1, hw, 16))).astype(np.float32)
    x[..., 4:8] = -37.5
    g, b = (rng.standard_normal(16).astype(np.float32) for _ in range(2))
    X, Y = Maps(dev, 1, hw, 16, F32, x), Maps(dev, 1, hw, 16, F32, np.zeros_like(x))
    got = call(dev, X, Y, 4, g, b)
    check(got, x, 4, g, b, "none", F32)


@pytest.mark.gpu
@pytest.mark.parametrize("hw", [40, 40000])
def test_groupnorm_nan_stays_in_its_group(dev, hw):
    rng = np.random.default_rng(hw)
    x = maps(rng, 2, hw, 32, F32)
    x[0, hw // 2, 9] = np.nan
    x[1, hw - 1, 0] = np.inf
    X, Y = Maps(dev, 2, hw, 32, F32, x), Maps(dev, 2, hw, 32, F32, np.zeros_like(x))
    got = call(dev, X, Y, 4, None, None)
    assert np.isnan(got[0, :, 8:16]).all()
    assert np.isnan(got[1, :, :8]).all()
    clean = x.copy()
    clean[0, :, 8:16] = 1.0
    clean[1, :, :8] = 1.0
    want = ref.groupnorm(clean, 4)
    ok = np.ones(x.shape, bool)
    ok[0, :, 8:16] = ok[1, :, :8] = False
    assert np.abs(got[ok] - want[ok]).max() <= 1e-4
