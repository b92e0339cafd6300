# SPDX-License-Identifier: Unlicense
"""ops_groupnorm_cl of finite values whose squares pass float32's range (GPU):
the group's variance is infinite and its result act(b), exactly; other groups
keep theirs."""

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from test_groupnorm_gpu import TYPES, Maps, call

CASES = [
    # images, pixels, channels, groups, pitch: a cluster, the grid, single
    # values, rows in fours, threads of many vectors, a group wider than a block.
    (1, 40, 32, 4, 32),
    (2, 1225, 512, 32, 512),
    (1, 90001, 64, 16, 64),
    (1, 3001, 34, 2, 35),
    (1, 40009, 63, 7, 63),
    (1, 20011, 1002, 2, 1003),
    (1, 50, 9000, 2, 9000),
    # Runs of 512 pixels of either sign, so that every thread has as many of both
    # and all their means are equal.
    (1, 8192, 32, 4, 32),
    (1, 8192, 32, 4, 33),
    (2, 131072, 32, 4, 32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_infinite_variance(dev, case, t):
    n, hw, C, groups, ld = case
    per = C // groups
    rng = np.random.default_rng(C)
    x = rng.choice(np.float32([-1, 1]), (n, hw, C))
    if hw % 8192 == 0:
        x[..., :per] = np.where(np.arange(hw) // 512 % 2, -1, 1)[:, None]
    x[..., :per] *= np.float32(2.0 ** 67)
    g, b = (rng.standard_normal(C).astype(np.float32) for _ in range(2))
    X = Maps(dev, n, hw, C, TYPES[t], x, ld=ld)
    Y = Maps(dev, n, hw, C, coreg.OPS_FP32, np.zeros_like(x), ld=ld)
    got = call(dev, X, Y, groups, g, b, "relu")
    assert (got[..., :per] == np.maximum(b[:per], 0)).all()
    x[..., :per] = 1
    want = ref.groupnorm(x, groups, g, b, kind="relu")
    # |z| is about 1: 80 steps of it and 8 of b, as in test_groupnorm_gpu.py.
    tol = 2.0 ** -24 * (90 * np.abs(g) + 8 * np.abs(b)) * 1.2 + 2.0 ** -24 * np.abs(want)
    assert (np.abs(got - want) <= tol)[..., per:].all()
