# SPDX-License-Identifier: Unlicense
"""ops_groupnorm_cl where a thread has many vectors (GPU): more than it keeps
in shared memory and more than one run of sums, in whole vectors and single
values, over the grid and in clusters; and with a first pixel far off the
others, about which no sums may be taken.

The bound is test_groupnorm_gpu.py's. A thread's sums are chains of at most 8
+ 16 additions, joined in 64 bits: the mean is off by 24 steps of 2^-24 of the
largest |x|, the variance by as many relative, for any number of pixels. A
far first value of K (in sigmas of the others) leaves squares of about (K /
8)^2 in the 128 values after it: 24 steps of 2 K^2, of the K^2 that it adds to
the group's M2 itself, 48 relative to a variance that it makes up: 24 of z,
which the bound's 40 (A + |z|), A >= |z|, holds."""

import numpy as np
import pytest

from test_groupnorm_gpu import TYPES, Maps, call, check
from typed_ops import rounded

CASES = [
    # images, pixels, channels, groups, X and Y pitch, type
    # Single values: groups too many for a block (clusters, threads of
    # thousands of values), and over the grid.
    (1, 46657, 1002, 2, 1003, "f32"),
    (1, 20011, 1002, 2, 1003, "bf16"),
    (1, 400003, 30, 5, 31, "f32"),
    (1, 700003, 30, 5, 31, "bf16"),
    (2, 100003, 62, 31, 63, "f32"),
    # Whole vectors: merged by four, two and one channels, in fours of rows with
    # the map's end inside one.
    (1, 1250003, 32, 8, 32, "f32"),
    (1, 1250003, 32, 16, 32, "f32"),
    (1, 640003, 63, 7, 63, "f32"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("far", [0, 1e4], ids=["plain", "far"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_long_maps(dev, case, far):
    n, hw, C, groups, ld, t = case
    rng = np.random.default_rng(C)
    x = rng.standard_normal((n, hw, C), np.float32)
    x += rng.standard_normal(C).astype(np.float32)
    if far:
        x[:, 0] = far
        x[:, 1, ::2] = -far
    x = rounded(x, TYPES[t])
    g, b = (rng.standard_normal(C).astype(np.float32) for _ in range(2))
    X = Maps(dev, n, hw, C, TYPES[t], x, ld=ld)
    Y = Maps(dev, n, hw, C, TYPES["f32"], np.zeros_like(x), ld=ld)
    check(call(dev, X, Y, groups, g, b), x, groups, g, b, "none", TYPES["f32"])
