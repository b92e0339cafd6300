# SPDX-License-Identifier: Unlicense
"""ops_groupnorm_cl over groups wider than a block's threads hold vectors of
(GPU), at sizes where a chain of float32 sums goes wrong: in the bound of
test_groupnorm_gpu.py, whose statistics' errors do not grow with the size."""

import numpy as np
import pytest

from test_groupnorm_gpu import TYPES, Maps, call, check
from typed_ops import rounded

CASES = [
    # images, pixels, channels, groups, pitch, mean in sigmas, input type
    # 36 million values of one group far from zero: a float32 sum of raw
    # values passes 1e8, where its steps are 8.
    (1, 46657, 771, 1, 771, 1003, "f32"),
    (1, 20000, 2052, 1, 2052, -500, "f32"),
    # The variance's own chain.
    (1, 50000, 1001, 1, 1001, 0, "f32"),
    (1, 9001, 4104, 1, 4104, 0, "bf16"),
    (2, 3001, 1206, 2, 1207, 30, "f32"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_wide_groups(dev, case):
    n, hw, C, groups, ld, mean, t = case
    rng = np.random.default_rng(C)
    x = rounded(mean + rng.standard_normal((n, hw, C), np.float32), TYPES[t])
    g, b = (rng.standard_normal(C).astype(np.float32) for _ in range(2))
    X = Maps(dev, n, hw, C, TYPES[t], x, ld=ld)
    Y = Maps(dev, n, hw, C, TYPES["f32"], np.zeros_like(x), ld=ld)
    check(call(dev, X, Y, groups, g, b), x, groups, g, b, "none", TYPES["f32"])
