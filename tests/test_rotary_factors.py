# SPDX-License-Identifier: Unlicense
"""The magnitude factor that ops_rotary_plan sets for frequencies changed by
parts (CPU): 0.1 ln(factor) + 1 from a factor of 1 on, and 1 below, where the
logarithm would shrink the values and, below e^-10, turn them round."""

import math

import pytest

from test_rotary_gpu import make_plan


@pytest.mark.parametrize("factor", [1e-6, 1e-3, 0.5, 0.999, 1.0, 1.001, 2.0, 16.0, 1e6])
def test_parts_magnitude(factor):
    want = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    got = make_plan(64, 1, 0, 10000.0, "parts", factor, 4096).mscale
    assert abs(got - want) <= 2.0 ** -24 * want


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk"])
def test_other_scalings_keep_magnitudes(scaling):
    assert make_plan(64, 1, 0, 10000.0, scaling, 8.0, 4096).mscale == 1.0
