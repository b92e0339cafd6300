# SPDX-License-Identifier: Unlicense
"""ops_rotary against its plain form in 64 bits (GPU), and ops_rotary_plan
(CPU: it needs no device).

Bound of a rotated value, of m (|a| + |b|): the cosine and sine to 2 steps
of 2^-24 (their fraction of a turn is exact to 2^-33 and rounds once more to
2^-24 of itself, within half a turn: pi 2^-24), the factor and the two
products and their sum a step each: under 12 steps; the store half a step of
the type. Other columns are copied."""

import ctypes as C

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from typed_ops import BF16, F32, HALF_STEP, Rows, close, rounded

TYPES = {"f32": F32, "bf16": BF16}
SCALINGS = ("none", "linear", "ntk", "parts")


def make_plan(rot, axes, inter, base, scaling="none", factor=1.0, length=1):
    lib = coreg.load()
    lib.coreg_set_error_mode(coreg.ERRORS_RECORD)
    r = coreg.Rotary()
    lib.ops_rotary_plan(r, rot, axes, inter, base, SCALINGS.index(scaling), factor, length)
    coreg.check(lib)
    return r


@pytest.mark.parametrize("rot,axes", [(2, 1), (4, 2), (64, 1), (64, 2), (96, 1), (100, 2), (256, 1)])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_plan_frequencies(rot, axes, scaling):
    """Turns per position to 2^-64 and the rounding of a long double power
    (2^-60 relative covers powl on both sides)."""
    for base, factor, length in ((10000.0, 8.0, 4096), (100.0, 2.5, 40)):
        r = make_plan(rot, axes, 1, base, scaling, factor, length)
        w, m = ref.frequencies(rot, axes, base, scaling, factor, length)
        assert (r.rot, r.axes, r.interleaved) == (rot, axes, 1)
        assert abs(r.mscale - m) <= 2.0 ** -23 * abs(m)
        turns = w / (2 * ref.PI)
        got = np.array([np.longdouble(int(v)) for v in r.step[:rot // 2]]) / np.longdouble(2.0) ** 64
        want = np.tile(turns, axes)
        assert (np.abs(got - want) <= want * np.longdouble(2.0) ** -58 + np.longdouble(2.0) ** -63).all()
        assert not any(r.step[rot // 2:])


def test_plan_refusals():
    for bad in ((3, 1, 0, 1e4), (0, 1, 0, 1e4), (258, 1, 0, 1e4), (6, 2, 0, 1e4), (8, 3, 0, 1e4),
                (8, 0, 0, 1e4), (8, 1, 0, 0.0), (8, 1, 0, -1.0), (8, 1, 0, float("nan")),
                (8, 1, 0, float("inf"))):
        with pytest.raises(coreg.CoregError, match="ops_rotary_plan"):
            make_plan(*bad)
    for scaling, factor, length in (("linear", 0.0, 1), ("ntk", -1.0, 1), ("parts", 2.0, 0),
                                    ("parts", float("nan"), 10)):
        with pytest.raises(coreg.CoregError, match="ops_rotary_plan"):
            make_plan(8, 1, 0, 1e4, scaling, factor, length)
    lib = coreg.load()
    lib.ops_rotary_plan(coreg.Rotary(), 8, 1, 0, 1e4, 4, 1.0, 1)
    with pytest.raises(coreg.CoregError, match="scaling 4"):
        coreg.check(lib)
    lib.ops_rotary_plan(C.POINTER(coreg.Rotary)(), 8, 1, 0, 1e4, 0, 1.0, 1)
    with pytest.raises(coreg.CoregError, match="no struct"):
        coreg.check(lib)


CASES = [
    # rows, nh, d, rot, axes, interleaved, scaling, X offset, X extra pitch, Y offset, Y extra
    (1, 1, 2, 2, 1, 0, "none", 0, 0, 0, 0),
    (1, 40, 128, 96, 1, 1, "parts", 0, 0, 0, 0),
    (3, 3, 7, 4, 1, 0, "linear", 1, 2, 3, 1),
    (3, 3, 7, 4, 2, 1, "ntk", 1, 2, 3, 1),
    (50, 8, 32, 32, 2, 0, "none", 0, 0, 0, 0),
    (50, 8, 32, 32, 2, 1, "none", 0, 0, 0, 0),
    (257, 16, 64, 64, 2, 0, "none", 0, 64, 0, 0),
    (100, 4, 80, 40, 1, 0, "none", 16, 16, 8, 8),
    (100, 4, 80, 40, 1, 1, "none", 16, 16, 8, 8),
    (61, 5, 73, 40, 1, 1, "ntk", 0, 0, 0, 0),
    (33, 2, 256, 256, 1, 0, "parts", 0, 0, 0, 0),
    (33, 2, 256, 256, 2, 1, "parts", 4, 4, 4, 4),
    (9, 48, 12, 12, 1, 0, "none", 0, 0, 0, 0),
    (1000, 1, 24, 8, 1, 1, "linear", 0, 0, 0, 0),
    (4, 3, 64, 32, 2, 0, "none", 1, 0, 0, 0),
]


def run(dev, t, case, inplace):
    rows, nh, d, rot, axes, inter, scaling, xo, xp, yo, yp = case
    T = TYPES[t]
    rng = np.random.default_rng(rows * 3 + d)
    x = rounded(rng.standard_normal((rows, nh * d)), T)
    pos = rng.integers(0, 5000, (rows, axes)).astype(np.int32)
    pos[0] = 2 ** 31 - 1
    if rows > 2:
        pos[1], pos[2] = -(2 ** 31), 0
    r = make_plan(rot, axes, inter, 10000.0, scaling, 4.0, 100)
    w, m = ref.frequencies(rot, axes, 10000.0, scaling, 4.0, 100)
    X = Rows(dev, rows, nh * d, T, x, off=xo, ld=nh * d + xp)
    Y = X if inplace else Rows(dev, rows, nh * d, T, off=yo, ld=nh * d + yp)
    Pb = dev.upload(pos)
    dev.lib.ops_rotary(dev.ops_p, r, rows, nh, d, X.opnd, Y.opnd, T, Pb.handle, 5)
    want = ref.rotary(x, pos.astype(np.int64) + 5, nh, d, rot, axes, inter, w, m)
    xh, mag = np.abs(x.astype(np.float64)).reshape(rows, nh, d), np.zeros((rows, nh, d))
    half = rot // 2
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, half), slice(half, rot))
    mag[..., a] = mag[..., b] = xh[..., a] + xh[..., b]
    mag = mag.reshape(rows, nh * d)
    # An angle of w |p| radians in the 64-bit long double of the reference is
    # itself off by up to |p| w 2^-62; the plan's by |p| 2^-64 turns.
    tol = m * mag * (12 * 2.0 ** -24 + 2.0 ** -30) + np.where(mag > 0, HALF_STEP[T], 0) * np.abs(want)
    close(Y.read(), want, tol)
    if not inplace:
        assert (X.read() == x).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotary(dev, case, t):
    run(dev, t, case, False)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotary_in_place(dev, case, t):
    run(dev, t, case, True)


@pytest.mark.gpu
@pytest.mark.parametrize("pos0", [0, 7, 2 ** 33])
def test_rotary_rows_as_positions(dev, pos0):
    """pos NULL: positions pos0 + row, beyond 32 bits too."""
    rows, nh, d, rot = 70, 2, 16, 16
    x = np.random.default_rng(1).standard_normal((rows, nh * d)).astype(np.float32)
    r = make_plan(rot, 1, 0, 100.0)
    w, _ = ref.frequencies(rot, 1, 100.0)
    X, Y = Rows(dev, rows, nh * d, F32, x), Rows(dev, rows, nh * d, F32)
    dev.lib.ops_rotary(dev.ops_p, r, rows, nh, d, X.opnd, Y.opnd, F32, None, pos0)
    pos = (pos0 + np.arange(rows, dtype=np.int64))[:, None]
    want = ref.rotary(x, pos, nh, d, rot, 1, 0, w)
    mag = np.abs(x).reshape(rows, nh, 2, 8).sum(2, keepdims=True).repeat(2, 2).reshape(rows, -1)
    # 2^34 positions: the step's 2^-64 turns make 2^-30, the reference's angle
    # of 2^34 radians in 64 bits about as much.
    close(Y.read(), want, mag * (13 * 2.0 ** -24 + 2 ** -27))


@pytest.mark.gpu
def test_rotary_of_separate_columns(dev):
    """Queries and keys of one qkv buffer: the keys turned into the place of
    the values' columns is refused, into separate columns of the same rows
    runs; infinities stay within their pair."""
    rows, nh, d = 40, 2, 8
    E = nh * d
    x = np.random.default_rng(2).standard_normal((rows, 3 * E)).astype(np.float32)
    x[5, 1] = np.inf
    r = make_plan(8, 1, 1, 100.0)
    w, _ = ref.frequencies(8, 1, 100.0)
    B = dev.upload(x)
    lib = dev.lib
    at = [coreg.Opnd(B.handle, i * E, 3 * E, 0, 0) for i in range(3)]
    lib.ops_rotary(dev.ops_p, r, rows, nh, d, at[0], at[2], F32, None, 0)
    got = B.read().reshape(rows, 3 * E)
    assert (got[:, :2 * E] == x[:, :2 * E]).all()
    keep = np.ones((rows, E), bool)
    keep[5, :2] = False
    with np.errstate(invalid="ignore"):
        want = ref.rotary(x[:, :E], np.arange(rows)[:, None], nh, d, 8, 1, 1, w)
    mag = np.abs(x[:, :E]).reshape(rows, E // 2, 2).sum(2).repeat(2, 1)
    close(got[:, 2 * E:][keep], want[keep], mag[keep] * 13 * 2.0 ** -24)
    lib.ops_rotary(dev.ops_p, r, rows, nh, d, at[0], coreg.Opnd(B.handle, E - 1, 3 * E, 0, 0), F32,
                   None, 0)
    with pytest.raises(coreg.CoregError, match="overlap"):
        coreg.check(lib)
