# SPDX-License-Identifier: Unlicense
"""ops_quant_i8, ops_gemm_i8 and ops_linear_i8 against their plain forms in
64 bits (GPU). The quantised values and scales are whole numbers and single
roundings: they have to be equal.

Products: the integer sum is exact; its conversion, the two scales and the
bias are at most 5 roundings of 2^-24 of the terms' magnitude; the
activation (Lipschitz constant below 1.2, its own error below 4 steps of its
argument's magnitude, and for SiLU's fast exponential |v| 2^-22 more at
|v| <= 30 relative to the result, which is at most |v|) stays within 32 such
steps of the magnitude; the residual adds one of the sum, and the store half
a step of the type."""

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from typed_ops import BF16, F32, HALF_STEP, Rows, close, rounded

TYPES = {"f32": F32, "bf16": BF16}


def tokens(rng, rows, C, t):
    x = rng.standard_normal((rows, C)) * np.exp(rng.standard_normal((rows, 1)))
    x[:, rng.random(C) < 0.02] *= 20
    return rounded(x, t)


def quant(dev, X, t, rows, C, qoff=0, qld=None):
    Q = Rows(dev, rows, C, None, off=qoff, ld=C if qld is None else qld)
    S = Rows(dev, rows, 1, F32, off=3)
    dev.lib.ops_quant_i8(dev.ops_p, rows, C, X.opnd, t, Q.opnd, S.handle, 3)
    return Q.read(), S.read()[:, 0]


QUANT = [
    # rows, C, X offset, X pitch, Q offset, Q pitch
    (1, 1, 0, 1, 0, 1),
    (3, 16, 0, 16, 0, 16),
    (5, 17, 1, 19, 3, 21),
    (2, 127, 0, 128, 0, 128),
    (33, 256, 8, 264, 16, 272),
    (9, 1024, 0, 1024, 0, 1024),
    (7, 1000, 4, 1004, 0, 1008),
    (4, 4096, 0, 4096, 0, 4096),
    (3, 5000, 0, 5008, 0, 5008),
    (2, 8192, 0, 8192, 0, 8192),
    (2, 20001, 0, 20001, 5, 20003),
    (1601, 96, 0, 96, 0, 96),
    (1, 40000, 0, 40000, 0, 40000),
    # Rows aligned to two values, or to one: short, and long beyond the registers.
    (35, 30, 2, 30, 0, 32),
    (4, 3758, 0, 3758, 0, 3760),
    (3, 4101, 1, 4101, 0, 4112),
    (2, 9003, 2, 9006, 2, 9006),
    (2, 5001, 3, 5003, 1, 5001),
]


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", QUANT, ids=str)
def test_quant_equals(dev, shape, t):
    rows, C, xo, xl, qo, ql = shape
    rng = np.random.default_rng(rows * 7 + C)
    x = tokens(rng, rows, C, TYPES[t])
    X = Rows(dev, rows, C, TYPES[t], x, off=xo, ld=xl)
    q, s = quant(dev, X, TYPES[t], rows, C, qo, ql)
    wq, ws = ref.quant_i8(x)
    assert (s == ws).all()
    assert (q == wq).all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("C", [5, 48, 1024, 9000, 26, 4098, 4097])
def test_quant_edge_rows(dev, C, t):
    """Zeros, infinities, NaN, the type's extremes, denormal rows and exact
    ties (multiples of half a scale)."""
    T = TYPES[t]
    rng = np.random.default_rng(C)
    big = np.float32(3.3e38)
    x = np.zeros((14, C), np.float32)
    x[1] = -0.0
    x[2, C // 2] = np.inf
    x[3] = rng.standard_normal(C)
    x[3, C - 1] = np.nan
    x[4] = rng.standard_normal(C)
    x[4, 0] = -np.inf
    x[5] = big * rng.uniform(-1, 1, C)
    x[5, 1] = -big
    x[6] = 1e-45 * rng.integers(-200, 201, C)
    x[7] = 1e-40 * rng.standard_normal(C)
    x[8] = 1e-37 * rng.standard_normal(C)
    x[9] = 127.0
    x[10] = rng.integers(-127, 127, C) + 0.5  # ties: the scale below is exactly 1
    x[10, 0] = 127.0
    x[11] = (rng.integers(-31, 31, C) + 0.5) * 2.0 ** -60
    x[11, 0] = 127 * 2.0 ** -60
    x[12, C - 1] = 1e-45
    x[13] = 2.0 ** -91 * rng.standard_normal(C)
    x = rounded(x, T)
    q, s = quant(dev, Rows(dev, 14, C, T, x), T, 14, C)
    wq, ws = ref.quant_i8(x)
    np.testing.assert_array_equal(s, ws)
    np.testing.assert_array_equal(q, wq)


def i8_rows(dev, q, off=0, extra=0):
    K = q.shape[1]
    return Rows(dev, q.shape[0], K, None, q, off=off, ld=(K + 15) // 16 * 16 + extra)


def operands(rng, M, N, K):
    a = rng.integers(-127, 128, (M, K)).astype(np.int8)
    b = rng.integers(-128, 128, (N, K)).astype(np.int8)
    sa = np.exp(rng.standard_normal(M) - 4).astype(np.float32)
    sb = np.exp(rng.standard_normal(N) - 5).astype(np.float32)
    return a, sa, b, sb, rng.standard_normal(N).astype(np.float32)


def tolerance(want, mag, res, t):
    tol = 32 * 2.0 ** -24 * mag + HALF_STEP[t] * np.abs(want) + 1e-37
    return tol + (2.0 ** -24 * (np.abs(want) + np.abs(res)) if res is not None else 0)


GEMM = [
    # M, N, K, extra pitch of A and B, C offset, C pitch beyond N
    (1, 1, 1, 0, 0, 0),
    (1, 1000, 1024, 0, 0, 0),
    (2, 17, 40, 16, 1, 3),
    (7, 64, 129, 0, 0, 0),
    (8, 333, 2000, 0, 0, 0),
    (9, 128, 64, 0, 8, 8),
    (16, 96, 4096, 0, 0, 0),
    (17, 100, 300, 0, 0, 0),
    (31, 2049, 77, 0, 0, 1),
    (32, 64, 512, 0, 0, 0),
    (33, 65, 513, 16, 0, 0),
    (64, 256, 1024, 0, 0, 0),
    (100, 31, 100, 0, 0, 0),
    (127, 129, 127, 0, 0, 0),
    (128, 128, 128, 0, 0, 0),
    (129, 257, 131, 32, 4, 4),
    (200, 1000, 1111, 0, 0, 0),
    (256, 256, 4096, 0, 0, 0),
    (257, 513, 640, 0, 0, 0),
    (700, 24, 48, 0, 0, 0),
    (1000, 777, 333, 0, 0, 7),
    (513, 16, 9000, 0, 0, 0),
    (2, 7000, 700, 0, 0, 0),
    (3, 6145, 530, 0, 0, 0),
    (8, 6144, 96, 0, 0, 0),
    (9, 4096, 200, 16, 1, 1),
    (16, 4100, 144, 0, 0, 0),
    (300, 1, 200, 0, 0, 0),
    # Wide tiles, and deep ones by CTA pairs: one tile and more of a CTA or pair,
    # ragged rows, columns and depths.
    (1000, 4096, 256, 0, 0, 0),
    (1025, 3850, 130, 16, 0, 2),
    (2000, 4090, 700, 0, 0, 0),
    (700, 4096, 2048, 0, 0, 0),
    (1025, 3850, 2100, 16, 0, 2),
    (2600, 4352, 2050, 0, 0, 0),
    (5000, 2100, 2064, 0, 1, 4),
    (129, 9000, 4000, 0, 0, 0),
    # Pairs whose second half has no rows of A, or of B.
    (2600, 4160, 2048, 0, 0, 0),
    # Few tiles of a deep product, the depth split; the narrowest and shallowest.
    (3, 130, 8200, 0, 0, 0),
    (24, 8192, 520, 0, 0, 0),
    (32, 900, 4097, 16, 4, 4),
    (33, 1000, 4096, 0, 0, 0),
    (10, 1, 700, 0, 0, 0),
    (48, 2100, 1500, 0, 1, 3),
    (129, 257, 4097, 0, 2, 2),
    (256, 300, 3333, 0, 0, 0),
    (777, 1000, 4100, 0, 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", GEMM, ids=str)
def test_gemm(dev, shape, t):
    M, N, K, extra, co, cp = shape
    T = TYPES[t]
    rng = np.random.default_rng(M * 31 + N * 7 + K)
    a, sa, b, sb, bias = operands(rng, M, N, K)
    A, B = i8_rows(dev, a, 16, extra), i8_rows(dev, b, 0, extra)
    SA, SB, BI = dev.upload(sa), dev.upload(sb), dev.upload(bias)
    C = Rows(dev, M, N, T, off=co, ld=N + cp)
    dev.lib.ops_gemm_i8(dev.ops_p, M, N, K, A.opnd, SA.handle, B.opnd, SB.handle, BI.handle,
                        C.opnd, T, None, 0, 0, 0.1)
    want, mag = ref.gemm_i8(a, sa, b, sb, bias)
    close(C.read(), want, tolerance(want, mag, None, T))
    assert dev.lib.coreg_tc_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", ref.ACTS)
@pytest.mark.parametrize("shape", [(2, 200, 272), (5, 200, 272), (300, 200, 272), (257, 9000, 2050),
                                   (13, 203, 2100), (100, 300, 2100)], ids=str)
def test_gemm_activations_residual(dev, shape, kind, t):
    """Each activation, without a bias, with a residual of its own and in place."""
    (M, N, K), T = shape, TYPES[t]
    rng = np.random.default_rng(M + len(kind))
    a, sa, b, sb, _ = operands(rng, M, N, K)
    res = rounded(rng.standard_normal((M, N)), T)
    A, B, SA, SB = i8_rows(dev, a), i8_rows(dev, b), dev.upload(sa), dev.upload(sb)
    want, mag = ref.gemm_i8(a, sa, b, sb, None, kind, 0.1, res)
    R, C = Rows(dev, M, N, T, res, off=8, ld=N + 8), Rows(dev, M, N, T, ld=N + 8)
    D = Rows(dev, M, N, T, res, ld=N)
    for out, r, roff in ((C, R.handle, 8), (D, D.handle, 0)):
        dev.lib.ops_gemm_i8(dev.ops_p, M, N, K, A.opnd, SA.handle, B.opnd, SB.handle, None,
                            out.opnd, T, r, roff, ref.ACTS.index(kind), 0.1)
        close(out.read(), want, tolerance(want, mag, res, T))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 12, 20, 140])
def test_gemm_largest_sums(dev, M):
    """The deepest product of the largest values: 2^31 - 2^14, exact; and K = 0."""
    N, K = 40, coreg.I8_MAX_K
    a = np.full((M, K), -128, np.int8)
    b = np.full((N, K), -128, np.int8)
    b[1::2] = 127
    one = np.ones(max(M, N), np.float32)
    A, B, S = i8_rows(dev, a), i8_rows(dev, b), dev.upload(one)
    C = Rows(dev, M, N, F32)
    dev.lib.ops_gemm_i8(dev.ops_p, M, N, K, A.opnd, S.handle, B.opnd, S.handle, None, C.opnd, F32,
                        None, 0, 0, 0.0)
    want = np.where(np.arange(N) % 2, -128.0 * 127 * K, 128.0 * 128 * K).astype(np.float32)
    assert (C.read() == want).all()
    bias = dev.upload(np.arange(N, dtype=np.float32) - 7)
    dev.lib.ops_gemm_i8(dev.ops_p, M, N, 0, A.opnd, S.handle, B.opnd, S.handle, bias.handle,
                        C.opnd, F32, None, 0, coreg.ACT_RELU, 0.0)
    assert (C.read() == np.maximum(np.arange(N) - 7, 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ref.ACTS)
@pytest.mark.parametrize("N,K", [(201, 4200), (1030, 2048), (4097, 1000), (4160, 2048), (301, 0)])
def test_gemm_rows_do_not_depend_on_their_number(dev, N, K, kind):
    """A row's results are the same bits whichever kernel its product takes: by
    the number of rows the streaming ones, split depths, tiles and pairs."""
    M = 2600
    rng = np.random.default_rng(N + K)
    a, sa, b, sb, bias = operands(rng, M, N, K)
    A, B = i8_rows(dev, a, extra=16), i8_rows(dev, b, extra=16)
    SA, SB, BI = dev.upload(sa), dev.upload(sb), dev.upload(bias)
    R = Rows(dev, M, N, F32, rng.standard_normal((M, N)).astype(np.float32))
    got = {}
    for m in (1, 2, 8, 9, 33, 128, 200, 700, M):
        C = Rows(dev, m, N, F32)
        dev.lib.ops_gemm_i8(dev.ops_p, m, N, K, A.opnd, SA.handle, B.opnd, SB.handle, BI.handle,
                            C.opnd, F32, R.handle, 0, ref.ACTS.index(kind), 0.1)
        got[m] = C.read()
    for m, c in got.items():
        assert (c == got[M][:m]).all(), m


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gelu", "silu"])
@pytest.mark.parametrize("rows,K,N", [(1, 300, 5001), (1, 9000, 70), (2, 4000, 333),
                                      (8, 1024, 8191), (8, 1100, 200), (9, 500, 77),
                                      (40, 2048, 130), (3, 0, 33)])
def test_linear_is_quant_then_gemm(dev, rows, K, N, kind):
    """Bit for bit, whether or not the layer is one launch."""
    rng = np.random.default_rng(rows + K + N)
    x = tokens(rng, rows, K, F32) if K else np.zeros((rows, 0))
    qw, sw = ref.quant_i8(rng.standard_normal((N, K))) if K else (np.zeros((N, 0)), np.ones(N))
    X, W = Rows(dev, rows, K, F32, x, ld=max(K, 1)), i8_rows(dev, qw.astype(np.int8), extra=16)
    SW, BI = dev.upload(sw), dev.upload(rng.standard_normal(N).astype(np.float32))
    Q = Rows(dev, rows, K, None, ld=(K + 15) // 16 * 16 + 16)
    S = dev.upload(np.ones(rows, np.float32))
    Y, Z = Rows(dev, rows, N, F32), Rows(dev, rows, N, F32)
    need = dev.lib.ops_linear_i8_bytes(rows, K)
    work = dev.alloc(need) if need else None
    act = ref.ACTS.index(kind)
    dev.lib.ops_linear_i8(dev.ops_p, rows, K, N, X.opnd, F32, W.opnd, SW.handle, BI.handle, Y.opnd,
                          F32, None, 0, act, 0.0, coreg.handle(work))
    dev.lib.ops_quant_i8(dev.ops_p, rows, K, X.opnd, F32, Q.opnd, S.handle, 0)
    dev.lib.ops_gemm_i8(dev.ops_p, rows, N, K, Q.opnd, S.handle, W.opnd, SW.handle, BI.handle,
                        Z.opnd, F32, None, 0, act, 0.0)
    assert (Y.read() == Z.read()).all()


@pytest.mark.gpu
def test_gemm_single_rows_of_any_pitch(dev):
    """A pitch that a single row of weights or tokens does not have is not used."""
    K = 100
    rng = np.random.default_rng(1)
    for M, N in ((40, 1), (1, 40)):
        a, sa, b, sb, _ = operands(rng, M, N, K)
        A, B, SA, SB = i8_rows(dev, a), i8_rows(dev, b), dev.upload(sa), dev.upload(sb)
        C = Rows(dev, M, N, F32)
        oa, ob = A.opnd, B.opnd
        (ob if N == 1 else oa).ld = -7
        dev.lib.ops_gemm_i8(dev.ops_p, M, N, K, oa, SA.handle, ob, SB.handle, None, C.opnd, F32,
                            None, 0, 0, 0.0)
        want, mag = ref.gemm_i8(a, sa, b, sb)
        close(C.read(), want, tolerance(want, mag, None, F32))


LINEAR = [
    # rows, in, out, X offset, X pitch beyond in
    (1, 1, 3, 0, 0),
    (1, 1024, 4096, 0, 0),
    (2, 1000, 50, 0, 0),
    (5, 37, 129, 3, 2),
    (1, 16384, 33, 0, 0),
    (1, 16385, 33, 0, 0),
    (2, 515, 40, 1, 0),
    (3, 4099, 70, 0, 0),
    (4, 4096, 130, 0, 1),
    (8, 4096, 256, 0, 0),
    (9, 1500, 5000, 0, 4),
    (16, 1024, 16, 0, 0),
    (16, 512, 512, 8, 8),
    (17, 5000, 64, 0, 0),
    (32, 2048, 100, 0, 0),
    (33, 48, 48, 0, 0),
    (130, 1024, 300, 0, 0),
    (1601, 160, 96, 0, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("xt", TYPES)
@pytest.mark.parametrize("yt", TYPES)
@pytest.mark.parametrize("shape", LINEAR, ids=str)
def test_linear(dev, shape, xt, yt):
    """Quantised exactly as by ops_quant_i8, so the product's bound holds for
    the layer; a row with a NaN makes its own outputs NaN and no others."""
    rows, K, N, xo, xp = shape
    T = TYPES[yt]
    rng = np.random.default_rng(rows + K + N)
    x = tokens(rng, rows, K, TYPES[xt])
    if rows > 4:
        x[2] = 0
        x[3, K // 3] = np.nan
    w = rng.standard_normal((N, K)).astype(np.float32)
    qw, sw = ref.quant_i8(w)
    bias = rng.standard_normal(N).astype(np.float32)
    res = rounded(rng.standard_normal((rows, N)), T)
    X, W = Rows(dev, rows, K, TYPES[xt], x, off=xo, ld=K + xp), i8_rows(dev, qw)
    SW, BI = dev.upload(sw), dev.upload(bias)
    Y = Rows(dev, rows, N, T, res)
    need = dev.lib.ops_linear_i8_bytes(rows, K)
    work = dev.alloc(need) if need else None
    dev.lib.ops_linear_i8(dev.ops_p, rows, K, N, X.opnd, TYPES[xt], W.opnd, SW.handle, BI.handle,
                          Y.opnd, T, Y.handle, 0, coreg.ACT_GELU, 0.0, coreg.handle(work))
    q, s = ref.quant_i8(x)
    want, mag = ref.gemm_i8(q, s, qw, sw, bias, "gelu", 0, res)
    close(Y.read(), want, tolerance(want, mag, res, T))
    assert dev.lib.coreg_tc_status() == 0
