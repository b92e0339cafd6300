# SPDX-License-Identifier: Unlicense
"""What ops_quant_i8, ops_gemm_i8, ops_linear_i8, ops_rotary and
ops_groupnorm_cl refuse (CPU: every check comes before the first CUDA call,
so handles over host memory and an empty backend do), and the empty calls
that do nothing."""

import ctypes as C

import numpy as np
import pytest

import coreg

F32, BF16 = coreg.OPS_FP32, coreg.OPS_BF16
BIG = 1 << 16


class Host:
    def __init__(self):
        self.lib = coreg.load()
        self.lib.coreg_set_error_mode(coreg.ERRORS_RECORD)
        self.lib.coreg_clear_error()
        self.ocl = coreg.OclBackend()
        self.ocl.device = 77  # never to be reached
        self.ops = coreg.Ops()
        self.ops.ocl = C.pointer(self.ocl)
        self.o = C.pointer(self.ops)
        self.mem = np.zeros(32 * BIG + 64, np.uint8)
        self.base = (self.mem.ctypes.data + 63) // 64 * 64
        self.next = 0

    def buf(self, n=BIG, shift=0):
        at = self.base + self.next + shift
        self.next += BIG + 64
        return self.lib.ocl_wrap(at, n)

    def refuses(self, match, fn, *args):
        getattr(self.lib, fn)(self.o, *args)
        with pytest.raises(coreg.CoregError, match=match):
            coreg.check(self.lib)

    def runs_nothing(self, fn, *args):
        getattr(self.lib, fn)(self.o, *args)
        coreg.check(self.lib)


@pytest.fixture
def h():
    return Host()


def M(buf, ld, off=0, s0=0):
    return coreg.Opnd(buf, off, ld, s0, 0)


def test_quant_refusals(h):
    X, Q, S = h.buf(), h.buf(), h.buf()
    f = "ops_quant_i8"
    h.refuses("element type 2", f, 4, 8, M(X, 8), 2, M(Q, 16), S, 0)
    h.refuses("X is NULL", f, 4, 8, M(None, 8), F32, M(Q, 16), S, 0)
    h.refuses("Q is NULL", f, 4, 8, M(X, 8), F32, M(None, 16), S, 0)
    h.refuses("S is NULL", f, 4, 8, M(X, 8), F32, M(Q, 16), None, 0)
    h.refuses("X at offset 0, -1 rows", f, -1, 8, M(X, 8), F32, M(Q, 16), S, 0)
    h.refuses("leading dimension 7", f, 4, 8, M(X, 7), F32, M(Q, 16), S, 0)
    h.refuses("leading dimension 7", f, 4, 8, M(X, 8), F32, M(Q, 7), S, 0)
    h.refuses("leading dimension -8", f, 4, 8, M(X, -8), F32, M(Q, 16), S, 0)
    h.refuses("offset -1", f, 4, 8, M(X, 8, -1), F32, M(Q, 16), S, 0)
    h.refuses("passes its buffer", f, 4, 8, M(X, 8, BIG // 4 - 31), F32, M(Q, 16), S, 0)
    h.refuses("passes its buffer", f, BIG // 16 + 1, 8, M(X, 4096), F32, M(Q, 16), S, 0)
    h.refuses("passes its buffer", f, 4, 8, M(X, 8), F32, M(Q, 16, BIG), S, 0)
    h.refuses("passes its buffer", f, 4, 8, M(X, 8), F32, M(Q, 16), S, BIG // 4 - 3)
    h.refuses("passes its buffer", f, 4, 8, M(X, 8, 2 ** 62), F32, M(Q, 16), S, 0)
    h.refuses("passes its buffer", f, 2 ** 62, 8, M(X, 2 ** 31 - 1), F32, M(Q, 16), S, 0)
    h.refuses("not aligned", f, 4, 8, M(h.buf(1024, 2), 8), F32, M(Q, 16), S, 0)
    h.refuses("rows of 1073741825", f, 0, 2 ** 30 + 1, M(X, 8), F32, M(Q, 8), S, 0)
    h.refuses("overlaps", f, 4, 8, M(X, 8), F32, M(X, 8, 100), S, 0)
    h.refuses("overlaps", f, 4, 8, M(X, 8), F32, M(Q, 8), X, 3)
    h.refuses("overlaps", f, 4, 8, M(X, 8), F32, M(Q, 8), Q, 0)
    h.runs_nothing(f, 0, 8, M(X, 8), F32, M(Q, 16), S, 0)
    h.runs_nothing(f, 4, 0, M(X, 8), F32, M(Q, 16), S, 0)


def test_gemm_refusals(h):
    A, B, S, T, Cb, R = (h.buf() for _ in range(6))
    f = "ops_gemm_i8"

    def args(m=4, n=8, k=32, a=None, sa=S, b=None, sb=T, bias=None, c=None, t=F32, r=None, roff=0,
             act=0):
        return (m, n, k, a or M(A, 32), sa, b or M(B, 32), sb, bias, c or M(Cb, 8), t, r, roff,
                act, 0.0)

    h.refuses("-1 x 8 x 32", f, *args(m=-1))
    h.refuses("4 x -8", f, *args(n=-8))
    h.refuses("4 x 8 x -1", f, *args(k=-1))
    h.refuses("depth 0..131071", f, *args(k=131072))
    h.refuses("2147483647 x 8", f, *args(m=2 ** 31 - 1))
    h.refuses("4 x 2147483647", f, *args(n=2 ** 31 - 1))
    h.refuses("element type 7", f, *args(t=7))
    h.refuses("activation 6", f, *args(act=6))
    h.refuses("activation -1", f, *args(act=-1))
    h.refuses("A is NULL", f, *args(a=M(None, 32)))
    h.refuses("B is NULL", f, *args(b=M(None, 32)))
    h.refuses("C is NULL", f, *args(c=M(None, 32)))
    h.refuses("scales of A is NULL", f, *args(sa=None))
    h.refuses("scales of B is NULL", f, *args(sb=None))
    h.refuses("16-byte aligned", f, *args(a=M(A, 40)))
    h.refuses("16-byte aligned", f, *args(b=M(B, 33)))
    h.refuses("16-byte aligned", f, *args(a=M(A, 32, 8)))
    h.refuses("16-byte aligned", f, *args(b=M(h.buf(4096, 4), 32)))
    h.refuses("leading dimension 16", f, *args(a=M(A, 16)))
    h.refuses("leading dimension 7", f, *args(c=M(Cb, 7)))
    h.refuses("passes its buffer", f, *args(a=M(A, 32, BIG - 112)))
    h.refuses("passes its buffer", f, *args(n=8, sb=h.buf(28)))
    h.refuses("passes its buffer", f, *args(bias=h.buf(28)))
    h.refuses("passes its buffer", f, *args(sa=h.buf(12)))
    h.refuses("passes its buffer", f, *args(r=R, roff=BIG // 4 - 31))
    h.refuses("R at offset -1", f, *args(r=R, roff=-1))
    h.refuses("R and C overlap", f, *args(r=Cb, roff=3))
    h.refuses("overlaps an input", f, *args(c=M(A, 8)))
    h.refuses("overlaps an input", f, *args(c=M(S, 8)))
    h.refuses("overlaps an input", f, *args(bias=Cb))
    h.runs_nothing(f, *args(m=0))
    h.runs_nothing(f, *args(n=0))


def test_linear_refusals(h):
    X, W, S, Y, wk = (h.buf() for _ in range(5))
    f = "ops_linear_i8"
    need = h.lib.ops_linear_i8_bytes(40, 20)
    assert need == 160 + 40 * 32 and h.lib.ops_linear_i8_bytes(0, 20) == 0

    def args(m=40, k=20, n=8, x=None, xt=F32, w=None, y=None, yt=F32, r=None, act=0, work=wk):
        return (m, k, n, x or M(X, 20), xt, w or M(W, 32), S, None, y or M(Y, 8), yt, r, 0, act,
                0.0, work)

    h.refuses("element type 3", f, *args(xt=3))
    h.refuses("element type -1", f, *args(yt=-1))
    h.refuses("X is NULL", f, *args(x=M(None, 20)))
    h.refuses("passes its buffer", f, *args(x=M(X, 20, BIG // 4)))
    h.refuses("16-byte aligned", f, *args(w=M(W, 20)))
    h.refuses("work buffer is NULL", f, *args(work=None))
    h.refuses("work buffer .* passes", f, *args(work=h.buf(need - 1)))
    h.refuses("work buffer is not 16-byte", f, *args(work=h.buf(4096, 8)))
    h.refuses("overlaps", f, *args(work=X))
    h.refuses("overlaps", f, *args(work=Y))
    h.refuses("overlaps", f, *args(work=wk, r=wk))
    h.refuses("overlaps", f, *args(y=M(X, 8)))
    h.runs_nothing(f, *args(m=0, work=None))
    h.runs_nothing(f, *args(n=0, work=None))


def test_rotary_refusals(h):
    X, Y, pos = h.buf(), h.buf(), h.buf()
    r, two, f = coreg.Rotary(), coreg.Rotary(), "ops_rotary"
    h.lib.ops_rotary_plan(r, 8, 1, 0, 100.0, 0, 1.0, 1)
    h.lib.ops_rotary_plan(two, 8, 2, 0, 100.0, 0, 1.0, 1)

    def args(plan=r, rows=4, nh=2, d=10, x=None, y=None, t=F32, p=pos):
        return (plan, rows, nh, d, x or M(X, 20), y or M(Y, 20), t, p, 0)

    h.refuses("no frequencies", f, *args(plan=coreg.Rotary()))
    h.refuses("no frequencies", f, *args(plan=None))
    for rot, axes in ((3, 1), (300, 1), (8, 3), (6, 2), (-2, 1)):
        bad = coreg.Rotary()
        bad.rot, bad.axes = rot, axes
        h.refuses("no frequencies", f, *args(plan=bad))
    h.refuses("8 rotated", f, *args(d=7))
    h.refuses("-2 heads", f, *args(nh=-2))
    h.refuses("heads", f, *args(nh=2 ** 30))
    h.refuses("heads", f, *args(nh=2 ** 27, d=16))
    h.refuses("element type 5", f, *args(t=5))
    h.refuses("two axes need positions", f, *args(plan=two, p=None))
    h.refuses("X is NULL", f, *args(x=M(None, 20)))
    h.refuses("Y is NULL", f, *args(y=M(None, 20)))
    h.refuses("leading dimension 19", f, *args(x=M(X, 19)))
    h.refuses("leading dimension 19", f, *args(y=M(Y, 19)))
    h.refuses("-4 rows", f, *args(rows=-4))
    h.refuses("passes its buffer", f, *args(rows=BIG))
    h.refuses("positions .* passes", f, *args(plan=two, p=h.buf(28)))
    h.refuses("overlap", f, *args(y=M(X, 20, 4)))
    h.refuses("overlap", f, *args(y=M(X, 24)))
    h.refuses("overlaps the positions", f, *args(y=M(pos, 20)))
    h.runs_nothing(f, *args(rows=0))
    h.runs_nothing(f, *args(nh=0))


def test_groupnorm_refusals(h):
    X, Y, G = h.buf(), h.buf(), h.buf()
    f = "ops_groupnorm_cl"

    def args(n=2, hw=9, c=12, groups=3, x=None, xt=F32, y=None, yt=F32, g=None, b=None, eps=1e-5,
             act=0, work=None):
        return (n, hw, c, groups, x or M(X, 12, 0, 108), xt, y or M(Y, 12, 0, 108), yt, g, b, eps,
                act, 0.0, work)

    h.refuses("element type 2", f, *args(xt=2))
    h.refuses("element type 2", f, *args(yt=2))
    h.refuses("activation 9", f, *args(act=9))
    h.refuses("in 5 groups", f, *args(groups=5))
    h.refuses("in 0 groups", f, *args(groups=0))
    h.refuses("-1 maps", f, *args(n=-1))
    h.refuses("of -9 x", f, *args(hw=-9))
    h.refuses("eps", f, *args(eps=-1.0))
    h.refuses("eps", f, *args(eps=float("nan")))
    h.refuses("gamma without beta", f, *args(g=G))
    h.refuses("gamma without beta", f, *args(b=G))
    h.refuses("gamma .* passes", f, *args(g=h.buf(44), b=G))
    h.refuses("X is NULL", f, *args(x=M(None, 12)))
    h.refuses("Y is NULL", f, *args(y=M(None, 12)))
    h.refuses("leading dimension 11", f, *args(x=M(X, 11, 0, 108)))
    h.refuses("passes its buffer", f, *args(hw=BIG))
    h.refuses("pass the buffer", f, *args(x=M(X, 12, 0, BIG)))
    h.refuses("images 107 elements apart", f, *args(y=M(Y, 12, 0, 107)))
    h.refuses("images -1 elements apart", f, *args(x=M(X, 12, 0, -1)))
    h.refuses("overlaps", f, *args(y=M(X, 12, 0, 120)))
    h.refuses("overlaps", f, *args(y=M(X, 12, 4, 108)))
    h.refuses("overlaps", f, *args(y=M(X, 12, 0, 108), yt=BF16))
    h.refuses("overlaps", f, *args(g=Y, b=G))
    need = h.lib.ops_groupnorm_cl_bytes(2, 9, 12, 3)
    assert need > 0 and h.lib.ops_groupnorm_cl_bytes(0, 9, 12, 3) == 0
    h.refuses("work buffer is NULL", f, *args())
    h.refuses("work buffer .* passes", f, *args(work=h.buf(need - 1)))
    h.refuses("work buffer is not 16-byte", f, *args(work=h.buf(BIG, 8)))
    h.refuses("work buffer overlaps", f, *args(work=X))
    h.refuses("work buffer overlaps", f, *args(work=Y))
    h.refuses("maps of", f, *args(n=65536))
    h.refuses("maps of", f, *args(hw=2 ** 30 + 1))
    h.runs_nothing(f, *args(n=0))
    h.runs_nothing(f, *args(hw=0))
    h.runs_nothing(f, *args(c=0, groups=1))
