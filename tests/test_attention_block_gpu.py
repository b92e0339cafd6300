# SPDX-License-Identifier: Unlicense
"""The typed operations of ops_b200.h together, as an attention block over a
channels-last feature map runs them (GPU): group norm and SiLU, the 8-bit
qkv product, rotary positions of queries and keys at their row and column,
attention, the 8-bit output layer onto the map; and the ways a program calls
them: captured into a CUDA graph and replayed on new data, on two backends
at once, and after a product has written what the next one reads.

The chain's bound: every step is checked on its own elsewhere; here the
whole is held to 2e-2 of its norm, ten times the quantisation error of the
two layers (1 / 127 / sqrt(12) of the largest value a row holds, about 4 rms:
1e-2 per element before the sums over 128 terms average it)."""

import ctypes as C

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from oracle.ops_ref import attention as ref_attention
from typed_ops import BF16, F32, rounded

H, W, D, HEADS, GROUPS = 13, 17, 128, 2, 8
N, HD = H * W, D // HEADS


class Block:
    """The block's weights, plan and buffers on one device, and its calls."""

    def __init__(self, dev, seed=0):
        self.dev, rng = dev, np.random.default_rng(seed)
        lib, o = dev.lib, dev.ops_p
        self.wqkv = (rng.standard_normal((3 * D, D)) / np.sqrt(D)).astype(np.float32)
        self.wo = (rng.standard_normal((D, D)) / np.sqrt(D)).astype(np.float32)
        self.g, self.b, self.bqkv, self.bo = (
            (m + 0.2 * rng.standard_normal(n)).astype(np.float32)
            for m, n in ((1, D), (0, D), (0, 3 * D), (0, D)))
        self.pos = np.stack(np.mgrid[:H, :W], -1).reshape(N, 2).astype(np.int32)
        up = dev.upload
        self.G, self.B, self.BQ, self.BO, self.P = map(up, (self.g, self.b, self.bqkv, self.bo,
                                                             self.pos))
        self.QW, self.SW = [], []
        for w in (self.wqkv, self.wo):
            Wf, Q, S = up(w), dev.alloc(w.shape[0] * D), dev.zeros(w.shape[0])
            lib.ops_quant_i8(o, w.shape[0], D, coreg.Opnd(Wf.handle, 0, D, 0, 0), F32,
                             coreg.Opnd(Q.handle, 0, D, 0, 0), S.handle, 0)
            dev.finish()
            self.QW.append(Q)
            self.SW.append(S)
        self.plan = coreg.Rotary()
        lib.ops_rotary_plan(self.plan, HD, 2, 0, 100.0, coreg.ROTARY_PLAIN, 1.0, 1)
        self.gw = dev.alloc(lib.ops_groupnorm_cl_bytes(1, N, D, GROUPS))
        self.lw = dev.alloc(lib.ops_linear_i8_bytes(N, D))
        self.X, self.Y = dev.zeros(N * D), dev.zeros(N * D)
        self.T = dev.alloc(N * D * 2)
        self.QKV, self.O = dev.zeros(N * 3 * D), dev.zeros(N * D)

    def run(self):
        lib, o, m = self.dev.lib, self.dev.ops_p, coreg.Opnd
        lib.ops_groupnorm_cl(o, 1, N, D, GROUPS, m(self.X.handle, 0, D, 0, 0), F32,
                             m(self.T.handle, 0, D, 0, 0), BF16, self.G.handle, self.B.handle,
                             1e-5, coreg.ACT_SILU, 0.0, self.gw.handle)
        lib.ops_linear_i8(o, N, D, 3 * D, m(self.T.handle, 0, D, 0, 0), BF16,
                          m(self.QW[0].handle, 0, D, 0, 0), self.SW[0].handle, self.BQ.handle,
                          m(self.QKV.handle, 0, 3 * D, 0, 0), F32, None, 0, 0, 0.0,
                          self.lw.handle)
        # Queries and keys: 2 HEADS heads side by side, in place.
        qk = m(self.QKV.handle, 0, 3 * D, 0, 0)
        lib.ops_rotary(o, self.plan, N, 2 * HEADS, HD, qk, qk, F32, self.P.handle, 0)
        lib.ops_attention_qkv(o, self.QKV.handle, N, D, HEADS, 1 / np.sqrt(HD), self.O.handle)
        lib.ops_linear_i8(o, N, D, D, m(self.O.handle, 0, D, 0, 0), F32,
                          m(self.QW[1].handle, 0, D, 0, 0), self.SW[1].handle, self.BO.handle,
                          m(self.Y.handle, 0, D, 0, 0), F32, self.X.handle, 0, 0, 0.0,
                          self.lw.handle)

    def want(self, x):
        t = rounded(ref.groupnorm(x[None], GROUPS, self.g, self.b, kind="silu")[0], BF16)
        qkv, _ = ref.gemm_i8(*ref.quant_i8(t), *ref.quant_i8(self.wqkv), self.bqkv)
        w, _ = ref.frequencies(HD, 2, 100.0)
        qkv[:, :2 * D] = ref.rotary(qkv[:, :2 * D], self.pos, 2 * HEADS, HD, HD, 2, 0, w)
        q = qkv.astype(np.float32)
        a = ref_attention(q[:, :D], q[:, D:2 * D], q[:, 2 * D:], N, N, HEADS, HD,
                          np.float32(1 / np.sqrt(HD)))
        y, _ = ref.gemm_i8(*ref.quant_i8(a), *ref.quant_i8(self.wo), self.bo)
        return x + y


def maps(seed):
    return np.random.default_rng(seed).standard_normal((N, D)).astype(np.float32)


def near(got, want):
    assert np.linalg.norm(got - want) <= 2e-2 * np.linalg.norm(want)


@pytest.mark.gpu
@pytest.mark.parametrize("prec", [coreg.OPS_FP32, coreg.OPS_BF16], ids=["fp32", "bf16"])
def test_block(prec):
    dev = coreg.Device(0, precision=prec)
    blk, x = Block(dev), maps(1)
    blk.X.write(x)
    blk.run()
    got = blk.Y.read().reshape(N, D)
    near(got, blk.want(x))
    assert dev.lib.coreg_tc_status() == 0
    # The same inputs give the same bits.
    blk.run()
    assert (blk.Y.read().reshape(N, D) == got).all()
    dev.close()


@pytest.mark.gpu
def test_block_captured_and_replayed():
    """One capture, replayed on new contents of its input, between eager runs
    of the same block."""
    rt = C.CDLL("libcudart.so.12")
    dev = coreg.Device(0)
    blk = Block(dev)
    eager = []
    for seed in (1, 2, 3):
        blk.X.write(maps(seed))
        blk.run()
        eager.append(blk.Y.read())
    st, graph, exe = C.c_void_p(dev.ocl.queue), C.c_void_p(), C.c_void_p()
    assert rt.cudaStreamBeginCapture(st, 1) == 0  # thread-local
    blk.run()
    coreg.check(dev.lib)
    assert rt.cudaStreamEndCapture(st, C.byref(graph)) == 0
    assert rt.cudaGraphInstantiate(C.byref(exe), graph, 0) == 0
    for turn in range(2):
        for seed in (3, 1, 2):
            blk.X.write(maps(seed))
            blk.Y.write(np.zeros(N * D, np.float32))
            assert rt.cudaGraphLaunch(exe, st) == 0
            assert rt.cudaGraphLaunch(exe, st) == 0
            assert (blk.Y.read() == eager[seed - 1]).all()
        blk.X.write(maps(2))
        blk.run()
        assert (blk.Y.read() == eager[1]).all()
    assert rt.cudaGraphExecDestroy(exe) == 0 and rt.cudaGraphDestroy(graph) == 0
    dev.close()


FIRST_CALL = """
import sys
sys.path[:0] = {path!r}
import ctypes as C
import numpy as np
import coreg
from oracle import ops_b200_ref as ref
rt = C.CDLL("libcudart.so.12")
dev = coreg.Device(0)
lib, o, m = dev.lib, dev.ops_p, coreg.Opnd
rng = np.random.default_rng(0)
# Every kind of launch: a whole-device team, a cluster team, tensor cores,
# streamed weights, the quantiser, the rotation.
maps = [(2, 260000, 64), (1, 500, 64)]
xs = [rng.standard_normal(s).astype(np.float32) for s in maps]
X = [dev.upload(x) for x in xs]
Y = [dev.zeros(x.size) for x in xs]
work = [dev.alloc(lib.ops_groupnorm_cl_bytes(*s, 8)) for s in maps]
M, K = 200, 128
t = rng.standard_normal((M, K)).astype(np.float32)
qw, sw = ref.quant_i8(rng.standard_normal((K, K)))
T, Q, S, QW, SW, Z, R = (dev.upload(t), dev.alloc(M * K), dev.zeros(M), dev.upload(qw),
                         dev.upload(sw), dev.zeros(M * K), dev.zeros(M * K))
P = coreg.Rotary()
lib.ops_rotary_plan(P, 64, 1, 1, 100.0, 0, 1.0, 1)
st, graph, exe = C.c_void_p(dev.ocl.queue), C.c_void_p(), C.c_void_p()
assert rt.cudaStreamBeginCapture(st, 1) == 0
for x, y, w, s in zip(X, Y, work, maps):
    lib.ops_groupnorm_cl(o, *s, 8, m(x.handle, 0, 64, s[1] * 64, 0), 0,
                         m(y.handle, 0, 64, s[1] * 64, 0), 0, None, None, 1e-5, 0, 0.0, w.handle)
lib.ops_quant_i8(o, M, K, m(T.handle, 0, K, 0, 0), 0, m(Q.handle, 0, K, 0, 0), S.handle, 0)
for rows in (M, 5, 1):
    lib.ops_gemm_i8(o, rows, K, K, m(Q.handle, 0, K, 0, 0), S.handle, m(QW.handle, 0, K, 0, 0),
                    SW.handle, None, m(Z.handle, 0, K, 0, 0), 0, None, 0, 0, 0.0)
lib.ops_rotary(o, P, M, 2, 64, m(Z.handle, 0, K, 0, 0), m(R.handle, 0, K, 0, 0), 0, None, 0)
coreg.check(lib)
assert rt.cudaStreamEndCapture(st, C.byref(graph)) == 0
assert rt.cudaGraphInstantiate(C.byref(exe), graph, 0) == 0
for turn in range(3):
    assert rt.cudaGraphLaunch(exe, st) == 0
for x, y in zip(xs, Y):
    want = ref.groupnorm(x, 8)
    assert np.abs(y.read().reshape(x.shape) - want).max() < 1e-4
z, _ = ref.gemm_i8(*ref.quant_i8(t), qw, sw)
w, _ = ref.frequencies(64, 1, 100.0)
want = ref.rotary(z, np.arange(M)[:, None], 2, 64, 64, 1, 1, w)
assert np.abs(R.read().reshape(M, K) - want).max() < 1e-4 * np.abs(want).max()
print("captured first")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_captured():
    """A process whose first call of every entry point is the captured one."""
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    code = FIRST_CALL.format(path=[str(root), str(root / "i.coregistration.opencl_b200")])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_two_backends_at_once():
    """Two blocks with their own buffers on two streams, many runs under way
    together: each keeps its own results."""
    devs = [coreg.Device(0), coreg.Device(0)]
    blks = [Block(d, seed) for seed, d in enumerate(devs)]
    want = []
    for i, b in enumerate(blks):
        b.X.write(maps(10 + i))
        b.run()
        want.append(b.Y.read())
        b.Y.write(np.zeros(N * D, np.float32))
    for _ in range(20):
        for b in blks:
            b.run()
    for b, w in zip(blks, want):
        assert (b.Y.read() == w).all()
    for d in devs:
        d.close()


@pytest.mark.gpu
def test_product_of_a_product(dev):
    """Calls that follow at once on what the one before wrote: a chain of
    quantisations and products, each launch started while the last one ends."""
    lib, o, m = dev.lib, dev.ops_p, coreg.Opnd
    rng = np.random.default_rng(5)
    M, K, steps = 300, 256, 12
    w = (rng.standard_normal((K, K)) / np.sqrt(K)).astype(np.float32)
    qw, sw = ref.quant_i8(w)
    x = rng.standard_normal((M, K)).astype(np.float32)
    QW, SW, Q, S = dev.upload(qw), dev.upload(sw), dev.alloc(M * K), dev.zeros(M)
    bufs = [dev.upload(x), dev.zeros(M * K)]
    for rows in (M, 7, 1):
        bufs[0].write(x)
        for i in range(steps):
            a, c = bufs[i % 2], bufs[(i + 1) % 2]
            lib.ops_quant_i8(o, rows, K, m(a.handle, 0, K, 0, 0), F32, m(Q.handle, 0, K, 0, 0),
                             S.handle, 0)
            lib.ops_gemm_i8(o, rows, K, K, m(Q.handle, 0, K, 0, 0), S.handle,
                            m(QW.handle, 0, K, 0, 0), SW.handle, None, m(c.handle, 0, K, 0, 0),
                            F32, None, 0, 0, 0.0)
        got = bufs[steps % 2].read().reshape(M, K)[:rows]
        y = x[:rows]
        for i in range(steps):
            # (As the device does it: one rounding per scale.)
            q, s = ref.quant_i8(y)
            acc = (q.astype(np.int64) @ qw.astype(np.int64).T).astype(np.float32)
            y = (acc * s[:, None]).astype(np.float32) * sw
        assert np.linalg.norm(got - y) <= 1e-6 * np.linalg.norm(y)
