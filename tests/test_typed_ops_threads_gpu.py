# SPDX-License-Identifier: Unlicense
"""The first calls of a process by several host threads at once (GPU), each with
a backend of its own: every kind of launch whose device has to be asked for
its limits first, results as of one thread."""

import subprocess
import sys
from pathlib import Path

import pytest

CODE = """
import sys
sys.path[:0] = {path!r}
import threading
import numpy as np
import coreg
from oracle import ops_b200_ref as ref
m = coreg.Opnd
rng = np.random.default_rng(0)
maps = [(2, 260000, 64), (1, 500, 64), (1, 3001, 33)]
xs = [rng.standard_normal(s).astype(np.float32) for s in maps]
want = [ref.groupnorm(x, 8 if x.shape[2] == 64 else 11) for x in xs]
prods = [(33, 300, 4096), (8, 1024, 8192), (256, 300, 3333), (700, 4096, 2048), (3, 40, 90)]
ops = [(rng.integers(-127, 128, (M, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8))
       for M, N, K in prods]
sums = [a.astype(np.float64) @ b.astype(np.float64).T for a, b in ops]
THREADS = 6
devs = [coreg.Device(0) for _ in range(THREADS)]
start, bad = threading.Barrier(THREADS), []


def pad(q):
    out = np.zeros((q.shape[0], (q.shape[1] + 15) // 16 * 16), np.int8)
    out[:, :q.shape[1]] = q
    return out


def work(i):
    try:
        dev = devs[i]
        lib, o = dev.lib, dev.ops_p
        X, Y = [dev.upload(x) for x in xs], [dev.zeros(x.size) for x in xs]
        ws = [dev.alloc(lib.ops_groupnorm_cl_bytes(*s, 11)) for s in maps]
        one = dev.upload(np.ones(5000, np.float32))
        AB = [(dev.upload(pad(a)), dev.upload(pad(b))) for a, b in ops]
        Z = [dev.zeros(s.size) for s in sums]
        start.wait()
        order = np.random.default_rng(i).permutation(len(maps) + len(prods))
        for k in order:
            if k < len(maps):
                n, hw, c = maps[k]
                lib.ops_groupnorm_cl(o, n, hw, c, 8 if c == 64 else 11, m(X[k].handle, 0, c, hw * c, 0), 0,
                                     m(Y[k].handle, 0, c, hw * c, 0), 0, None, None, 1e-5, 0, 0.0,
                                     ws[k].handle)
            else:
                k -= len(maps)
                M, N, K = prods[k]
                ld = lib.ops_i8_ld(K)
                lib.ops_gemm_i8(o, M, N, K, m(AB[k][0].handle, 0, ld, 0, 0), one.handle,
                                m(AB[k][1].handle, 0, ld, 0, 0), one.handle, None,
                                m(Z[k].handle, 0, N, 0, 0), 0, None, 0, 0, 0.0)
        coreg.check(lib)
        for y, w in zip(Y, want):
            assert np.abs(y.read().reshape(w.shape) - w).max() < 1e-4
        for z, s in zip(Z, sums):
            assert (z.read().reshape(s.shape) == s.astype(np.float32)).all()
    except BaseException as e:
        bad.append((i, repr(e)))
        start.abort()


ts = [threading.Thread(target=work, args=(i,)) for i in range(THREADS)]
[t.start() for t in ts]
[t.join() for t in ts]
assert not bad, bad
print("all threads")
"""


@pytest.mark.gpu
def test_first_calls_of_several_threads():
    root = Path(__file__).resolve().parents[1]
    code = CODE.format(path=[str(root), str(root / "i.coregistration.opencl_b200")])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all threads" in r.stdout, r.stderr[-2000:]
