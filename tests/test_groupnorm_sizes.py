# SPDX-License-Identifier: Unlicense
"""ops_groupnorm_cl at the largest channel counts: what passes 2^30 is refused
(CPU), and a count whose rows in eights wrap round in 32 bits runs (GPU)."""

import numpy as np
import pytest

import coreg
from oracle import ops_b200_ref as ref
from test_typed_ops_refusals import Host
from test_typed_ops_refusals import M as opnd
from typed_ops import BF16, F32


def test_channel_limit():
    h = Host()
    X, Y, work = h.buf(), h.buf(), h.buf()
    for C in (2 ** 30 + 1, 2 ** 31 - 1):
        h.refuses("1 maps of 1 x", "ops_groupnorm_cl", 1, 1, C, 1, opnd(X, C), F32, opnd(Y, C), F32,
                  None, None, 1e-5, 0, 0.0, work)


@pytest.mark.gpu
def test_one_pixel_of_half_a_billion_channels(dev):
    """One pixel of 2^29 + 1 bfloat16 channels, one group: 64 values in turn, the
    first of them once more at the end."""
    C = 2 ** 29 + 1
    p = np.random.default_rng(0).integers(-64, 65, 64).astype(np.float32)  # exact in bfloat16
    bits = (p.view(np.uint32) >> 16).astype(np.uint16)
    x = np.empty(C, np.uint16)
    x[:-1].reshape(-1, 64)[:] = bits
    x[-1] = bits[0]
    X, Y = dev.upload(x), dev.alloc(2 * C)
    work = dev.alloc(dev.lib.ops_groupnorm_cl_bytes(1, 1, C, 1))
    dev.lib.ops_groupnorm_cl(dev.ops_p, 1, 1, C, 1, opnd(X.handle, C), BF16, opnd(Y.handle, C), BF16,
                             None, None, 1e-5, 0, 0.0, work.handle)
    got = Y.read(np.uint16, C)
    coreg.check(dev.lib)
    # (One value more moves the mean and the variance by 2^-29 of the values.)
    want = ref.groupnorm(p[None, :, None], 1)[0, :, 0]
    first = (got[:64].astype(np.uint32) << 16).view(np.float32)
    assert (np.abs(first - want) <= 2.0 ** -8 * np.abs(want) + 1e-5).all()
    assert (got[:-1].reshape(-1, 64) == got[:64]).all() and got[-1] == got[0]
