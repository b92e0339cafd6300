# SPDX-License-Identifier: Unlicense
"""Plain 64-bit forms of the operations of include/ops_b200.h that take
typed buffers: row quantisation to 8 bits, the 8-bit product and linear
layer, rotary positions and channels-last group norm (numpy, one step per
line of their formulas)."""

import math

import numpy as np

# Pi to the long double's 64 bits (numpy's is a double: 2^-54 off).
PI = np.longdouble("3.141592653589793238462643383279503")
ACTS = ("none", "gelu", "relu", "leaky", "gelu_tanh", "silu")


def act(v, kind, slope=0.1):
    v = np.asarray(v, np.float64)
    if kind == "gelu":
        return 0.5 * v * (1 + np.vectorize(math.erf)(v * math.sqrt(0.5)))
    if kind == "relu":
        return np.maximum(v, 0)
    if kind == "leaky":
        return np.where(v >= 0, v, np.float64(np.float32(slope)) * v)
    if kind == "gelu_tanh":
        return 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if kind == "silu":
        with np.errstate(over="ignore"):
            return v / (1 + np.exp(-v))
    return v


def quant_i8(x):
    """(q, s) of float32 (or narrower) rows: s the float32 nearest to a 127th
    of the largest magnitude, q the nearest integers to x / s. A float64
    quotient of two float32 numbers is a tie only where the real one is."""
    x = np.asarray(x, np.float32)
    a = np.abs(x)
    bad = ~np.isfinite(x).all(1)
    amax = np.where(bad, 0, a.max(1, initial=0)).astype(np.float64)
    s = (amax / 127.0).astype(np.float32)
    live = s > 0
    with np.errstate(invalid="ignore"):
        q = np.rint(x.astype(np.float64) / np.where(live, s, 1).astype(np.float64)[:, None])
        q = np.where(live[:, None], np.clip(q, -127, 127), 0).astype(np.int8)
    return q, np.where(bad, np.float32(np.nan), s).astype(np.float32)


def gemm_i8(a, sa, b, sb, bias=None, kind="none", slope=0.1, residual=None):
    """(result, magnitude of what is added before the activation)."""
    acc = a.astype(np.float64) @ b.astype(np.float64).T  # exact below 2^53
    v = acc * np.asarray(sa, np.float64)[:, None] * np.asarray(sb, np.float64)
    mag = np.abs(v)
    if bias is not None:
        v = v + bias.astype(np.float64)
        mag = mag + np.abs(bias)
    v = act(v, kind, slope)
    return (v if residual is None else v + residual.astype(np.float64)), mag


def frequencies(rot, axes, base, scaling="none", factor=1.0, length=1):
    """(radians per position of each pair of an axis, magnitude factor)."""
    n = rot // axes
    i = np.arange(n // 2, dtype=np.longdouble)
    b = np.longdouble(base)
    if scaling == "ntk" and n > 2:
        b = b * np.longdouble(factor) ** (np.longdouble(n) / (n - 2))
    w = b ** (-2 * i / n)
    if scaling == "linear":
        w = w / factor
    if scaling == "parts":
        g = np.clip((length * w / (2 * PI) - 1) / 31, 0, 1)
        w = g * w + (1 - g) * w / factor
    return w, 0.1 * math.log(factor) + 1 if scaling == "parts" and factor > 1 else 1.0


def rotary(x, pos, nh, d, rot, axes, interleaved, w, m=1.0):
    """x (rows, nh d) turned at pos (rows, axes)."""
    x = np.asarray(x, np.float64).reshape(len(x), nh, d)
    y = x.copy()
    half, per = rot // 2, rot // 2 // axes
    for f in range(half):
        t = (pos[:, f // per].astype(np.longdouble) * w[f % per]).astype(np.float64)[:, None]
        i0, i1 = (2 * f, 2 * f + 1) if interleaved else (f, f + half)
        y[:, :, i0] = m * (x[:, :, i0] * np.cos(t) - x[:, :, i1] * np.sin(t))
        y[:, :, i1] = m * (x[:, :, i0] * np.sin(t) + x[:, :, i1] * np.cos(t))
    return y.reshape(len(x), nh * d)


def groupnorm(x, groups, g=None, b=None, eps=1e-5, kind="none", slope=0.1):
    """x (images, pixels, channels)."""
    n, hw, c = x.shape
    v = np.asarray(x, np.float64).reshape(n, hw, groups, c // groups)
    v = v - v.mean((1, 3), keepdims=True)
    v = v / np.sqrt((v * v).mean((1, 3), keepdims=True) + np.float64(np.float32(eps)))
    v = v.reshape(n, hw, c)
    if g is not None:
        v = v * g.astype(np.float64) + b.astype(np.float64)
    return act(v, kind, slope)
