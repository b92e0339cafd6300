# SPDX-License-Identifier: Unlicense
"""Timed cases of the 8-bit linear layers, rotary positions and group norm
of include/ops_b200.h: each operator's plain form in torch, its value in
64 bits, and the library's own call."""

import math
import sys
from pathlib import Path

import torch

own = False

ACTS = ("none", "gelu", "relu", "leaky", "gelu_tanh", "silu")
SCALINGS = ("none", "linear", "ntk", "parts")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # The tokens of one tile pair (2 images of 1 + 40 x 40 patches, 1024
        # channels) quantised before a linear layer of the ViT.
        {"name": "quant tokens bf16", "op": "quant", "rows": 3202, "C": 1024, "ld": 1024,
         "type": "bf16"},
        # A wide float32 feature map whose pixels are quantised as tokens, of an
        # odd width in padded rows.
        {"name": "quant map f32 odd", "op": "quant", "rows": 46657, "C": 771, "ld": 772,
         "type": "f32"},
        # First MLP layer of the ViT for a batch of eight tile pairs: the
        # largest product.
        {"name": "gemm_i8 mlp in, 8 pairs", "op": "gemm", "M": 25616, "N": 4096, "K": 1024,
         "type": "bf16", "act": "gelu", "bias": True, "residual": False},
        # Second MLP layer of one tile pair, onto the float32 residual stream.
        {"name": "gemm_i8 mlp out, 1 pair", "op": "gemm", "M": 3202, "N": 1024, "K": 4096,
         "type": "f32", "act": "none", "bias": True, "residual": True},
        # Ragged sizes in every dimension.
        {"name": "gemm_i8 ragged", "op": "gemm", "M": 777, "N": 1001, "K": 1111, "type": "f32",
         "act": "silu", "bias": True, "residual": False},
        # One token (a class token's head, a single descriptor) through a
        # layer: the weights bound it.
        {"name": "linear_i8 one token", "op": "linear", "rows": 1, "in": 1024, "out": 4096,
         "xtype": "bf16", "ytype": "bf16", "act": "gelu", "bias": True, "residual": False},
        # The attention's output projection of one tile pair, float tokens in,
        # added onto the residual stream.
        {"name": "linear_i8 projection", "op": "linear", "rows": 3202, "in": 1024, "out": 1024,
         "xtype": "bf16", "ytype": "f32", "act": "none", "bias": True, "residual": True},
        # Queries and keys of four tile pairs (16 + 16 heads of 64) at their
        # image row and column.
        {"name": "rotary axial 4 pairs", "op": "rotary", "rows": 12808, "nh": 32, "d": 64,
         "rot": 64, "axes": 2, "interleaved": False, "base": 100.0, "scaling": "none",
         "factor": 1.0, "length": 40, "far": 130, "type": "bf16"},
        # One token at a far position, part of each head turned, frequencies
        # stretched by parts.
        {"name": "rotary far token", "op": "rotary", "rows": 1, "nh": 40, "d": 128, "rot": 96,
         "axes": 1, "interleaved": True, "base": 10000.0, "scaling": "parts", "factor": 16.0,
         "length": 4096, "far": 1000000, "type": "f32"},
        # A coarse feature map (35 x 35 x 512) before an attention block: latency.
        {"name": "groupnorm coarse map", "op": "groupnorm", "nimg": 1, "HW": 1225, "C": 512,
         "groups": 32, "xtype": "bf16", "ytype": "bf16", "act": "silu"},
        # Odd map and channel counts, three images, float32.
        {"name": "groupnorm odd f32", "op": "groupnorm", "nimg": 3, "HW": 8137, "C": 120,
         "groups": 5, "xtype": "f32", "ytype": "f32", "act": "gelu"},
        # The full-resolution map of a tile pair (864 x 864 x 64, both images):
        # the largest, beyond the L2 cache.
        {"name": "groupnorm 864 maps", "op": "groupnorm", "nimg": 2, "HW": 746496, "C": 64,
         "groups": 32, "xtype": "bf16", "ytype": "bf16", "act": "relu"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "linear", "rotary", "groupnorm"])
    t, u, act = rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16"]), rng.choice(ACTS)
    if op == "quant":
        C = _log(rng, 16, 8192)
        rows = min(_log(rng, 1, 60000), 35_000_000 // C)
        return {"op": op, "rows": rows, "C": C, "ld": C + rng.choice([0, 0, 1, 8, 16]), "type": t}
    if op in ("gemm", "linear"):
        N, K = _log(rng, 16, 8192), _log(rng, 16, 8192)
        M = max(1, min(_log(rng, 1, 25000), 100_000_000_000 // (N * K), 100_000_000 // N))
        flags = {"act": act, "bias": rng.random() < 0.7, "residual": rng.random() < 0.4}
        if op == "gemm":
            return {"op": op, "M": M, "N": N, "K": K, "type": t, **flags}
        return {"op": op, "rows": M, "in": K, "out": N, "xtype": t, "ytype": u, **flags}
    if op == "rotary":
        axes = rng.choice([1, 2])
        rot = 2 * axes * rng.randint(1, 64 // axes)
        d = rot + rng.choice([0, 0, 8, 32, 33])
        nh = rng.randint(1, 48)
        rows = max(1, min(_log(rng, 1, 50000), 26_000_000 // (nh * d)))
        return {"op": op, "rows": rows, "nh": nh, "d": d, "rot": rot, "axes": axes,
                "interleaved": rng.random() < 0.5, "base": rng.choice([100.0, 10000.0, 500000.0]),
                "scaling": rng.choice(SCALINGS), "factor": rng.choice([2.0, 4.0, 7.5]),
                "length": rng.choice([40, 2048, 8192]), "far": _log(rng, 64, 4000000), "type": t}
    per = rng.choice([1, 2, 3, 4, 6, 8, 16, 24, 32])
    groups = rng.randint(1, max(1, min(64, 1024 // per)))
    C, nimg = per * groups, rng.randint(1, 6)
    HW = max(1, min(_log(rng, 1, 700000), 90_000_000 // (C * nimg)))
    return {"op": op, "nimg": nimg, "HW": HW, "C": C, "groups": groups, "xtype": t, "ytype": u,
            "act": act}


def _quant(x):
    """Row scales and 8-bit values, in 64 bits where a quotient may lie next
    to a border between two integers."""
    s = (x.abs().amax(1).double() / 127).float()
    q = torch.round(x.double() / torch.where(s > 0, s, 1).double()[:, None]).clamp(-127, 127)
    return torch.where(s[:, None] > 0, q, 0).to(torch.int8), s


def _tokens(rows, C, t, gen):
    """Activations as layers see them: unit variance, a few channels many times
    larger, rows of differing size, a row in 97 empty (padding)."""
    x = torch.randn(rows, C, device="cuda", generator=gen)
    x *= torch.where(torch.rand(C, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=gen))
    if rows > 97:
        x[::97] = 0
    return x.to(t)


def _pitch(C):
    return (C + 15) // 16 * 16


def _i8_rows(q):
    """8-bit rows in the layout that the product reads: a multiple of 16 bytes apart."""
    out = torch.zeros(q.shape[0], _pitch(q.shape[1]), dtype=torch.int8, device=q.device)
    out[:, :q.shape[1]] = q
    return out


def prepare(case, seed):
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    c, op = case, case["op"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    s = {"case": dict(case)}
    if op == "quant":
        s["x"] = torch.zeros(c["rows"], c["ld"], device="cuda", dtype=TYPES[c["type"]])
        s["x"][:, :c["C"]] = _tokens(c["rows"], c["C"], TYPES[c["type"]], gen)
        s["q"] = torch.zeros(c["rows"], _pitch(c["C"]), dtype=torch.int8, device="cuda")
        s["s"] = torch.zeros(c["rows"], device="cuda")
    elif op in ("gemm", "linear"):
        M, N, K = (c[k] for k in (("M", "N", "K") if op == "gemm" else ("rows", "out", "in")))
        yt = TYPES[c["type" if op == "gemm" else "ytype"]]
        qw, s["sw"] = _quant(randn(N, K) / math.sqrt(K))
        s["qw"] = _i8_rows(qw)
        if op == "gemm":
            qx, s["sx"] = _quant(_tokens(M, K, torch.float32, gen))
            s["qx"] = _i8_rows(qx)
        else:
            s["x"] = _tokens(M, K, TYPES[c["xtype"]], gen)
        s["bias"] = 0.1 * randn(N) if c["bias"] else None
        # The residual stream, read beside the output so that passes repeat.
        s["r"] = randn(M, N).to(yt) if c["residual"] else None
        s["y"] = torch.zeros(M, N, dtype=yt, device="cuda")
    elif op == "rotary":
        t = TYPES[c["type"]]
        s["x"] = randn(c["rows"], c["nh"] * c["d"]).to(t)
        s["y"] = torch.zeros_like(s["x"])
        s["pos"] = torch.randint(0, c["far"], (c["rows"], c["axes"]), device="cuda",
                                 generator=gen, dtype=torch.int32)
    else:
        x = randn(c["nimg"], c["HW"], c["C"])
        x *= torch.exp(0.5 * randn(c["C"]))
        x += 2 * randn(c["C"])
        s["x"] = x.to(TYPES[c["xtype"]])
        s["y"] = torch.zeros(x.shape, dtype=TYPES[c["ytype"]], device="cuda")
        s["g"], s["b"] = 1 + 0.2 * randn(c["C"]), 0.2 * randn(c["C"])
    return s


def _act(v, name):
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "relu":
        return v.clamp(min=0)
    if name == "leaky":
        return torch.where(v >= 0, v, 0.1 * v)
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _frequencies(c):
    """Radians per position of the rotated pairs of one axis, and the factor
    on the turned values (1 but for frequencies stretched by parts)."""
    n = c["rot"] // c["axes"]
    i = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    base = c["base"]
    if c["scaling"] == "ntk" and n > 2:
        base = base * c["factor"] ** (n / (n - 2))
    w = base ** (-2 * i / n)
    if c["scaling"] == "linear":
        w = w / c["factor"]
    if c["scaling"] == "parts":
        keep = ((w * c["length"] / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        w = w * (keep + (1 - keep) / c["factor"])
    return w, 0.1 * math.log(c["factor"]) + 1 if c["scaling"] == "parts" else 1.0


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "quant":
        q, scale = _quant(s["x"][:, :c["C"]])
        return {"q": q, "s": scale}
    if op in ("gemm", "linear"):
        if op == "linear":
            qx, sx = _quant(s["x"])
            K = c["in"]
        else:
            qx, sx, K = s["qx"], s["sx"], c["K"]
        v = qx[:, :K].float() @ s["qw"][:, :K].float().t()
        v = v * sx[:, None] * s["sw"]
        if c["bias"]:
            v = v + s["bias"]
        v = _act(v, c["act"])
        if c["residual"]:
            v = v + s["r"].float()
        return v.to(s["y"].dtype)
    if op == "rotary":
        rows, nh, d, rot = (c[k] for k in ("rows", "nh", "d", "rot"))
        w, m = _frequencies(c)
        t = (s["pos"].double()[:, :, None] * w).reshape(rows, 1, rot // 2)
        co, si = (m * torch.cos(t)).float(), (m * torch.sin(t)).float()
        x = s["x"].float().reshape(rows, nh, d)
        if c["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            turned = torch.stack([a * co - b * si, a * si + b * co], -1).flatten(-2)
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            turned = torch.cat([a * co - b * si, a * si + b * co], -1)
        return torch.cat([turned, x[..., rot:]], -1).reshape(rows, nh * d).to(s["y"].dtype)
    x = s["x"].float().reshape(c["nimg"], c["HW"], c["groups"], -1)
    mean = x.mean((1, 3), keepdim=True)
    x = x - mean
    x = x / torch.sqrt((x * x).mean((1, 3), keepdim=True) + 1e-5)
    v = _act(x.reshape(c["nimg"], c["HW"], c["C"]) * s["g"] + s["b"], c["act"])
    return v.to(s["y"].dtype)


_coreg = _device = None


def _bind(s):
    """The library's call for a state: its entry point and arguments over the
    state's tensors, as a caller sets them up beside its buffers."""
    global _coreg, _device
    package = str(Path(__file__).resolve().parents[1] / "i.coregistration.opencl_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import coreg

    if _device is None:
        _coreg, _device = coreg, coreg.Device(torch.cuda.current_device())
    lib, o = _device.lib, _device.ops_p
    s["buffers"] = []
    c, op = s["case"], s["case"]["op"]

    def buf(t):
        if t is None:
            return None
        n = t.numel() * t.element_size()
        s["buffers"].append(coreg.Buffer(_device, lib.ocl_wrap(t.data_ptr(), n), n))
        return s["buffers"][-1].handle

    def mat(t, s0=0):
        return coreg.Opnd(buf(t), 0, t.shape[-1], s0, 0)

    def kind(t):
        return coreg.OPS_BF16 if t.dtype == torch.bfloat16 else coreg.OPS_FP32

    if op == "quant":
        args = (o, c["rows"], c["C"], mat(s["x"]), kind(s["x"]), mat(s["q"]), buf(s["s"]), 0)
        out = {"q": s["q"][:, :c["C"]], "s": s["s"]}
        return lib.ops_quant_i8, args, out
    act = ACTS.index(c["act"]) if "act" in c else 0
    if op == "gemm":
        args = (o, c["M"], c["N"], c["K"], mat(s["qx"]), buf(s["sx"]), mat(s["qw"]), buf(s["sw"]),
                buf(s["bias"]), mat(s["y"]), kind(s["y"]), buf(s["r"]), 0, act, 0.1)
        return lib.ops_gemm_i8, args, s["y"]
    if op == "linear":
        n = lib.ops_linear_i8_bytes(c["rows"], c["in"])
        s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        args = (o, c["rows"], c["in"], c["out"], mat(s["x"]), kind(s["x"]), mat(s["qw"]),
                buf(s["sw"]), buf(s["bias"]), mat(s["y"]), kind(s["y"]), buf(s["r"]), 0, act, 0.1,
                buf(s["work"]))
        return lib.ops_linear_i8, args, s["y"]
    if op == "rotary":
        plan = coreg.Rotary()
        lib.ops_rotary_plan(plan, c["rot"], c["axes"], int(c["interleaved"]), c["base"],
                            SCALINGS.index(c["scaling"]), c["factor"], c["length"])
        args = (o, plan, c["rows"], c["nh"], c["d"], mat(s["x"]), mat(s["y"]), kind(s["x"]),
                buf(s["pos"]), 0)
        return lib.ops_rotary, args, s["y"]
    n = lib.ops_groupnorm_cl_bytes(c["nimg"], c["HW"], c["C"], c["groups"])
    s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    image = c["HW"] * c["C"]
    args = (o, c["nimg"], c["HW"], c["C"], c["groups"], mat(s["x"], image), kind(s["x"]),
            mat(s["y"], image), kind(s["y"]), buf(s["g"]), buf(s["b"]), 1e-5, act, 0.1,
            buf(s["work"]))
    return lib.ops_groupnorm_cl, args, s["y"]


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _bind(s)
        call, args, out = s["call"]
        call(*args)
        _coreg.check(_device.lib)
        return out
    return _plain(s)


def work(case):
    c, op = case, case["op"]
    size = {"f32": 4, "bf16": 2}
    if op == "quant":
        n = c["rows"] * c["C"]
        return {"bytes": n * size[c["type"]] + n + 4 * c["rows"], "flops": 4 * n}
    if op in ("gemm", "linear"):
        M, N, K = (c[k] for k in (("M", "N", "K") if op == "gemm" else ("rows", "out", "in")))
        y = M * N * size[c["type" if op == "gemm" else "ytype"]]
        x = M * K + 4 * M if op == "gemm" else M * K * size[c["xtype"]]
        return {"bytes": x + N * K + 4 * N + 4 * N * c["bias"] + y + y * c["residual"],
                "flops": 2 * M * N * K}
    if op == "rotary":
        n = c["rows"] * c["nh"] * c["d"]
        return {"bytes": 2 * n * size[c["type"]] + 4 * c["rows"] * c["axes"],
                "flops": 3 * c["rows"] * c["nh"] * c["rot"]}
    n = c["nimg"] * c["HW"] * c["C"]
    return {"bytes": n * (size[c["xtype"]] + size[c["ytype"]]) + 8 * c["C"], "flops": 10 * n}


def _act64(v, name):
    phi = {"none": lambda: v, "relu": lambda: torch.maximum(v, torch.zeros_like(v)),
           "leaky": lambda: torch.maximum(v, 0.1 * v),
           "silu": lambda: v * torch.special.expit(v),
           "gelu": lambda: v * torch.special.ndtr(v),
           "gelu_tanh": lambda: v * torch.special.expit(
               2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}
    return phi[name]()


def _quant64(x):
    """The nearest integers to x over its row's scale, which is the float32
    number nearest to a 127th of the row's largest magnitude."""
    s = (torch.linalg.vector_norm(x.double(), float("inf"), dim=1) / 127.0).float().double()
    live = (s > 0).double()
    ratio = live[:, None] * x.double() / (s + 1.0 - live)[:, None]
    return torch.clip(ratio.round(), -127.0, 127.0), s


def exact(case, seed):
    s, c, op = prepare(case, seed), case, case["op"]
    if op == "quant":
        q, scale = _quant64(s["x"].narrow(1, 0, c["C"]))
        return {"q": q.to(torch.int8), "s": scale}
    if op in ("gemm", "linear"):
        if op == "gemm":
            q, scale = s["qx"].narrow(1, 0, c["K"]).double(), s["sx"].double()
        else:
            q, scale = _quant64(s["x"])
        v = torch.einsum("mk,nk->mn", q, s["qw"].narrow(1, 0, q.shape[1]).double())
        v = torch.einsum("mn,m,n->mn", v, scale, s["sw"].double())
        v = _act64(v if s["bias"] is None else v + s["bias"].double(), c["act"])
        return v if s["r"] is None else v + s["r"].double()
    if op == "rotary":
        n, half = c["rot"] // c["axes"], c["rot"] // 2
        i = torch.arange(n // 2, device="cuda").double()
        ln = math.log(c["base"])
        if c["scaling"] == "ntk" and n > 2:
            ln += math.log(c["factor"]) * n / (n - 2)
        w, m = torch.exp(-ln * 2 * i / n), 1.0
        if c["scaling"] == "linear":
            w = w / c["factor"]
        if c["scaling"] == "parts":
            turns = c["length"] * w / (2 * math.pi)
            share = torch.clip((turns - 1) / 31, 0.0, 1.0)
            w = share * w + (1 - share) * w / c["factor"]
            m = 1 + 0.1 * math.log(c["factor"])
        axis = torch.arange(half, device="cuda") // (n // 2)
        angle = s["pos"].double()[:, axis] * w.repeat(c["axes"])
        z = torch.polar(torch.full_like(angle, m), angle)[:, None, :]
        x = s["x"].double().view(c["rows"], c["nh"], c["d"])
        y = x.clone()
        k = torch.arange(half, device="cuda")
        first, second = (2 * k, 2 * k + 1) if c["interleaved"] else (k, k + half)
        turned = torch.complex(x[..., first], x[..., second]) * z
        y[..., first], y[..., second] = turned.real, turned.imag
        return y.view(c["rows"], -1)
    x = s["x"].double().unflatten(2, (c["groups"], -1))
    var, mean = torch.var_mean(x, dim=(1, 3), correction=0, keepdim=True)
    y = ((x - mean) * torch.rsqrt(var + 1e-5)).flatten(2)
    return _act64(torch.addcmul(s["b"].double(), y, s["g"].double()), c["act"])
