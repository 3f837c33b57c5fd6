"""Timed operators of a decoder block's memory-bound chain, with its activations kept in 8 bits.

* ``rows8``: rows into and out of the 8-bit activation store (``capture.save_rows`` into
  ``ops.Rows8``, ``ops.unpack_rows8``).
* ``norm8``: RMSNorm and its backward from 8-bit rows (``ops.rmsnorm``, ``ops.rmsnorm_backward``).
* ``swiglu8``: SwiGLU and its backward from 8-bit gate/up rows (``ops.swiglu``,
  ``ops.swiglu_backward``).
* ``join``: the norm after a block, its gate, the scaled residual add and the norm before the next
  block, and their backward (``ops.residual_norm``, ``ops.residual_norm_backward``).
* ``rotary``: rotary positions in both layouts, over part of the head, scaled for long contexts, and
  their backward (``ops.rotary``, ``ops.rotary_backward``).

A case is a dict of plain values; ``prepare`` builds from it and a seed what a user's program holds
before the call, ``run`` makes one pass (the framework's kernels where ``own`` is true, the plain form
in elementary torch operations elsewhere), ``exact`` states the same result in 64 bits.

8-bit rows: codes (e4m3 or int8) [rows, width] and a byte per 32 columns of a row, the exponent of
their scale + 127: the least power of two that brings the largest magnitude to at most 448 (e4m3) or
127 (int8). The value is code·2^(byte − 127).
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deltaserve-vllm_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DEV = "cuda"
BF16 = torch.bfloat16
F32 = torch.float32
F64 = torch.float64
F8 = torch.float8_e4m3fn
TYPES = {"bf16": BF16, "fp16": torch.float16, "fp32": F32}
BLOCK = 32

# (hidden, intermediate, query heads, key/value heads, head width, theta) of the models the repository
# configures, but for the smallest one's MLP
MODELS = {"qwen3-0.6b": (1024, None, 16, 8, 128, 1e6), "llama3.2-1b": (2048, 8192, 32, 8, 64, 5e5),
          "llama3-8b": (4096, 14336, 32, 8, 128, 5e5), "qwen3-14b": (5120, 17408, 40, 8, 128, 1e6)}
MOST_BYTES = 1.1e9  # of a drawn case
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


def listed():
    return [
        # One layer's save of a serving step: 256 finetuning rows picked out of a flat batch of 384,
        # the residual stream as the fused add-norm leaves it (x + r). Launches count.
        dict(name="save-14b-256", kind="rows8", to="codes", code="e4m3", width=5120, rows=384, ft=256,
             resid=True, dtype="bf16"),
        # The gate/up save point of one layer at the headline packing.
        dict(name="save-gate-up-8192", kind="rows8", to="codes", code="e4m3", width=28672, rows=8192,
             ft=8192, resid=False, dtype="bf16"),
        # Restoring one layer's rows, in the integer code, for whatever takes bf16 rows.
        dict(name="restore-8b-4718", kind="rows8", to="rows", code="int8", width=4096, rows=4718),
        # The norm before the attention of a short cycle, recomputed from the store.
        dict(name="norm8-14b-256", kind="norm8", direction="fwd", code="e4m3", width=5120, rows=256),
        # Its backward at the headline packing: the fp32 gradient of the projections, the residual
        # stream's gradient added.
        dict(name="norm8-bwd-8b-8192", kind="norm8", direction="bwd", code="e4m3", width=4096, rows=8192,
             grad="fp32", resid=True),
        # The down projection's input recomputed from the stored gate and up rows.
        dict(name="swiglu8-1b-2048", kind="swiglu8", direction="fwd", code="int8", inter=8192, rows=2048),
        # The MLP's elementwise backward, which leaves the down projection's input too.
        dict(name="swiglu8-bwd-8b-8192", kind="swiglu8", direction="bwd", code="e4m3", inter=14336,
             rows=8192),
        # A forward join of the 8B width: a norm after the block, a gate by channel, a scaled branch.
        dict(name="join-8b-8191", kind="join", direction="fwd", width=4096, rows=8191, stream="bf16",
             post=True, gate="channel", scale=0.5),
        # A short cycle's backward from bf16 rows without a gate or a norm after the block.
        dict(name="join-bwd-0.6b-504", kind="join", direction="bwd", width=1024, rows=504, stream="bf16",
             block="bf16", post=False, gate="none", scale=1.0, grad="fp32", carry="fp32"),
        # The headline packing's from 8-bit rows: everything on, all weight gradients.
        dict(name="join-bwd-8b-8192", kind="join", direction="bwd", width=4096, rows=8192, stream="e4m3",
             block="e4m3", post=True, gate="channel", scale=0.5, grad="bf16", carry="fp32"),
        # Queries and keys of a short packing, a quarter of each head rotated in pairs of neighbours.
        dict(name="rotary-14b-256", kind="rotary", direction="fwd", heads=48, others=8, head=128, rot=32,
             interleaved=True, theta=1e6, scaling="none", rows=256, nseq=2, offset=0, dtype="bf16"),
        # The backward of the long-context packing, positions far out, frequencies scaled for them.
        dict(name="rotary-bwd-8b-16384", kind="rotary", direction="bwd", heads=40, others=8, head=128,
             rot=128, interleaved=False, theta=5e5, scaling="yarn", rows=16384, nseq=2, offset=1 << 20,
             dtype="bf16"),
    ]


# ---------------------------------------------------------------- drawing

def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _draw(rng)
    while work(case)["bytes"] > MOST_BYTES:
        case["rows"] = -(-case["rows"] // 2)
        if "ft" in case:
            case["ft"] = -(-case["ft"] // 2)
    return case


def _draw(rng):
    kind = rng.choice(["rows8", "norm8", "swiglu8", "join", "join", "rotary", "rotary"])
    code = rng.choice(["e4m3", "int8"])
    fwd = rng.choice(["fwd", "bwd"])
    rows = _logint(rng, 1, 8192)
    width = rng.choice([rng.choice([m[0] for m in MODELS.values()]), 8 * _logint(rng, 1, 1024)])
    if kind == "rows8":
        width = rng.choice([width, _logint(rng, 1, 30000)])
        if rng.random() < 0.4:
            return dict(kind=kind, to="rows", code=code, width=width, rows=rows)
        ft = rng.randint(max(1, rows // 3), rows)
        return dict(kind=kind, to="codes", code=code, width=width, rows=rows, ft=ft,
                    resid=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind == "norm8":
        return dict(kind=kind, direction=fwd, code=code, width=width, rows=rows,
                    grad=rng.choice(["bf16", "fp32"]), resid=rng.random() < 0.7)
    if kind == "swiglu8":
        inter = rng.choice([rng.choice([8192, 14336]), 8 * _logint(rng, 1, 1792)])
        return dict(kind=kind, direction=fwd, code=code, inter=inter, rows=rows)
    if kind == "join":
        case = dict(kind=kind, direction=fwd, width=width, rows=rows, stream=rng.choice(["bf16", "fp32"]),
                    post=rng.random() < 0.6, gate=rng.choice(["none", "channel", "row", "full"]),
                    scale=rng.choice([1.0, 0.5, 0.25]))
        if fwd == "bwd":
            case.update(stream=rng.choice(["bf16", "fp32", "e4m3", "int8"]),
                        block=rng.choice(["bf16", "e4m3", "int8"]), grad=rng.choice(["bf16", "fp32"]),
                        carry=rng.choice(["bf16", "fp32"]))
        return case
    head = rng.choice([64, 128, 128, 2 * _logint(rng, 16, 128)])
    rot = rng.choice([head, head, head // 2 // 2 * 2, 2 * rng.randint(1, head // 2)])
    heads = rng.choice([24, 40, 48, rng.randint(1, 48)])
    return dict(kind=kind, direction=fwd, heads=heads, others=rng.choice([0, 8]), head=head, rot=rot,
                interleaved=rng.random() < 0.5, theta=rng.choice([5e5, 1e6]),
                scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                rows=_logint(rng, 1, 16384), nseq=rng.randint(1, 8),
                offset=rng.choice([0, rng.randint(1, 1 << 20)]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


# ---------------------------------------------------------------- inputs

def _stream(g, n, width):
    """Rows as a residual stream has them: sizes vary by row, a few channels are far larger."""
    x = torch.randn(n, width, generator=g, device=DEV) * torch.exp(
        0.3 * torch.randn(n, 1, generator=g, device=DEV))
    big = torch.randint(0, width, (max(1, width // 1000),), generator=g, device=DEV)
    x[:, big] *= 40
    return x


def _codes(x, code):
    """8-bit rows of x, (codes, scale bytes): rows of codes lie a multiple of 16 apart."""
    n, w = x.shape
    nb = -(-w // BLOCK)
    v = torch.zeros(n, nb * BLOCK, device=DEV)
    v[:, :w] = x
    v = v.view(n, nb, BLOCK)
    most = 448.0 if code == "e4m3" else 127.0
    mant, e = torch.frexp(v.abs().amax(2) / most)  # amax = mant·2^e·most, mant in [1/2, 1)
    e = torch.where(mant == 0.5, e - 1, e).clamp(min=-126)
    e = torch.where(mant == 0, -126, e)
    q = (v * torch.exp2(-e.float())[:, :, None]).view(n, -1)[:, :w]
    q = q.to(F8).view(torch.uint8) if code == "e4m3" else q.round().to(torch.int8).view(torch.uint8)
    buf = torch.zeros(n, -(-w // 16) * 16, dtype=torch.uint8, device=DEV)[:, :w]
    buf.copy_(q)
    return buf.view(F8 if code == "e4m3" else torch.int8), (e + 127).to(torch.uint8)


def _values(codes, scales, dtype=F32):
    w = codes.shape[1]
    s = torch.exp2(scales.to(dtype) - 127).repeat_interleave(BLOCK, 1)[:, :w]
    return codes.to(dtype) * s


def _rows8(s, name):
    """What a program holds of 8-bit rows: their two tensors, or the framework's handle of them."""
    if own:
        from deltaserve_amd import ops

        return ops.Rows8(*s[name])
    return s[name]


def _frequencies(c):
    """(inv_freq [rot / 2] in 64 bits, factor of cos and sin)."""
    d, theta, kind = c["rot"], c["theta"], c["scaling"]
    i = torch.arange(d // 2, dtype=F64)
    inv = theta ** (-2 * i / d)
    if kind == "linear":
        return inv / 8, 1.0
    if kind == "llama3":
        turns = 8192 * inv / (2 * math.pi)  # over the original length
        smooth = ((turns - 1) / (4 - 1)).clamp(0, 1)
        return inv * (smooth + (1 - smooth) / 8), 1.0
    if kind == "yarn":
        at = lambda turns: d * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), d - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv * (1 - ramp) + inv / 16 * ramp, 0.1 * math.log(16) + 1
    return inv, 1.0


def _scaling(c):
    return {"none": None, "linear": {"rope_type": "linear", "factor": 8.0}, "llama3": LLAMA3,
            "yarn": {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 8192}
            }[c["scaling"]]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    c, s = case, {"case": case}
    n = c["rows"]
    if c["kind"] == "rows8":
        w = c["width"]
        if c["to"] == "rows":
            s["q"] = _codes(_stream(g, n, w), c["code"])
        else:
            s["x"] = _stream(g, n, w).to(TYPES[c["dtype"]])
            s["r"] = _stream(g, n, w).to(TYPES[c["dtype"]]) if c["resid"] else None
            s["src"] = torch.randperm(n, generator=g, device=DEV)[:c["ft"]].sort()[0]
            s["dst"] = torch.arange(c["ft"], device=DEV)
            s["q"] = _codes(torch.zeros(c["ft"] + 1, w, device=DEV), c["code"])
        s["handle"] = _rows8(s, "q")
    elif c["kind"] == "norm8":
        w = c["width"]
        s["q"] = _codes(_stream(g, n, w), c["code"])
        s["handle"] = _rows8(s, "q")
        s["w"] = (1 + 0.2 * rand(w)).to(BF16)
        if c["direction"] == "bwd":
            s["g"] = (rand(n, w) * 1e-3).to(TYPES[c["grad"]])
            s["resid"] = (rand(n, w) * 1e-3).to(BF16) if c["resid"] else None
    elif c["kind"] == "swiglu8":
        s["q"] = _codes(1.5 * rand(n, 2 * c["inter"]), c["code"])
        s["handle"] = _rows8(s, "q")
        if c["direction"] == "bwd":
            s["dh"] = (rand(n, c["inter"]) * 1e-3).to(BF16)
    elif c["kind"] == "join":
        w = c["width"]
        s["w_in"] = (1 + 0.2 * rand(w)).to(BF16)
        s["w_out"] = (0.3 + 0.1 * rand(w)).to(BF16) if c["post"] else None
        shape = {"none": None, "channel": (w,), "row": (n,), "full": (n, w)}[c["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(rand(*shape)).to(BF16)
        for name, kind in (("x", c["stream"]), ("y", c.get("block", "bf16"))):
            v = _stream(g, n, w) if name == "x" else 0.5 * rand(n, w)
            if kind in TYPES:
                s[name] = s[name + "h"] = v.to(TYPES[kind])
            else:
                s[name] = _codes(v, kind)
                s[name + "h"] = _rows8(s, name)
        if c["direction"] == "bwd":
            s["dn"] = (rand(n, w) * 1e-3).to(TYPES[c["grad"]])
            s["dx"] = (rand(n, w) * 1e-3).to(TYPES[c["carry"]])
    else:
        width = c["heads"] * c["head"]
        rows = rand(n, width + c["others"] * c["head"]).to(TYPES[c["dtype"]])
        s["x"] = rows[:, :width].unflatten(1, (c["heads"], c["head"]))  # of rows that hold v too
        per = -(-n // c["nseq"])
        s["pos"] = (torch.arange(n, device=DEV) % per + c["offset"]).to(torch.int32)
        if own:
            from deltaserve_amd import ops

            s["plan"] = ops.rotary_plan(c["head"], c["theta"], _scaling(c), rotary_dim=c["rot"],
                                        interleaved=c["interleaved"])
        else:
            inv, factor = _frequencies(c)
            s["inv"], s["factor"] = inv.to(DEV), factor
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    kind, fwd = c["kind"], c.get("direction") == "fwd"
    if own:
        from deltaserve_amd import capture, ops
    if kind == "rows8" and c["to"] == "codes":
        if own:
            capture.save_rows(s["x"], s["r"], s["handle"], s["src"], s["dst"])
        else:
            _save_plain(s)
        return {"codes": s["q"][0], "scales": s["q"][1]}
    if kind == "rows8":
        return {"rows": ops.unpack_rows8(s["handle"]) if own else _values(*s["q"]).to(BF16)}
    if kind == "norm8" and fwd:
        if own:
            return {"y": ops.rmsnorm(s["handle"], s["w"], 1e-5)}
        x = _values(*s["q"])
        return {"y": (x * (x.square().mean(1, keepdim=True) + 1e-5).rsqrt() * s["w"].float()).to(BF16)}
    if kind == "norm8":
        if own:
            return {"dx": ops.rmsnorm_backward(s["handle"], s["g"], s["w"], 1e-5, resid=s["resid"])}
        dx = _norm_back(_values(*s["q"]), s["g"].float() * s["w"].float())[0]
        return {"dx": (dx if s["resid"] is None else dx + s["resid"].float()).to(BF16)}
    if kind == "swiglu8" and fwd:
        if own:
            return {"h": ops.swiglu(s["handle"])}
        a, u = _values(*s["q"]).chunk(2, 1)
        return {"h": (a * torch.sigmoid(a) * u).to(BF16)}
    if kind == "swiglu8":
        if own:
            dgu, h = ops.swiglu_backward(s["handle"], s["dh"], with_h=True)
            return {"dgu": dgu, "h": h}
        a, u = _values(*s["q"]).chunk(2, 1)
        sig, d = torch.sigmoid(a), s["dh"].float()
        silu = a * sig
        return {"dgu": torch.cat([d * u * sig * (1 + a * (1 - sig)), d * silu], 1).to(BF16),
                "h": (silu * u).to(BF16)}
    if kind == "join" and fwd:
        if own:
            x, normed = ops.residual_norm(s["x"], s["y"], s["w_in"], 1e-5, w_out=s["w_out"],
                                          gate=s["gate"], scale=c["scale"])
            return {"x": x, "normed": normed}
        return _join_plain(s)
    if kind == "join":
        if own:
            out = ops.residual_norm_backward(s["xh"], s["yh"], s["dn"], s["w_in"], 1e-5, dx_new=s["dx"],
                                             w_out=s["w_out"], gate=s["gate"], scale=c["scale"])
            return dict(zip(("dx", "dy", "dgate", "dw_out", "dw_in"), out))
        return _join_back_plain(s)
    if own:
        turn = ops.rotary if fwd else ops.rotary_backward
        return {"y": turn(s["x"], s["pos"], s["plan"])}
    return {"y": _rotary_plain(s)}


def _save_plain(s):
    x = s["x"].index_select(0, s["src"])
    if s["r"] is not None:
        x = x + s["r"].index_select(0, s["src"])
    codes, scales = _codes(x.float(), s["case"]["code"])
    # (bytes: indexed copies of 8-bit floats are not everywhere)
    s["q"][0].view(torch.uint8).index_copy_(0, s["dst"], codes.view(torch.uint8))
    s["q"][1].index_copy_(0, s["dst"], scales)


def _norm_back(x, gw):
    """(gradient of x, 1 / rms, x / rms) of x / rms(x) with the gradient gw."""
    inv = (x.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    hat = x * inv
    return (gw - hat * (gw * hat).mean(1, keepdim=True)) * inv, inv, hat


def _gate(s, dtype=F32):
    """The gate, for rows."""
    if s["gate"] is None:
        return 1.0
    g = s["gate"].to(dtype)
    return g[:, None] if s["case"]["gate"] == "row" else g


def _join_plain(s):
    x, y, w = s["x"], s["y"].float(), s["w_out"]
    z = y if w is None else y * (y.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w.float()
    x = (x.float() + s["case"]["scale"] * _gate(s) * z).to(x.dtype)
    v = x.float()
    return {"x": x, "normed": (v * (v.square().mean(1, keepdim=True) + 1e-5).rsqrt()
                               * s["w_in"].float()).to(BF16)}


def _float(t):
    return t.float() if torch.is_tensor(t) else _values(*t)


def _join_back_plain(s):
    c = s["case"]
    x, y, dn = _float(s["x"]), _float(s["y"]), s["dn"].float()
    t, _, hat = _norm_back(x, dn * s["w_in"].float())
    t = t + s["dx"].float()
    dw_in = (dn * hat).sum(0)
    dz = c["scale"] * _gate(s) * t
    z, dy, dw_out = y, dz, None
    if s["w_out"] is not None:
        w = s["w_out"].float()
        dy, _, hat = _norm_back(y, dz * w)
        dw_out = (dz * hat).sum(0)
        z = hat * w
    dgate = c["scale"] * t * z if c["gate"] != "none" else None
    if c["gate"] == "channel":
        dgate = dgate.sum(0)
    elif c["gate"] == "row":
        dgate = dgate.sum(1)
    elif c["gate"] == "full":
        dgate = dgate.to(BF16)
    return {"dx": t.to(s["dx"].dtype), "dy": dy.to(BF16), "dgate": dgate, "dw_out": dw_out, "dw_in": dw_in}


def _rotary_plain(s):
    c, x = s["case"], s["x"].float()
    angle = s["pos"].double()[:, None, None] * s["inv"]
    cos = (angle.cos() * s["factor"]).float()
    sin = (angle.sin() * (s["factor"] if c["direction"] == "fwd" else -s["factor"])).float()
    turned, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if c["interleaved"] else turned.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1).to(s["x"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    n = c["rows"]
    code = 1 + 1 / BLOCK
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": code, "int8": code}
    if c["kind"] == "rows8":
        if c["to"] == "rows":
            return {"bytes": n * c["width"] * (code + 2), "flops": n * c["width"]}
        m = c["ft"] * c["width"]
        return {"bytes": m * (size[c["dtype"]] * (1 + c["resid"]) + code) + 16 * c["ft"], "flops": 3 * m}
    if c["kind"] == "norm8":
        m = n * c["width"]
        if c["direction"] == "fwd":
            return {"bytes": m * (code + 2), "flops": 5 * m}
        return {"bytes": m * (code + size[c["grad"]] + 2 * c["resid"] + 2), "flops": 10 * m}
    if c["kind"] == "swiglu8":
        m = n * c["inter"]
        return {"bytes": m * (2 * code + (2 if c["direction"] == "fwd" else 8)),
                "flops": (8 if c["direction"] == "fwd" else 16) * m}
    if c["kind"] == "join":
        m = n * c["width"]
        gate = {"none": 0, "channel": 0, "row": 0, "full": 2}[c["gate"]]
        if c["direction"] == "fwd":
            return {"bytes": m * (2 * size[c["stream"]] + 2 + 2 + gate), "flops": 12 * m}
        return {"bytes": m * (size[c["stream"]] + size[c["block"]] + size[c["grad"]] + 2 * size[c["carry"]]
                              + 2 + 2 * gate), "flops": 40 * m}
    m = n * c["heads"] * c["head"]
    return {"bytes": 2 * m * size[c["dtype"]] + 4 * n, "flops": 3 * n * c["heads"] * c["rot"]}


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rows8" and case["to"] == "codes":
        return _exact_save(s)
    if case["kind"] == "rows8":
        return {"rows": _wide(s["q"])}
    return {"norm8": _exact_norm, "swiglu8": _exact_swiglu, "join": _exact_join,
            "rotary": _exact_rotary}[case["kind"]](s)


def _wide(t):
    """Rows, 8-bit or not, in 64 bits."""
    if torch.is_tensor(t):
        return t.double()
    codes, scales = t
    n, w = codes.shape
    out = torch.empty(n, w, dtype=F64, device=DEV)
    for b in range(scales.shape[1]):
        part = slice(BLOCK * b, min(w, BLOCK * (b + 1)))
        out[:, part] = torch.ldexp(codes[:, part].double(), scales[:, b:b + 1].int() - 127)
    return out


def _exact_save(s):
    x = s["x"][s["src"]]
    if s["r"] is not None:
        x = x + s["r"][s["src"]]  # a sum in the rows' own type is part of the definition
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
    most, least = (448.0, -126) if s["case"]["code"] == "e4m3" else (127.0, -126)
    e = torch.ceil(torch.log2(x.abs().amax(2).clamp(min=2.0 ** -130) / most)).clamp(min=least)
    q = (x / torch.exp2(e)[:, :, None]).flatten(1)[:, :s["x"].shape[1]]
    if s["case"]["code"] == "e4m3":
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
        q = (q / step).round() * step
    codes = torch.zeros(s["q"][0].shape, dtype=F64, device=DEV)
    scales = torch.zeros(s["q"][1].shape, dtype=torch.uint8, device=DEV)
    codes[s["dst"]], scales[s["dst"]] = q.round() if s["case"]["code"] == "int8" else q, (e + 127).to(torch.uint8)
    scales[-1] = 1  # of a row of zeros
    return {"codes": codes if s["case"]["code"] == "e4m3" else codes.to(torch.int8), "scales": scales}


def _rms(x, w):
    return torch.nn.functional.rms_norm(x, x.shape[1:], w, 1e-5)


def _exact_norm(s):
    x, w = _wide(s["q"]).requires_grad_(), s["w"].double()
    with torch.enable_grad():
        y = _rms(x, w)
    if s["case"]["direction"] == "fwd":
        return {"y": y.detach()}
    dx, = torch.autograd.grad(y, x, s["g"].double())
    return {"dx": dx if s["resid"] is None else dx + s["resid"].double()}


def _exact_swiglu(s):
    gu = _wide(s["q"]).requires_grad_()
    with torch.enable_grad():
        a, u = gu.chunk(2, 1)
        h = torch.nn.functional.silu(a) * u
    if s["case"]["direction"] == "fwd":
        return {"h": h.detach()}
    return {"dgu": torch.autograd.grad(h, gu, s["dh"].double())[0], "h": h.detach()}


def _exact_join(s):
    c = s["case"]
    if c["direction"] == "fwd":
        z = s["y"].double()
        if s["w_out"] is not None:
            z = _rms(z, s["w_out"].double())
        x = s["x"].double() + c["scale"] * _gate(s, F64) * z
        # the second norm is of the rows that are returned, in their type
        return {"x": x, "normed": _rms(x.to(s["x"].dtype).double(), s["w_in"].double())}
    x, y = _wide(s["x"]).requires_grad_(), _wide(s["y"]).requires_grad_()
    leaves = {"dw_in": s["w_in"].double().requires_grad_()}
    if s["w_out"] is not None:
        leaves["dw_out"] = s["w_out"].double().requires_grad_()
    if s["gate"] is not None:
        leaves["dgate"] = s["gate"].double().requires_grad_()
    with torch.enable_grad():
        normed = _rms(x, leaves["dw_in"])
    dx, dw_in = torch.autograd.grad(normed, (x, leaves.pop("dw_in")), s["dn"].double())
    dx = dx + s["dx"].double()
    with torch.enable_grad():
        z = _rms(y, leaves["dw_out"]) if "dw_out" in leaves else y
        gate = leaves.get("dgate", 1.0)
        z = c["scale"] * (gate[:, None] if c["gate"] == "row" else gate) * z
    names = list(leaves)
    got = torch.autograd.grad(z, (y, *leaves.values()), dx)
    return {"dx": dx, "dy": got[0], "dgate": None, "dw_out": None, "dw_in": dw_in, **dict(zip(names, got[1:]))}


def _exact_rotary(s):
    c = s["case"]
    inv, factor = _frequencies(c)
    turn = torch.polar(torch.tensor(factor, dtype=F64), s["pos"].cpu().double()[:, None] * inv).to(DEV)
    if c["direction"] == "bwd":
        turn = turn.conj()
    y = s["x"].double()
    r = c["rot"]
    first = slice(0, r, 2) if c["interleaved"] else slice(0, r // 2)
    second = slice(1, r, 2) if c["interleaved"] else slice(r // 2, r)
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return {"y": y}
