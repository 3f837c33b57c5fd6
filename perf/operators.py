"""Timed operators of training from feedback, through the framework's public entry points.

* ``logp`` / ``logp_bwd``: log probabilities of the labels of packed rows through the LM head, and
  the gradient of the rows (``ops.token_logprobs``, ``ops.token_logprobs_backward``).
* ``pref``: a preference loss over pairs of answers, with its gradient (``ops.preference_loss``).
* ``policy``: a clipped policy loss with a KL term, with its gradient (``ops.policy_loss``).
* ``adam``: clip and AdamW over many tensors with the moments in 8 or 32 bits (``ops.AdamW``).

A case is a dict of plain values; ``prepare`` builds from it and a seed what a user's program holds
before the call, ``run`` makes one pass (the framework's kernels where ``own`` is true, the plain form
in elementary torch operations elsewhere), ``exact`` states the same result in 64 bits.
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
BLOCK = 256  # elements that share the scales of an 8-bit moment

# (hidden, vocabulary) of the models the repository configures
HEADS = {"qwen3-0.6b": (1024, 151936), "llama3.2-1b": (2048, 128256), "llama3-8b": (4096, 128256),
         "qwen3-14b": (5120, 151936)}
# (layers, hidden, query width, key/value width) of their attention projections
ATTN = {"qwen3-0.6b": (28, 1024, 2048, 1024), "llama3.2-1b": (16, 2048, 2048, 512),
        "llama3-8b": (32, 4096, 4096, 1024), "qwen3-14b": (40, 5120, 5120, 1024)}


def listed():
    return [
        # The serving preset's 256 tokens of the 14B model, prompts unscored: few rows against the
        # whole head, which streams once.
        dict(name="logp-14b-256", kind="logp", model="qwen3-14b", nseq=2, lo=64, hi=192, total=256,
             lens=0, prompt=0.4),
        # Rollout scoring of the headline packing: 8192 tokens in 32 sequences, Llama-3-8B's head.
        dict(name="logp-8b-8192", kind="logp", model="llama3-8b", nseq=32, lo=64, hi=512, total=8192,
             lens=0, prompt=0.4),
        # The gradient of 504 rows at the smallest model, every predicting row scored.
        dict(name="logp-bwd-0.6b-504", kind="logp_bwd", model="qwen3-0.6b", nseq=4, lo=32, hi=256,
             total=504, lens=0, prompt=0.0, zero=0.0),
        # The gradient of 4097 rows at Llama-3-8B's head, prompts unscored and a tenth of the scored
        # rows clipped to a zero gradient.
        dict(name="logp-bwd-8b-4097", kind="logp_bwd", model="llama3-8b", nseq=16, lo=64, hi=512,
             total=4097, lens=1, prompt=0.4, zero=0.1),
        # A micro-batch of 4 pairs: launches count.
        dict(name="pref-4", kind="pref", nseq=8, lo=32, hi=256, total=1100, lens=0, prompt=0.4,
             loss="sigmoid", beta=0.1, smooth=0.0, margin=0.0, average=False, ref=True),
        # A large batch: 4096 pairs of ragged answers, 4 M rows, smoothed labels.
        dict(name="pref-4096", kind="pref", nseq=8192, lo=8, hi=1024, total=1 << 22, lens=0, prompt=0.3,
             loss="sigmoid", beta=0.1, smooth=0.05, margin=0.0, average=False, ref=True),
        # A micro-batch of 8 answers, one advantage each, with a reference policy: launches count.
        dict(name="policy-8", kind="policy", nseq=8, lo=64, hi=512, total=2048, lens=0, prompt=0.4,
             per_row=False, ref=True, kl=0.04, est="k3", reduction="sequence"),
        # One rollout batch whole: 4096 answers, 16 M rows, advantages by row.
        dict(name="policy-16m", kind="policy", nseq=4096, lo=64, hi=8192, total=(1 << 24) - 5, lens=0,
             prompt=0.2, per_row=True, ref=True, kl=0.04, est="k3", reduction="token"),
        # The attention adapters of the smallest model at rank 8, fp32, clipped by layer: 224 small
        # tensors.
        dict(name="adam8-0.6b-r8", kind="adam", model="qwen3-0.6b", r=8, layers=28, full=False, bits=8,
             dtype="fp32", clip=True, odd=0, shift=0),
        # The adapters of the 8B model at rank 64 with fp32 moments, clipped by layer.
        dict(name="adam32-8b-r64", kind="adam", model="llama3-8b", r=64, layers=32, full=False, bits=32,
             dtype="fp32", clip=True, odd=0, shift=0),
        # The 14B model's with 8-bit moments, ragged tensors among them, no clip.
        dict(name="adam8-14b-r64", kind="adam", model="qwen3-14b", r=64, layers=40, full=False, bits=8,
             dtype="fp32", clip=False, odd=7, shift=0),
        # Six layers' attention weights of the 8B model whole, bf16 weights and gradients: 252 M
        # elements.
        dict(name="adam8-bf16-252m", kind="adam", model="llama3-8b", r=0, layers=6, full=True, bits=8,
             dtype="bf16", clip=True, odd=3, shift=0),
    ]


# ---------------------------------------------------------------- drawing

def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_packing(rng, least, most, longest, even):
    total = _logint(rng, least, most)
    nseq = max(2 if even else 1, min(_logint(rng, 1, 8192), total // 8))
    nseq = max(nseq, -(-total // longest))
    nseq += nseq % 2 if even else 0
    mean = total / nseq
    return dict(nseq=nseq, lo=int(mean / 3), hi=int(mean * 2) + 1, total=total, lens=rng.randrange(1 << 20))


def draw(rng):
    kind = rng.choice(["logp", "logp_bwd", "pref", "policy", "adam", "adam"])
    if kind in ("logp", "logp_bwd"):
        model = rng.choice(list(HEADS))
        D, V = HEADS[model]
        # at most about 8e12 flops forward, 9e12 backward, as the largest listed ones take
        most = min(8192, int((8e12 if kind == "logp" else 9e12) / ((2 if kind == "logp" else 4) * D * V)))
        case = dict(kind=kind, model=model, **_draw_packing(rng, 24, most, 8192, False),
                    prompt=rng.choice([0.0, 0.4, 0.8]))
        if kind == "logp_bwd":
            case["zero"] = rng.choice([0.0, 0.1, 0.5])
        return case
    if kind == "pref":
        loss = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
        return dict(kind=kind, **_draw_packing(rng, 64, 1 << 22, 1 << 17, True),
                    prompt=rng.choice([0.0, 0.3, 0.6]), loss=loss, beta=rng.choice([0.05, 0.1, 0.5]),
                    smooth=rng.choice([0.0, 0.1]) if loss == "sigmoid" else 0.0,
                    margin=rng.choice([0.0, 0.3]) if loss != "ipo" else 0.0,
                    average=rng.random() < 0.4, ref=rng.random() < 0.8)
    if kind == "policy":
        return dict(kind=kind, **_draw_packing(rng, 64, 1 << 24, 1 << 17, False),
                    prompt=rng.choice([0.0, 0.2, 0.6]), per_row=rng.random() < 0.5,
                    ref=rng.random() < 0.7, kl=rng.choice([0.01, 0.04]), est=rng.choice(["k3", "k2"]),
                    reduction=rng.choice(["token", "sequence", "sum"]))
    model = rng.choice(list(ATTN))
    L, D, q, kv = ATTN[model]
    r = rng.choice([4, 8, 13, 16, 32, 64])
    return dict(kind=kind, model=model, r=r, layers=max(1, _logint(rng, 1, L)), full=False,
                bits=rng.choice([8, 8, 32]), dtype=rng.choice(["fp32", "bf16"]), clip=rng.random() < 0.5,
                odd=rng.randrange(0, 9), shift=rng.choice([0, 0, 1]))


# ---------------------------------------------------------------- inputs

def _lens(c):
    """Ragged lengths in [lo, hi] that sum to total, the same for every seed."""
    rng = random.Random(c["lens"])
    lo, hi, k = max(0, c["lo"]), c["hi"], c["nseq"]
    v = [rng.randint(lo, hi) for _ in range(k)]
    off = c["total"] - sum(v)
    while off:
        step = max(1, abs(off) // k)
        for i in range(k):
            d = max(-step, min(step, off))
            w = min(hi, max(lo, v[i] + d))
            off -= w - v[i]
            v[i] = w
            if not off:
                break
    return v


def _rows(c, g):
    """Of a packing: (lengths, starts, row's sequence, rows scored): the last row of a sequence
    predicts nothing, the first `prompt` share of it (varied by sequence) is the prompt."""
    lens = _lens(c)
    n, k = sum(lens), len(lens)
    length = torch.tensor(lens, device=DEV)
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), length.cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(k, device=DEV), length, output_size=n)
    at = torch.arange(n, device=DEV) - start[seq]
    share = c["prompt"] * (0.5 + torch.rand(k, generator=g, device=DEV))
    mask = (at >= (share * length).floor()[seq]) & (at < length[seq] - 1)
    return lens, length, start, seq, mask


def _tensors(c):
    """[(elements, group)] of an adam case; groups are layers."""
    L, D, q, kv = ATTN[c["model"]]
    r, got = c["r"], []
    rng = random.Random(5 + c["odd"])
    for i in range(c["layers"]):
        if c["full"]:
            got += [(D * (q + 2 * kv), i), (q * D, i)]
        else:
            got += [(r * D, i), (q * r, i), (r * D, i), (kv * r, i), (r * D, i), (kv * r, i), (r * q, i),
                    (D * r, i)]
        if i < c["odd"]:
            got += [(1, i), (rng.randrange(2, 20000), i), (rng.randrange(200, 300), i)]
    return got


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    c, s = case, {"case": case}
    if c["kind"] in ("logp", "logp_bwd"):
        D, V = HEADS[c["model"]]
        lens, length, start, seq, mask = _rows(c, g)
        n = len(seq)
        W = torch.randn(V, D, generator=g, device=DEV, dtype=BF16) * 0.02
        lab = torch.randint(0, V, (n,), generator=g, device=DEV)
        # rows that know their label from not at all to almost surely
        pull = 12 * torch.rand(n, 1, generator=g, device=DEV) / (0.02 * math.sqrt(D))
        H = (rand(n, D) + pull * (W[lab].float() / (0.02 * math.sqrt(D)))).to(BF16)
        s.update(H=H, W=W, labels=torch.where(mask, lab, -1))
        if c["kind"] == "logp_bwd":
            s["logp"], s["other"] = _logp_plain(H, W, s["labels"])
            d = rand(n) * mask / n
            s["dlogp"] = d * (torch.rand(n, generator=g, device=DEV) >= c["zero"])
        return s
    if c["kind"] in ("pref", "policy"):
        lens, length, start, seq, mask = _rows(c, g)
        n, k = len(seq), len(lens)
        logp = -torch.rand(n, generator=g, device=DEV).mul_(-1).log1p_().mul_(-1.5)  # mean 1.5 nats
        ref = logp + 0.2 * rand(n)
        s.update(length=length, start=start, mask=mask, logp=logp, n=n, k=k,
                 ref=ref if c["ref"] else None)
        if c["kind"] == "policy":
            s["old"] = logp + 0.15 * rand(n)
            s["adv"] = rand(n if c["per_row"] else k)
        if own:  # what a program keeps of a packing
            from deltaserve_amd import ops

            s["plan"] = ops.pack_plan(lens, device=DEV)
        return s
    # adam: the tensors are views of one buffer, each from a multiple of BLOCK, so that the plain form
    # can take them all at once
    sizes = _tensors(c)
    blocks = [-(-e // BLOCK) for e, _ in sizes]
    nb = sum(blocks)
    dt = F32 if c["dtype"] == "fp32" else BF16
    live = torch.zeros(nb * BLOCK, dtype=torch.bool, device=DEV)
    at, views = 0, []
    for (e, _), b in zip(sizes, blocks):
        live[at:at + e] = True
        views.append((at, e))
        at += b * BLOCK
    flat = lambda x: torch.cat([x.new_zeros(c["shift"]), x])[c["shift"]:]  # noqa: E731
    w = flat((rand(nb * BLOCK) * 0.02 * live).to(dt))
    gr = flat((rand(nb * BLOCK) * torch.exp(rand(nb).repeat_interleave(BLOCK)) * 1e-3 * live).to(dt))
    m = rand(nb * BLOCK) * 5e-4 * live
    v = (rand(nb * BLOCK) * 1e-3).square() * live
    group = torch.repeat_interleave(torch.tensor([i for _, i in sizes], device=DEV),
                                    torch.tensor(blocks, device=DEV))
    ends = torch.cat([group.new_zeros(1), torch.bincount(group, minlength=c["layers"]).cumsum(0)])
    s.update(w=w, g=gr, group=group, ends=ends, ngroups=c["layers"], nb=nb,
             hyper=dict(lr=1e-4, step=100 + seed % 50, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.01,
                        max_norm=0.5 if c["clip"] else None, seed=seed & 0xffff))
    if c["bits"] == 8:
        s["m"], s["m_scale"] = _to8(m)
        s["r"], s["r_scale"] = _to8(v.sqrt())
    else:
        s["m"], s["v"] = m, v
    if own:  # the optimizer that a program keeps, its states as of the step before
        from deltaserve_amd import ops

        opt = ops.AdamW([w[a:a + e] for a, e in views], [gr[a:a + e] for a, e in views], bits=c["bits"],
                        groups=[i for _, i in sizes])
        for name in opt.state():
            opt.state()[name].copy_(s[name])
        s["opt"] = opt
    return s


def _to8(x):
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1) / 448
    q = torch.where(scale[:, None] > 0, x / scale[:, None], 0.0).clamp(-448, 448).to(F8)
    return q.view(-1), scale


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        from deltaserve_amd import ops
    if kind == "logp":
        logp, other = (ops.token_logprobs(s["H"], s["W"], s["labels"]) if own else
                       _logp_plain(s["H"], s["W"], s["labels"]))
        return {"logp": logp, "other": other}
    if kind == "logp_bwd":
        a = (s["H"], s["W"], s["labels"], s["logp"], s["other"], s["dlogp"])
        return {"dh": ops.token_logprobs_backward(*a) if own else _logp_bwd_plain(*a)}
    if kind == "pref":
        if own:
            loss, rewards, d = ops.preference_loss(s["logp"], s["ref"], s["plan"], mask=s["mask"],
                                                   kind=c["loss"], beta=c["beta"],
                                                   label_smoothing=c["smooth"], margin=c["margin"],
                                                   average=c["average"])
        else:
            loss, rewards, d = _pref_plain(s)
        return {"loss": loss, "rewards": rewards, "dlogp": d}
    if kind == "policy":
        if own:
            loss, stats, d = ops.policy_loss(s["logp"], s["old"], s["adv"], s["plan"], mask=s["mask"],
                                             ref_logp=s["ref"], clip_low=0.2, clip_high=0.25,
                                             kl_coef=c["kl"] if c["ref"] else 0.0, kl=c["est"],
                                             reduction=c["reduction"])
        else:
            loss, stats, d = _policy_plain(s)
        return {"loss": loss, "stats": stats, "dlogp": d}
    if own:
        norms, state = s["opt"].step(**s["hyper"]), s["opt"].state()
    else:
        norms, state = _adam_plain(s), {k: s[k] for k in ("m", "m_scale", "r", "r_scale", "v") if k in s}
    return {"w": s["w"], "norms": norms, **state}


def _logp_plain(H, W, labels):
    """(logp, other) in 32 bits: other is the log-sum-exp of the words but the label."""
    live = labels >= 0
    lab = labels[live, None]
    x = H[live].float() @ W.float().t()
    xt = x.gather(1, lab)[:, 0]
    x.scatter_(1, lab, -math.inf)
    top = x.amax(1)
    o = top + (x - top[:, None]).exp_().sum(1).log()
    z = o - xt
    logp, other = torch.zeros(len(labels), device=H.device), torch.zeros(len(labels), device=H.device)
    logp[live] = -(z.clamp(min=0) + (-z.abs()).exp().log1p())
    other[live] = o
    return logp, other


def _logp_bwd_plain(H, W, labels, logp, other, dlogp):
    live = (labels >= 0) & (dlogp != 0)
    lab = labels[live, None]
    Wf = W.float()
    p = H[live].float() @ Wf.t()
    p = (p - other[live, None]).exp_()  # of the other words, to a sum of one
    p.scatter_(1, lab, 0.0)
    d = (dlogp[live] * -logp[live].expm1())[:, None] * (Wf[lab[:, 0]] - p @ Wf)
    out = torch.zeros(H.shape, dtype=BF16, device=H.device)
    out[live] = d.to(BF16)
    return out


def _segments(x, start):
    """Sums of x by sequence, in 64 bits."""
    sums = torch.cat([x.new_zeros(1, dtype=F64), x.cumsum(0, dtype=F64)])[start]
    return sums[1:] - sums[:-1]


def _pref_plain(s):
    c, mask, beta = s["case"], s["mask"], s["case"]["beta"]
    seq = torch.repeat_interleave(torch.arange(s["k"], device=DEV), s["length"], output_size=s["n"])
    diff = s["logp"].double() if s["ref"] is None else s["logp"].double() - s["ref"]
    sums = _segments(torch.where(mask, diff, 0.0), s["start"])
    per = _segments(mask.double(), s["start"]).clamp(min=1) if c["average"] else torch.ones_like(sums)
    sums = sums / per
    h = sums[0::2] - sums[1::2]
    z = beta * h - c["margin"]
    if c["loss"] == "sigmoid":
        soft = lambda t: t.clamp(min=0) + (-t.abs()).exp().log1p()  # noqa: E731
        e = c["smooth"]
        loss = (1 - e) * soft(-z) + e * soft(z)
        dh = beta * (e / (1 + (-z).exp()) - (1 - e) / (1 + z.exp()))
    elif c["loss"] == "hinge":
        loss = (1 - z).clamp(min=0)
        dh = torch.where(z < 1, -beta, 0.0).double()
    else:
        loss = (h - 0.5 / beta).square()
        dh = 2 * (h - 0.5 / beta)
    ds = torch.stack([dh, -dh], 1).view(-1) / (per * len(h))
    d = torch.where(mask, ds[seq], 0.0)
    return loss.mean().float(), (beta * sums).float(), d.float()


def _policy_plain(s):
    c, mask, n = s["case"], s["mask"], s["n"]
    seq = torch.repeat_interleave(torch.arange(s["k"], device=DEV), s["length"], output_size=n)
    A = s["adv"] if c["per_row"] else s["adv"][seq]
    d = torch.where(mask, s["logp"].double() - s["old"], 0.0)
    high, low = d > math.log(1.25), d < math.log(0.8)
    rho = d.float().exp()
    gain = rho * A
    clipped = (high & (A > 0)) | (low & (A < 0))
    pol = -torch.where(clipped, torch.where(high, 1.25, 0.8) * A, gain)
    dpol = -torch.where(clipped, 0.0, gain)
    if c["ref"]:
        u = torch.where(mask, s["ref"].double() - s["logp"], 0.0)
        kl = (u.expm1() - u if c["est"] == "k3" else u.square() / 2).float()
        dkl = (-(u.expm1()) if c["est"] == "k3" else -u).float()
    count = _segments(mask.double(), s["start"])
    if c["reduction"] == "token":
        weight = (1 / count.sum().clamp(min=1)).float().expand(n)
    elif c["reduction"] == "sequence":
        weight = (1 / (count.clamp(min=1) * (count > 0).sum().clamp(min=1))).float()[seq]
    else:
        weight = torch.ones(n, device=DEV)
    weight = torch.where(mask, weight, 0.0)
    total = lambda x: torch.where(mask, weight * x, 0.0).sum(dtype=F64)  # noqa: E731
    coef = c["kl"] if c["ref"] else 0.0
    pl, kt = total(pol), total(kl) if c["ref"] else torch.zeros((), dtype=F64, device=DEV)
    share = (clipped & mask).sum() / count.sum().clamp(min=1)
    g = torch.where(mask, weight * (dpol + coef * dkl if c["ref"] else dpol), 0.0)
    return (pl + coef * kt).float(), torch.stack([pl, kt, share.double()]).float(), g


def _mix(x):
    """A 32-bit mix of non-negative int64 values."""
    low = 0xffffffff
    x = x & low
    x = x ^ (x >> 16)
    x = (x * 0x6a09e667) & low
    x = x ^ (x >> 15)
    x = (x * 0xbb67ae85) & low
    return x ^ (x >> 16)


def _uniform(nb, step, seed):
    """The [blocks, BLOCK] numbers of (0, 1) that round the second moments: 16 bits of a mix of seed,
    step, block and element, two elements to a mix."""
    key = _mix(torch.tensor(seed + step * 0x9e3779b9, device=DEV))
    b = torch.arange(nb, device=DEV)
    key = _mix(key ^ _mix(b))
    x = _mix(key[:, None] + torch.arange(BLOCK // 2, device=DEV) * 0x9e3779b9)
    return ((torch.stack([x & 0xffff, x >> 16], 2).float() + 0.5) / 65536).view(nb, BLOCK)


def _adam_plain(s):
    h, nb = s["hyper"], s["nb"]
    b1, b2, step = h["beta1"], h["beta2"], h["step"]
    g = s["g"].view(nb, BLOCK).float()
    norms = None
    if h["max_norm"] is not None:
        norms = _segments(g.square().sum(1, dtype=F64), s["ends"]).sqrt().float()
        g = g * (h["max_norm"] / (norms + 1e-6)).clamp(max=1)[s["group"], None]
    eight = "r" in s
    if eight:
        m = s["m"].view(nb, BLOCK).float() * s["m_scale"][:, None]
        v = (s["r"].view(nb, BLOCK).float() * s["r_scale"][:, None]).square()
    else:
        m, v = s["m"].view(nb, BLOCK), s["v"].view(nb, BLOCK)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g.square()
    r = v.sqrt()
    w = s["w"].view(nb, BLOCK).float()
    w = w * (1 - h["lr"] * h["wd"]) - h["lr"] / (1 - b1 ** step) * m / (r / math.sqrt(1 - b2 ** step) + h["eps"])
    s["w"].view(nb, BLOCK).copy_(w)
    if eight:
        q, s["m_scale"] = _to8(m)
        s["m"].copy_(q)
        top = r.amax(1)
        x = torch.where(top[:, None] > 0, r * (448 / top)[:, None], 0.0).clamp(max=448)
        grid = torch.exp2(x.clamp(min=2.0 ** -6).log2().floor() - 3)  # e4m3's step at x
        q = (x / grid + _uniform(nb, step, h["seed"])).floor() * grid
        q = torch.where(x > 0, q.clamp(min=2.0 ** -9), 0.0)
        s["r"].copy_(q.to(F8).view(-1))
        s["r_scale"] = top / 448
    else:
        s["m"].copy_(m.view(-1))
        s["v"].copy_(v.view(-1))
    return norms


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] in ("logp", "logp_bwd"):
        D, V = HEADS[c["model"]]
        lens = _lens(c)
        rows = sum(max(0, n - 1 - int(c["prompt"] * n)) for n in lens) * (1 - c.get("zero", 0.0))
        n = sum(lens)
        if c["kind"] == "logp":
            return {"bytes": 2 * D * (V + rows) + 16 * n, "flops": 2 * rows * D * V}
        return {"bytes": 2 * D * (V + rows + n) + 20 * n, "flops": 4 * rows * D * V}
    if c["kind"] == "pref":
        n = c["total"]
        return {"bytes": n * (9 + 4 * c["ref"]) + 4 * c["nseq"], "flops": 3 * n}
    if c["kind"] == "policy":
        n = c["total"]
        return {"bytes": n * (13 + 4 * c["ref"] + 4 * c["per_row"]) + 4 * c["nseq"], "flops": 20 * n}
    n = sum(e for e, _ in _tensors(c))
    e = 4 if c["dtype"] == "fp32" else 2
    state = 16 if c["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (3 * e + state), "flops": 20 * n}


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"logp": _exact_logp, "logp_bwd": _exact_logp_bwd, "pref": _exact_pref,
            "policy": _exact_policy, "adam": _exact_adam}[case["kind"]](s)


def _exact_rows(s, rows):
    """Of some rows with a label: (all logits, label's logit, logits of the others) in 64 bits."""
    x = s["H"][rows].double() @ s["W64"].t()
    lab = s["labels"][rows]
    i = torch.arange(len(rows), device=DEV)
    xt = x[i, lab].clone()
    x[i, lab] = -math.inf
    return x, xt, lab


def _exact_logp(s):
    s["W64"] = s["W"].double()
    n = len(s["labels"])
    logp, other = torch.zeros(n, dtype=F64, device=DEV), torch.zeros(n, dtype=F64, device=DEV)
    for rows in (s["labels"] >= 0).nonzero()[:, 0].split(1024):
        x, xt, _ = _exact_rows(s, rows)
        other[rows] = x.logsumexp(1)
        logp[rows] = torch.nn.functional.logsigmoid(xt - other[rows])
    return {"logp": logp, "other": other}


def _exact_logp_bwd(s):
    s["W64"] = s["W"].double()
    dh = torch.zeros(s["H"].shape, dtype=F64, device=DEV)
    for rows in (s["labels"] >= 0).nonzero()[:, 0].split(1024):
        x, xt, lab = _exact_rows(s, rows)
        q = x.softmax(1)
        rest = torch.sigmoid(x.logsumexp(1) - xt)  # 1 - p(label)
        dh[rows] = (s["dlogp"][rows].double() * rest)[:, None] * (s["W64"][lab] - q @ s["W64"])
    return {"dh": dh}


def _exact_pref(s):
    c, beta = s["case"], s["case"]["beta"]
    n, k = s["n"], s["k"]
    seq = torch.bucketize(torch.arange(n, device=DEV), s["start"][1:], right=True)
    rows = s["mask"].nonzero()[:, 0]
    diff = s["logp"].double()[rows] - (0.0 if s["ref"] is None else s["ref"].double()[rows])
    zero = torch.zeros(k, dtype=F64, device=DEV)
    sums, count = zero.index_add(0, seq[rows], diff), torch.bincount(seq[rows], minlength=k).double()
    if c["average"]:
        sums = sums / count.clamp(min=1)
    sums.requires_grad_()
    with torch.enable_grad():
        h = sums[0::2] - sums[1::2]
        z = beta * h - c["margin"]
        if c["loss"] == "sigmoid":
            ls = torch.nn.functional.logsigmoid
            loss = (-(1 - c["smooth"]) * ls(z) - c["smooth"] * ls(-z)).mean()
        elif c["loss"] == "hinge":
            loss = torch.relu(1 - z).mean()
        else:
            loss = ((h - 1 / (2 * beta)) ** 2).mean()
    ds, = torch.autograd.grad(loss, sums)
    if c["average"]:
        ds = ds / count.clamp(min=1)
    d = torch.zeros(n, dtype=F64, device=DEV)
    d[rows] = ds[seq[rows]]
    return {"loss": loss.detach(), "rewards": beta * sums.detach(), "dlogp": d}


def _exact_policy(s):
    c, n, k = s["case"], s["n"], s["k"]
    seq = torch.bucketize(torch.arange(n, device=DEV), s["start"][1:], right=True)
    rows = s["mask"].nonzero()[:, 0]
    seq = seq[rows]
    A = s["adv"].double()[rows if c["per_row"] else seq]
    x = s["logp"].double()[rows].requires_grad_()
    count = torch.bincount(seq, minlength=k).double()
    if c["reduction"] == "token":
        weight = torch.full_like(A, 1 / max(1, len(rows)))
    elif c["reduction"] == "sequence":
        weight = 1 / (count[seq] * max(1, int((count > 0).sum())))
    else:
        weight = torch.ones_like(A)
    with torch.enable_grad():
        rho = torch.exp(x - s["old"].double()[rows])
        a, b = rho * A, rho.clamp(0.8, 1.25) * A
        policy = (weight * -torch.minimum(a, b)).sum()
        kl = torch.zeros((), dtype=F64, device=DEV)
        if c["ref"]:
            u = s["ref"].double()[rows] - x
            kl = (weight * (torch.expm1(u) - u if c["est"] == "k3" else u * u / 2)).sum()
        loss = policy + (c["kl"] if c["ref"] else 0.0) * kl
    d = torch.zeros(n, dtype=F64, device=DEV)
    d[rows] = torch.autograd.grad(loss, x)[0]
    share = (b < a).double().sum() / max(1, len(rows))
    return {"loss": loss.detach(), "stats": torch.stack([policy.detach(), kl.detach(), share]), "dlogp": d}


def _exact_adam(s):
    h, c = s["hyper"], s["case"]
    eight = c["bits"] == 8
    spread = lambda x: x.double().repeat_interleave(BLOCK)  # noqa: E731
    grad = s["g"].double()
    norms = None
    if c["clip"]:
        per = s["group"].repeat_interleave(BLOCK)
        norms = torch.stack([grad[per == i].norm() for i in range(s["ngroups"])])
        grad = grad * torch.minimum(torch.ones_like(norms), h["max_norm"] / (norms + 1e-6))[per]
    m = s["m"].double() * spread(s["m_scale"]) if eight else s["m"].double()
    v = (s["r"].double() * spread(s["r_scale"])) ** 2 if eight else s["v"].double()
    m = m * h["beta1"] + grad * (1 - h["beta1"])
    v = v * h["beta2"] + grad * grad * (1 - h["beta2"])
    mhat, vhat = m / (1 - h["beta1"] ** h["step"]), v / (1 - h["beta2"] ** h["step"])
    w = s["w"].double()
    out = {"w": w - h["lr"] * h["wd"] * w - h["lr"] * mhat / (vhat.sqrt() + h["eps"]), "norms": norms}
    if not eight:
        return {**out, "m": m, "v": v}
    r = v.sqrt()
    ms, rs = (t.view(-1, BLOCK).abs().amax(1) / 448 for t in (m, r))
    unit = lambda t, sc: torch.where(spread(sc) > 0, t / spread(sc), 0.0)  # noqa: E731
    mant, e = torch.frexp(unit(r, rs))
    grid = torch.ldexp(torch.ones_like(mant), e.clamp(min=-5) - 4)
    q = torch.floor(unit(r, rs) / grid + _uniform(s["nb"], h["step"], h["seed"]).double().view(-1)) * grid
    q = torch.where(r > 0, q.clamp(2.0 ** -9, 448.0), 0.0)
    return {**out, "m": unit(m, ms).float().to(F8).double(), "m_scale": ms, "r": q, "r_scale": rs}
