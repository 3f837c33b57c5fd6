"""The operators for training from feedback against their formulas in 64 bits: log probabilities of
labels and their gradient, the preference and policy losses, AdamW with 8- and 32-bit moments, and
all of them together. Each tolerance counts the roundings of the path, with U32 = 2^-24 half a step
of fp32 and U16 = 2^-8 half a step of bf16 (both relative)."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
F8 = torch.float8_e4m3fn
U32, U16 = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _ops():
    from deltaserve_amd import ops

    return ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _within(got, want, tol):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bad.any(), (int(bad.sum()), float(d[bad].max()), float((d / tol)[bad].max()))


# ---------------------------------------------------------------- log probabilities

def _head_inputs(n, D, V, seed, scored="some", pull=8.0, ld=None):
    g = _gen(seed)
    W = (torch.randn(V, D, generator=g, device=DEV) / math.sqrt(D)).to(BF16)
    lab = torch.randint(0, V, (n,), generator=g, device=DEV)
    H = torch.randn(n, D, generator=g, device=DEV)
    H += pull * torch.rand(n, 1, generator=g, device=DEV) * W[lab].float()
    buf = torch.full((n, ld or D), 7.0, dtype=BF16, device=DEV)
    buf[:, :D] = H.to(BF16)
    if scored == "some":
        lab[torch.rand(n, generator=g, device=DEV) < 0.4] = -1
    elif scored == "none":
        lab[:] = -100
    return buf[:, :D], W, lab


def _head_exact(H, W, lab):
    """(logp, other, q) in 64 bits; q: the softmax of the other words."""
    x = H.double() @ W.double().t()
    i = torch.arange(len(lab), device=DEV)
    t = lab.clamp(min=0)
    xt = x[i, t].clone()
    x[i, t] = -math.inf
    other = x.logsumexp(1)
    return torch.nn.functional.logsigmoid(xt - other), other, (x - other[:, None]).exp()


def _head_tol(H, W):
    """A logit is a sum of D exact products in fp32: off by at most D·U32·Σ|h·w|. The statistics add:
    the exponent's argument is within 128 and rounded once or twice (256·U32 relative in e^x), the
    sums of V terms in runs and over runs (at most 300 additions deep), the logarithm's own."""
    S = (H.double().abs() @ W.double().abs().t()).amax(1)
    D = H.shape[1]
    return D * U32 * S, 2 * D * U32 * S + (256 + 300 + 64) * U32


SHAPES = [(1, 8, 2), (1, 64, 1000), (2, 72, 31), (5, 128, 257), (33, 64, 3), (130, 256, 5001),
          (257, 104, 20001), (300, 1024, 2000), (3001, 64, 50003), (130, 64, 70001)]


@pytest.mark.parametrize("scored", ["all", "some", "none"])
@pytest.mark.parametrize("n,D,V", SHAPES)
def test_token_logprobs(n, D, V, scored):
    ops = _ops()
    H, W, lab = _head_inputs(n, D, V, n + D + V, scored, ld=D + 8 if n % 2 else None)
    logp, other = ops.token_logprobs(H, W, lab)
    e_logp, e_other, _ = _head_exact(H, W, lab)
    live = lab >= 0
    _, tol = _head_tol(H, W)
    assert (logp[~live] == 0).all() and (other[~live] == 0).all()
    _within(logp[live], e_logp[live], (tol + 4 * U32 * e_logp.abs())[live])
    _within(other[live], e_other[live], (tol + 4 * U32 * e_other.abs())[live])


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("n,D,V", SHAPES)
def test_token_logprobs_backward(n, D, V, out_dtype):
    ops = _ops()
    H, W, lab = _head_inputs(n, D, V, 2 * n + D + V)
    g = _gen(n)
    d = torch.randn(n, generator=g, device=DEV)
    d[torch.rand(n, generator=g, device=DEV) < 0.2] = 0
    logp, other, q = _head_exact(H, W, lab)
    live = lab >= 0
    logp32, other32 = logp.float() * live, other.float() * live
    got = ops.token_logprobs_backward(H, W, lab, logp32, other32, d, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    W64 = W.double()
    want = torch.where(live, d.double() * -logp.expm1(), 0.0)[:, None] * (W64[lab.clamp(min=0)] - q @ W64)
    # q: rounded to bf16 (U16), its logit's and the given reference's errors (relative); the division by
    # the rounded sum doubles each. The product sums V terms in fp32 (at most 64 + V / 64 deep).
    # 1 − p_t: its argument's rounding, U32·|logp|. Last the output's own rounding.
    ex, _ = _head_tol(H, W)
    rel = 2 * (U16 + ex + other.abs() * U32 + 256 * U32) + (64 + V / 64) * U32
    spread = q @ W64.abs() + W64[lab.clamp(min=0)].abs()
    tol = (d.double().abs() * -logp.expm1() * rel)[:, None] * spread
    tol = tol + (d.double().abs() * logp.abs() * logp.exp() * U32)[:, None] * spread
    tol = tol + (U16 if out_dtype == BF16 else 4 * U32) * want.abs() + 2.0 ** -120
    _within(got, want, tol)
    assert (got[(~live) | (d == 0)] == 0).all()


def test_logprobs_of_many_rows_in_chunks():
    """More probabilities than one chunk of the vocabulary holds: the gradient's accumulators carry
    over, at two shares of scored rows (different K slices). Checked on a tenth of the rows."""
    ops = _ops()
    n, D, V = 8200, 64, 70001
    for seed, part in ((1, 0.7), (2, 0.05)):
        H, W, lab = _head_inputs(n, D, V, seed, "all")
        lab[torch.rand(n, generator=_gen(seed), device=DEV) >= part] = -1
        d = torch.randn(n, generator=_gen(9), device=DEV)
        logp, other = ops.token_logprobs(H, W, lab)
        got = ops.token_logprobs_backward(H, W, lab, logp, other, d, out_dtype=F32)
        assert (got[lab < 0] == 0).all()
        some = (lab >= 0).nonzero()[:, 0][::10]
        e_logp, e_other, q = _head_exact(H[some], W, lab[some])
        ex, tol = _head_tol(H[some], W)
        _within(logp[some], e_logp, tol + 4 * U32 * e_logp.abs())
        _within(other[some], e_other, tol + 4 * U32 * e_other.abs())
        W64, g = W.double(), d[some].double().abs() * -e_logp.expm1()
        want = (d[some].double() * -e_logp.expm1())[:, None] * (W64[lab[some]] - q @ W64)
        spread = q @ W64.abs() + W64[lab[some]].abs()
        rel = 2 * (U16 + ex + tol + 256 * U32) + (64 + V / 64) * U32
        bound = (g * rel)[:, None] * spread + (d[some].double().abs() * tol)[:, None] * spread
        _within(got[some], want, bound + 4 * U32 * want.abs() + 2.0 ** -120)


def test_logprobs_of_sure_and_hopeless_labels():
    """Labels 30 to 200 logits above or below the rest: no overflow, full relative precision of
    1 − p_t; a label that nothing else comes near has logp −0 and no gradient."""
    ops = _ops()
    D, V, n = 64, 777, 24
    W = torch.zeros(V, D, dtype=BF16, device=DEV)
    g = _gen(3)
    W[:, 1:] = (torch.randn(V, D - 1, generator=g, device=DEV) * 0.1).to(BF16)
    W[:, 0] = 0
    W[5, 0] = 1
    H = torch.randn(n, D, generator=g, device=DEV).to(BF16)
    H[:, 0] = torch.linspace(-200, 200, n, device=DEV).to(BF16)
    lab = torch.full((n,), 5, device=DEV)
    logp, other = ops.token_logprobs(H, W, lab)
    e_logp, e_other, q = _head_exact(H, W, lab)
    ex, tol = _head_tol(H, W)
    _within(other[H[:, 0] < 80], e_other[H[:, 0] < 80], tol[H[:, 0] < 80] + 4 * U32 * e_other[H[:, 0] < 80].abs())
    # relative in e^(other − x_t): the tolerance of its exponent; below 2^-126 it is denormal or 0
    _within(logp, e_logp, (2 * tol + 256 * U32) * e_logp.abs() + 2.0 ** -120)
    d = torch.ones(n, device=DEV)
    got = ops.token_logprobs_backward(H, W, lab, logp, other, d, out_dtype=F32)
    W64 = W.double()
    want = -e_logp.expm1()[:, None] * (W64[5] - q @ W64)
    spread = -e_logp.expm1()[:, None] * (q @ W64.abs() + W64[5].abs())
    _within(got, want, (2 * (U16 + 2 * ex + 2 * tol) + 1024 * U32)[:, None] * spread + 2.0 ** -110)
    assert torch.isfinite(got).all()
    # the words' roles swapped: one other word far above the label
    lab = torch.full((n,), 9, device=DEV)
    logp, other = ops.token_logprobs(H, W, lab)
    e_logp, e_other, _ = _head_exact(H, W, lab)
    _within(logp, e_logp, _head_tol(H, W)[1] + 4 * U32 * e_logp.abs())
    _within(other, e_other, _head_tol(H, W)[1] + 4 * U32 * e_other.abs())


def test_logprobs_of_labels_past_the_vocabulary():
    ops = _ops()
    H, W, lab = _head_inputs(9, 64, 300, 1, "all")
    want = ops.token_logprobs(H, W, lab)
    bad = lab.clone()
    bad[2], bad[7] = 300, 1 << 40
    logp, other = ops.token_logprobs(H, W, bad)
    keep = torch.tensor([0, 1, 3, 4, 5, 6, 8], device=DEV)
    assert logp[[2, 7]].isnan().all() and other[[2, 7]].isnan().all()
    assert torch.equal(logp[keep], want[0][keep]) and torch.equal(other[keep], want[1][keep])
    d = torch.ones(9, device=DEV)
    dh = ops.token_logprobs_backward(H, W, bad, logp, other, d)
    assert dh[[2, 7]].isnan().all()
    assert torch.equal(dh[keep], ops.token_logprobs_backward(H, W, lab, *want, d)[keep])


@pytest.mark.parametrize("n", [1023, 1024, 1025])
def test_logprobs_where_the_rows_are_counted_otherwise(n):
    """Scored rows, rows left out and labels past the vocabulary are the same on both sides of the size
    from which a kernel of its own counts the rows."""
    ops = _ops()
    V = 500
    H, W, lab = _head_inputs(n, 64, V, 3, "some")
    lab[5::11] = V
    d = torch.randn(n, generator=_gen(4), device=DEV)
    d[::7] = 0.0
    logp, other = ops.token_logprobs(H, W, lab)
    got = ops.token_logprobs_backward(H, W, lab, logp, other, d, F32)
    e_logp, e_other, _ = _head_exact(H, W, lab.clamp(max=V - 1))
    _, tol = _head_tol(H, W)
    past, live = lab >= V, (lab >= 0) & (lab < V)
    assert logp[past].isnan().all() and other[past].isnan().all()
    assert (logp[lab < 0] == 0).all() and (other[lab < 0] == 0).all()
    _within(logp[live], e_logp[live], (tol + 4 * U32 * e_logp.abs())[live])
    assert got[past & (d != 0)].isnan().all() and (got[(lab < 0) | (d == 0)] == 0).all()
    k = 300  # a shorter batch of the same rows, each row's gradient the same
    few = ops.token_logprobs_backward(H[:k], W, lab[:k], logp[:k], other[:k], d[:k], F32)
    rows = ((live & (d != 0))[:k]).nonzero()[:, 0]
    assert len(rows) > 50
    # sums of V terms in another order, of parts of at most |d| and |d|·|W| times 1 − p
    size = d[:k][rows, None].double().abs() * W.double().abs().max()
    _within(few[rows], got[:k][rows].double(), 4 * (V + 8) * U32 * size)


def test_logprobs_leave_unscored_rows_out():
    """NaN in an unscored row stays there, and a row's results do not depend on which others are
    scored beyond the tiles' sums (compared against a call on the scored rows alone)."""
    ops = _ops()
    H, W, lab = _head_inputs(150, 128, 3000, 4)
    live = lab >= 0
    H = H.clone()
    H[~live] = float("nan")
    a, b = ops.token_logprobs(H, W, lab)
    c, d = ops.token_logprobs(H[live].contiguous(), W, lab[live].contiguous())
    _, tol = _head_tol(H[live], W)
    _within(a[live], c.double(), 2 * tol)
    _within(b[live], d.double(), 2 * tol)
    assert (a[~live] == 0).all()
    g = torch.randn(150, generator=_gen(1), device=DEV)
    dh = ops.token_logprobs_backward(H, W, lab, a, b, g)
    assert torch.isfinite(dh).all() and (dh[~live] == 0).all()


def test_logprobs_empty():
    ops = _ops()
    H, W = torch.empty(0, 64, dtype=BF16, device=DEV), torch.zeros(10, 64, dtype=BF16, device=DEV)
    lab = torch.empty(0, dtype=torch.int64, device=DEV)
    logp, other = ops.token_logprobs(H, W, lab)
    assert logp.shape == (0,) and other.shape == (0,)
    assert ops.token_logprobs_backward(H, W, lab, logp, other, logp).shape == (0, 64)


def _replayed(make, refresh, want):
    """make() captured once; then for three sets of inputs: refresh(k), an eager result, a replay,
    eager work between, all compared."""
    refresh(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        make()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = make()
    for k in range(1, 4):
        refresh(k)
        ref = [t.clone() for t in want()]
        refresh(k)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, ref):
            assert torch.equal(a, b), k
        torch.ones(1000, device=DEV).sum().item()


def test_logprobs_captured_and_replayed():
    ops = _ops()
    sets = [_head_inputs(200, 128, 9000, 50 + k) for k in range(4)]
    H, W, lab = (t.clone() for t in sets[0])
    g = torch.randn(200, generator=_gen(8), device=DEV)

    def make():
        logp, other = ops.token_logprobs(H, W, lab)
        return logp, other, ops.token_logprobs_backward(H, W, lab, logp, other, g)

    def refresh(k):
        for t, s in zip((H, W, lab), sets[k]):
            t.copy_(s)

    _replayed(make, refresh, make)


# ---------------------------------------------------------------- packings

def _packing(lens, seed, values=1, masked=True):
    """(plan, row's sequence, mask, fp32 rows...), all on the device."""
    ops = _ops()
    g = _gen(seed)
    n = sum(lens)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens, dtype=torch.int64)).to(DEV)
    mask = torch.rand(n, generator=g, device=DEV) < 0.6 if masked else None
    rows = [torch.randn(n, generator=g, device=DEV) for _ in range(values)]
    return (ops.pack_plan(lens), seq, mask, *rows)


def _scored(lens, mask):
    if mask is not None:
        return mask
    last = torch.tensor(lens, dtype=torch.int64).cumsum(0)
    on = torch.ones(sum(lens), dtype=torch.bool)
    on[[int(e) - 1 for e, x in zip(last, lens) if x]] = False
    return on.to(DEV)


LENS = {"one": [1, 1], "empty": [0, 0], "pair": [5, 3], "ragged": [7, 0, 1, 130, 64, 65, 2, 0],
        "tiles": [4097, 4096, 1, 300, 8193, 2], "many": [3, 1, 0, 2] * 300, "long": [20011, 9003],
        "mostly_empty": [0] * 39 + [70001] + [0] * 20,
        "pairs": [3, 0, 700, 5, 1, 2, 2, 4, 1, 3] * 420, "crowd": [1, 2, 0, 3, 2, 1, 4, 1] * 2100}


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("lens", LENS.values(), ids=LENS.keys())
def test_next_token_labels(lens, masked):
    ops = _ops()
    n = sum(lens)
    ids = torch.randint(-3, 1000, (n,), generator=_gen(n), device=DEV)
    mask = torch.rand(n, generator=_gen(n + 1), device=DEV) < 0.5 if masked else None
    labels, rows = ops.next_token_labels(ids, ops.pack_plan(lens), mask)
    want, at = [], 0
    host, on = ids.tolist(), [True] * n if mask is None else mask.tolist()
    for x in lens:
        want += [host[t + 1] if t + 1 < at + x and on[t + 1] and host[t + 1] >= 0 else -1
                 for t in range(at, at + x)]
        at += x
    assert labels.tolist() == want and rows.tolist() == [w >= 0 for w in want]


# ---------------------------------------------------------------- preference loss

def _pref_exact(logp, ref, seq, on, nseq, kind, beta, smooth, margin, average):
    x = logp.double().detach().requires_grad_()
    d = x - (0.0 if ref is None else ref.double())
    d = torch.where(on, d, 0.0)
    s = torch.zeros(nseq, dtype=F64, device=DEV).index_add(0, seq, d)
    if average:
        s = s / torch.bincount(seq[on], minlength=nseq).clamp(min=1)
    h = s[0::2] - s[1::2]
    z = beta * h - margin
    if kind == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -(1 - smooth) * ls(z) - smooth * ls(-z)
    elif kind == "hinge":
        loss = torch.relu(1 - z)
    else:
        loss = (h - 0.5 / beta) ** 2
    loss = loss.mean()
    grad = torch.autograd.grad(loss, x, allow_unused=True)[0]
    return loss.detach(), beta * s.detach(), grad


PREF = [dict(), dict(label_smoothing=0.2, margin=0.5), dict(average=True, beta=2.0),
        dict(kind="hinge", margin=0.25), dict(kind="hinge", average=True, beta=3.0), dict(kind="ipo"),
        dict(kind="ipo", average=True, beta=0.5)]


@pytest.mark.parametrize("masked,with_ref", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("kw", PREF, ids=[str(k) for k in range(len(PREF))])
@pytest.mark.parametrize("lens", LENS.values(), ids=LENS.keys())
def test_preference_loss(lens, kw, masked, with_ref):
    ops = _ops()
    plan, seq, mask, logp, ref = _packing(lens, len(lens), 2, masked)
    on = _scored(lens, mask)
    full = {"kind": "sigmoid", "beta": 0.1, "label_smoothing": 0.0, "margin": 0.0, "average": False, **kw}
    ref = ref if with_ref else None
    loss, rewards, d = ops.preference_loss(logp, ref, plan, mask=mask, **kw)
    e_loss, e_rewards, e_d = _pref_exact(logp, ref, seq, on, len(lens), full["kind"], full["beta"],
                                         full["label_smoothing"], full["margin"], full["average"])
    # sums and pairs in 64 bits, each output rounded once
    _within(loss, e_loss, 2 * U32 * e_loss.abs() + 1e-12)
    _within(rewards, e_rewards, 2 * U32 * e_rewards.abs() + 1e-10)
    _within(d, e_d, 2 * U32 * e_d.abs() + 1e-13)
    assert (d[~on] == 0).all()


@pytest.mark.parametrize("lens", [LENS["ragged"], LENS["long"]], ids=["ragged", "long"])
def test_preference_loss_ignores_unscored_values(lens):
    ops = _ops()
    plan, seq, mask, logp, ref = _packing(lens, 3, 2)
    want = ops.preference_loss(logp, ref, plan, mask=mask)
    lo = torch.finfo(F32).min
    for v in (float("nan"), float("inf"), -float("inf"), lo):
        a, b = logp.masked_fill(~mask, v), ref.masked_fill(~mask, -v)
        for x, y in zip(ops.preference_loss(a, b, plan, mask=mask.view(torch.uint8)), want):
            assert torch.equal(x, y)
    # nothing scored at all: log 2, no gradient
    loss, rewards, d = ops.preference_loss(logp, ref, plan, mask=torch.zeros_like(mask))
    assert abs(loss.item() - math.log(2)) < 1e-7 and (rewards == 0).all() and (d == 0).all()


@pytest.mark.parametrize("lens", [[4, 3, 5, 2], [4000, 3000, 5000, 2000], [3000] * 4], ids=["small", "tiles", "pairs"])
def test_preference_loss_of_impossible_answers(lens):
    """A rejected answer of probability 0 costs nothing, a preferred one costs infinitely much; without a
    weight of its own the other term does not make it NaN."""
    ops = _ops()
    plan, seq, mask, logp, ref = _packing(lens, 3, 2, masked=False)
    first = [sum(lens[:i]) for i in range(4)]
    a = logp.clone()
    a[first[1]] = -float("inf")  # the first pair's rejected one
    loss, rewards, d = ops.preference_loss(a, ref, plan)
    assert rewards[1] == -float("inf") and loss.isfinite() and d.isfinite().all()
    assert (d[: first[2]] == 0).all()
    e = _pref_exact(logp, ref, seq, _scored(lens, None), 4, "sigmoid", 0.1, 0.0, 0.0, False)
    one = ops.preference_loss(logp[first[2]:].contiguous(), ref[first[2]:].contiguous(), ops.pack_plan(lens[2:]))
    _within(loss, one[0].double() / 2, 2 * U32 * loss.double() + 1e-12)
    assert e[0].isfinite()
    a = logp.clone()
    a[first[0]] = -float("inf")
    assert ops.preference_loss(a, ref, plan)[0] == float("inf")
    assert ops.preference_loss(a, ref, plan, label_smoothing=1.0)[0].isfinite()


@pytest.mark.parametrize("lens", [LENS["ragged"], LENS["tiles"]], ids=["ragged", "tiles"])
def test_preference_loss_extremes_and_scale(lens):
    """Sums far apart: the loss and its gradient keep their relative precision; grad_scale only
    scales the gradient."""
    ops = _ops()
    plan, seq, mask, logp, ref = _packing(lens, 5, 2)
    for scale in (300.0, 1e6):
        loss, rewards, d = ops.preference_loss(scale * logp, ref, plan, mask=mask, grad_scale=8.0)
        e = _pref_exact(scale * logp, ref, seq, mask, len(lens), "sigmoid", 0.1, 0.0, 0.0, False)
        _within(loss, e[0], 2 * U32 * e[0].abs())
        # 64-bit sums of values near 1e6 · 4: their errors reach the exponent, 1e-9 at most
        _within(d, 8 * e[2], (2 * U32 + 1e-8) * 8 * e[2].abs() + 1e-45)


@pytest.mark.parametrize("lens", [[5, 3, 9, 1], [5000, 4200]], ids=["small", "large"])
@pytest.mark.parametrize("kw", PREF, ids=[str(k) for k in range(len(PREF))])
def test_preference_loss_gradient_by_differences(lens, kw):
    """Central differences of the kernel's own loss; the step's loss changes are read in fp32."""
    ops = _ops()
    plan, seq, mask, logp, ref = _packing(lens, 6, 2)
    loss, _, d = ops.preference_loss(logp, ref, plan, mask=mask, **kw)
    way = torch.randn(len(logp), generator=_gen(9), device=DEV) * mask
    way = way / way.norm()
    e = 2.0 ** -7
    up, down = (ops.preference_loss(logp + s * e * way, ref, plan, mask=mask, **kw)[0].item() for s in (1, -1))
    slope = (d.double() * way.double()).sum().item()
    # loss read to U32 twice, the moved logp rounded (U32·4 each, spread over the rows), curvature
    # at most (beta or 2)²·e²
    per = d.double().abs()
    tol = (2 * U32 * max(loss.item(), 1.0) + 8 * U32 * per.sum().item()) / e + 9.0 * 4 * e * e
    assert abs((up - down) / (2 * e) - slope) < tol


# ---------------------------------------------------------------- policy loss

def _policy_exact(logp, old, A, ref, seq, on, nseq, low, high, coef, kl, reduction, divisor):
    x = logp.double().detach().requires_grad_()
    rows = on.nonzero()[:, 0]
    rho = (x[rows] - old.double()[rows]).exp()
    A = A.double()[rows] if A.shape[0] == len(logp) else A.double()[seq[rows]]
    a, b = rho * A, rho.clamp(1 - low, 1 + high) * A
    pol = -torch.minimum(a, b)
    k = torch.zeros_like(pol)
    if ref is not None:
        u = ref.double()[rows] - x[rows]
        k = torch.expm1(u) - u if kl == "k3" else u * u / 2
    count = torch.bincount(seq[rows], minlength=nseq).double()
    if reduction == "token":
        w = torch.full_like(pol, 1 / max(len(rows), 1)).detach()
    elif reduction == "sequence":
        w = (1 / (count[seq[rows]] * max(int((count > 0).sum()), 1))).detach()
    else:
        w = torch.full_like(pol, 1 / divisor).detach()
    P, K = (w * pol).sum(), (w * k).sum()
    loss = P + coef * K
    grad = torch.autograd.grad(loss, x)[0] if len(rows) else torch.zeros_like(logp, dtype=F64)
    share = (b < a).double().mean().item() if len(rows) else 0.0
    size = (w * (pol.abs() + abs(coef) * k)).sum().item(), (w * k).sum().item()
    gsize = torch.zeros(len(logp), dtype=F64, device=DEV)
    em = torch.expm1(u).abs() if ref is not None and kl == "k3" else (u.abs() if ref is not None else 0)
    gsize[rows] = (w * ((rho * A).abs() * (b >= a) + abs(coef) * em)).detach()
    return loss.detach(), P.detach(), K.detach(), share, grad, size, gsize


POLICY = [dict(), dict(ref=True, kl_coef=0.1), dict(ref=True, kl_coef=0.05, kl="k2", reduction="sequence"),
          dict(reduction="sequence", clip_low=0.1, clip_high=0.4), dict(ref=True, reduction="sum", divisor=7.0,
                                                                       kl_coef=-0.5),
          dict(clip_low=1.0, clip_high=float("inf"), reduction="sum")]


@pytest.mark.parametrize("masked,by_row", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("kw", POLICY, ids=[str(k) for k in range(len(POLICY))])
@pytest.mark.parametrize("lens", LENS.values(), ids=LENS.keys())
def test_policy_loss(lens, kw, masked, by_row):
    ops = _ops()
    plan, seq, mask, logp, noise, noise2, A = _packing(lens, len(lens) + 7, 4, masked)
    logp = logp - 3
    old, ref = logp + 0.4 * noise, logp + noise2
    A = A if by_row else torch.randn(len(lens), generator=_gen(2), device=DEV)
    kw = dict(kw)
    ref = ref if kw.pop("ref", False) else None
    on = _scored(lens, mask)
    loss, stats, d = ops.policy_loss(logp, old, A, plan, mask=mask, ref_logp=ref, **kw)
    f = {"clip_low": 0.2, "clip_high": 0.2, "kl_coef": 0.0, "kl": "k3", "reduction": "token", "divisor": 1.0, **kw}
    e_loss, P, K, share, e_d, (size, ksize), gsize = _policy_exact(
        logp, old, A, ref, seq, on, len(lens), f["clip_low"], f["clip_high"], f["kl_coef"], f["kl"],
        f["reduction"], f["divisor"])
    # a row's term: the ratio (argument rounded: |d| < 4, and exp 2 steps), the products, the weight, the
    # bounds and the coefficient, each U32; kl's polynomial some 12 more. The sums are in 64 bits.
    tol = 24 * U32
    _within(loss, e_loss, tol * size + 1e-30)
    _within(stats[0], P, tol * size + 1e-30)
    _within(stats[1], K, tol * ksize + 1e-30)
    _within(d, e_d, tol * gsize + 1e-30)
    assert abs(stats[2].item() - share) <= U32 and (d[~on] == 0).all()


@pytest.mark.parametrize("lens", [LENS["ragged"], LENS["long"]], ids=["ragged", "long"])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss_ignores_unscored_values(lens, reduction):
    ops = _ops()
    plan, seq, mask, logp, old, ref, A = _packing(lens, 11, 4)
    kw = dict(mask=mask, kl_coef=0.1, reduction=reduction)
    want = ops.policy_loss(logp, old, A, plan, ref_logp=ref, **kw)
    for v in (float("nan"), float("inf"), torch.finfo(F32).min):
        fill = lambda t: t.masked_fill(~mask, v)  # noqa: E731
        for x, y in zip(ops.policy_loss(fill(logp), fill(old), fill(A), plan, ref_logp=fill(ref), **kw), want):
            assert torch.equal(x, y)
    loss, stats, d = ops.policy_loss(logp, old, A, plan, mask=torch.zeros_like(mask), reduction=reduction)
    assert loss == 0 and (stats == 0).all() and (d == 0).all()


@pytest.mark.parametrize("n", [64, 20000])
def test_policy_loss_borders(n):
    """Ratios on and next to the clip's bounds, and KL terms from tiny to large, against 64 bits."""
    ops = _ops()
    lens = [n]
    plan = ops.pack_plan(lens)
    logp = -torch.rand(n, generator=_gen(1), device=DEV) - 1
    edge = torch.tensor([math.log(1.25), math.log(0.8)], dtype=F64, device=DEV).repeat(n // 2)
    old = (logp.double() - edge).float()
    step = torch.randint(-2, 3, (n,), generator=_gen(2), device=DEV)
    old = (old.view(torch.int32) + step.int()).view(F32)
    u = torch.logspace(-6, 1, n, device=DEV) * torch.where(torch.arange(n, device=DEV) % 3 > 0, 1.0, -1.0)
    ref = logp + u
    A = torch.where(torch.arange(n, device=DEV) % 4 < 2, 1.0, -1.0)
    seq, on = torch.zeros(n, dtype=torch.int64, device=DEV), _scored(lens, None)
    loss, stats, d = ops.policy_loss(logp, old, A, plan, ref_logp=ref, clip_low=0.2, clip_high=0.25, kl_coef=0.01)
    e_loss, P, K, share, e_d, (size, ksize), gsize = _policy_exact(
        logp, old, A, ref, seq, on, 1, 0.2, 0.25, 0.01, "k3", "token", 1.0)
    _within(loss, e_loss, 24 * U32 * size)
    _within(stats[1], K, 24 * U32 * ksize)
    _within(d, e_d, 24 * U32 * gsize + 1e-30)
    assert abs(stats[2].item() - share) <= U32


def test_losses_at_odd_addresses():
    """Rows that start anywhere in memory give the results of aligned ones."""
    ops = _ops()
    for lens in (LENS["ragged"], LENS["tiles"]):
        plan, seq, mask, logp, old, ref, A = _packing(lens, 13, 4)
        n = len(logp)

        def at(t, k):
            return torch.cat([t.new_zeros(k), t])[k:]

        want = (*ops.preference_loss(logp, ref, plan, mask=mask),
                *ops.policy_loss(logp, old, A, plan, mask=mask, ref_logp=ref, kl_coef=0.1, reduction="sequence"))
        for k in (1, 2, 3):
            a, b, c, e, m = at(logp, k), at(old, 1), at(ref, 2), at(A, 3), at(mask, k)
            got = (*ops.preference_loss(a, c, plan, mask=m),
                   *ops.policy_loss(a, b, e, plan, mask=m, ref_logp=c, kl_coef=0.1, reduction="sequence"))
            for x, y in zip(got, want):
                assert torch.equal(x, y)
        assert n == plan.n


@pytest.mark.parametrize("lens", [LENS["ragged"], LENS["tiles"], LENS["crowd"]], ids=["ragged", "tiles", "crowd"])
def test_any_byte_but_zero_is_set(lens):
    ops = _ops()
    plan, seq, mask, logp, old, ref, A = _packing(lens, 19, 4)
    n = len(logp)
    byte = torch.randint(1, 256, (n,), generator=_gen(5), device=DEV).to(torch.uint8)
    byte[::5], byte[1::5] = 128, 1
    byte = byte * mask
    ids = torch.arange(n, device=DEV)
    for f in (lambda m: ops.preference_loss(logp, ref, plan, mask=m),
              lambda m: ops.policy_loss(logp, old, A, plan, mask=m, ref_logp=ref, kl_coef=0.1),
              lambda m: ops.policy_loss(logp, old, A, plan, mask=m, reduction="sequence"),
              lambda m: ops.next_token_labels(ids, plan, m)):
        for x, y in zip(f(byte), f(mask)):
            assert torch.equal(x, y)


def test_losses_captured_and_on_a_side_stream():
    ops = _ops()
    for lens in (LENS["ragged"], LENS["long"]):
        sets = [_packing(lens, 70 + k, 4) for k in range(4)]
        plan = sets[0][0]
        mask, logp, old, ref, A = (t.clone() for t in sets[0][2:])

        def make():
            return (*ops.preference_loss(logp, ref, plan, mask=mask),
                    *ops.policy_loss(logp, old, A, plan, mask=mask, ref_logp=ref, kl_coef=0.1, reduction="sequence"),
                    *ops.policy_loss(logp, old, A, plan, mask=mask))

        def refresh(k):
            for t, s in zip((mask, logp, old, ref, A), sets[k][2:]):
                t.copy_(s)

        _replayed(make, refresh, make)
        side = torch.cuda.Stream()
        want = make()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = make()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_losses_of_nothing():
    ops = _ops()
    plan, none = ops.pack_plan([]), torch.empty(0, device=DEV)
    assert plan.n == 0 and plan.nseq == 0
    loss, stats, d = ops.policy_loss(none, none, none, plan, ref_logp=none, kl_coef=0.1, reduction="sequence")
    assert loss == 0 and (stats == 0).all() and d.shape == (0,)
    labels, rows = ops.next_token_labels(none.long(), plan)
    assert labels.shape == rows.shape == (0,)
    with pytest.raises(RuntimeError):
        ops.preference_loss(none, none, plan)


def test_loss_refusals_on_the_device():
    ops = _ops()
    plan, seq, mask, logp, ref = _packing([4, 5], 1, 2)
    for bad in (dict(logp=logp[:-1]), dict(logp=logp.double()), dict(ref_logp=ref.cpu()), dict(mask=mask.int()),
                dict(logp=torch.cat([logp, logp])[::2]), dict(kind="dpo")):
        with pytest.raises(ValueError):
            ops.preference_loss(**{"logp": logp, "ref_logp": ref, "plan": plan, **bad})
    for bad in (dict(adv=logp[:3]), dict(kl="k1"), dict(reduction="mean"), dict(old_logp=ref.half())):
        with pytest.raises(ValueError):
            ops.policy_loss(**{"logp": logp, "old_logp": ref, "adv": ref, "plan": plan, **bad})
    with pytest.raises(RuntimeError):
        ops.policy_loss(logp, ref, ref, plan, kl_coef=0.1)  # no reference policy


# ---------------------------------------------------------------- AdamW

def _mix(x):
    x = x & 0xffffffff
    x = x ^ (x >> 16)
    x = (x * 0x6a09e667) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0xbb67ae85) & 0xffffffff
    return x ^ (x >> 16)


def _numbers(nb, step, seed):
    key = _mix(torch.tensor(seed + step * 0x9e3779b9, device=DEV))
    key = _mix(key ^ _mix(torch.arange(nb, device=DEV)))
    x = _mix(key[:, None] + torch.arange(128, device=DEV) * 0x9e3779b9)
    return (torch.stack([x & 0xffff, x >> 16], 2).double() + 0.5).div(65536).view(nb, 256)


class Ref:
    """AdamW in 64 bits over the blocks of an ops.AdamW, from its moments as they are now."""

    def __init__(self, opt, ws, gs, groups):
        self.ws, self.opt, self.groups = ws, opt, groups
        self.w, self.g = self._blocks(ws), self._blocks(gs)
        self.live = self._blocks([torch.ones_like(w) for w in ws]) > 0
        s = opt.state()
        if opt.bits == 8:
            self.m = s["m"].float().double().view(-1, 256) * s["m_scale"].double()[:, None]
            self.v = (s["r"].float().double().view(-1, 256) * s["r_scale"].double()[:, None]) ** 2
        else:
            self.m, self.v = (s[k].double().view(-1, 256) for k in ("m", "v"))

    @staticmethod
    def _blocks(ts):
        pad = [torch.nn.functional.pad(t.reshape(-1).double(), (0, -t.numel() % 256)) for t in ts]
        return torch.cat(pad).view(-1, 256)

    def step(self, lr, step, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.0, max_norm=None, seed=0):
        g = self.g
        per = torch.repeat_interleave(torch.tensor(self.groups),
                                      torch.tensor([-(-w.numel() // 256) for w in self.ws])).to(DEV)
        self.norms = None
        if max_norm is not None:
            sq = torch.zeros(max(self.groups) + 1, dtype=F64, device=DEV).index_add(0, per, g.square().sum(1))
            self.norms = sq.sqrt()
            g = g * (max_norm / (self.norms + 1e-6)).clamp(max=1)[per, None]
        self.m_parts = (beta1 * self.m).abs() + ((1 - beta1) * g).abs()
        self.m = beta1 * self.m + (1 - beta1) * g
        self.v = beta2 * self.v + (1 - beta2) * g ** 2
        self.denom = (self.v / (1 - beta2 ** step)).sqrt() + eps
        self.update = lr / (1 - beta1 ** step) * self.m / self.denom
        self.update_size = lr / (1 - beta1 ** step) * self.m_parts / self.denom
        self.w = self.w - lr * wd * self.w - self.update
        self.unit = _numbers(len(self.m), step, seed)

    def check(self, dtype):
        opt, s = self.opt, self.opt.state()
        got = self._blocks(self.ws)
        # w: the decay's and the subtraction's rounding; the update: m's two roundings (against its
        # parts), sqrt and reciprocal (a step each), the products: 16 steps in all; then its own type's
        tol = 4 * U32 * self.w.abs() + 16 * U32 * self.update_size + 1e-30
        if dtype == BF16:
            tol = tol + U16 * (self.w.abs() + tol)
        _within(got[self.live], self.w[self.live], tol[self.live])
        assert (got[~self.live] == 0).all()
        if opt.bits == 32:
            _within(s["m"].view(-1, 256), self.m, 6 * U32 * self.m_parts + 1e-38)
            _within(s["v"].view(-1, 256), self.v, 8 * U32 * self.v + 1e-38)
            return
        r = self.v.sqrt()
        ms, rs = self.m.abs().amax(1) / 448, r.amax(1) / 448
        _within(s["m_scale"], ms, 8 * U32 * self.m_parts.amax(1) / 448 + 1e-33)
        _within(s["r_scale"], rs, 8 * U32 * rs + 1e-33)
        m = s["m"].float().double().view(-1, 256) * s["m_scale"].double()[:, None]
        q = s["r"].float().double().view(-1, 256) * s["r_scale"].double()[:, None]
        # nearest: half a step of 3 mantissa bits, or half the smallest step; at random: a whole one
        _within(m, self.m, 2.0 ** -4 * self.m.abs() + 2.0 ** -10 * ms[:, None] + 16 * U32 * self.m_parts + 1e-33)
        _within(q, r, 2.0 ** -3 * r + 2.0 ** -9 * rs[:, None] + 16 * U32 * r + 1e-33)
        assert ((s["r"].float().view(-1, 256) > 0) == (r > 0)).all()
        # and each code is the formula's, up to the error of its value in fp32 (16 steps of its parts and
        # of the scale): it lies between the codes of the value less and plus that. (On bf16 gradients
        # many values lie on a border exactly.)
        unit = lambda t, sc: torch.where(sc[:, None] > 0, t / sc[:, None], 0.0)  # noqa: E731

        def code(x):
            x = x.clamp(0, 448)
            e = torch.frexp(x)[1]
            grid = ((e.clamp(min=-5) - 4 + 1023).long() << 52).view(F64)  # 2^(e − 4), exactly
            c = torch.floor(x / grid + self.unit) * grid
            return torch.where(x > 0, c.clamp(2.0 ** -9, 448.0), 0.0)

        x, got = unit(r, rs), s["r"].float().double().view(-1, 256)
        assert ((code(x * (1 - 16 * U32)) <= got) & (got <= code(x * (1 + 16 * U32)))).all()
        # to nearest, the ends rounded to fp32 outwards
        x, off = unit(self.m, ms), 16 * U32 * unit(self.m_parts, ms)
        near = lambda v, to: torch.nextafter(v.float(), v.new_tensor(to, dtype=F32)).clamp(-448, 448).to(F8).float()  # noqa: E731
        got = s["m"].float().view(-1, 256)
        assert ((near(x - off, -math.inf) <= got) & (got <= near(x + off, math.inf))).all()
        # nearly all are the value's own
        assert (got != near(x, 0.0)).double().mean().item() < 0.01


SIZES = {"one": [1], "block": [256, 255, 257], "ragged": [3, 4096, 1, 4097, 0, 12289, 100], "many": [70, 513, 2] * 60,
         "large": [1 << 20, 333]}


def _adam_inputs(sizes, dtypes, seed, shift):
    g = _gen(seed)

    def make(n, dt, scale):
        x = torch.randn(n + shift, generator=g, device=DEV) * scale
        return x.to(dt)[shift:]

    return ([make(n, dtypes[0], 0.05) for n in sizes], [make(n, dtypes[1], 1e-3) for n in sizes])


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtypes", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)], ids=["ff", "bb", "fb", "bf"])
@pytest.mark.parametrize("clip", [None, 0.01, 1e4])
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_adamw(sizes, clip, dtypes, bits):
    ops = _ops()
    groups = [i // 3 for i in range(len(sizes))]
    shift = len(sizes) % 2
    ws, gs = _adam_inputs(sizes, dtypes, 17, shift)
    opt = ops.AdamW(ws, gs, bits=bits, groups=groups)
    for step in (1, 2, 3):
        for i, x in enumerate(gs):
            x.copy_(torch.randn(x.shape, generator=_gen(100 * step + i), device=DEV) * 10.0 ** (step - 4))
        kept = [x.clone() for x in gs]
        ref = Ref(opt, ws, gs, groups)
        hyper = dict(lr=1e-2, step=step, wd=0.1, max_norm=clip, seed=step * 7)
        norms = opt.step(**hyper)
        ref.step(**hyper)
        ref.check(dtypes[0])
        if clip is None:
            assert norms is None
        else:
            _within(norms, ref.norms, 4 * U32 * ref.norms)
        assert all(torch.equal(a, b) for a, b in zip(gs, kept))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("clip", [None, 0.01])
def test_adamw_codes_of_elementary_operations(clip, dtype):
    """8-bit moments, codes and scales, are bit for bit those of the formula taken in fp32 with every
    operation rounded, step after step: no tolerance. (Quotients and roots in 64 bits, then in 32, are
    rounded as one operation in 32 is: 53 bits are 2·24 + 2 and more.)"""
    ops = _ops()
    sizes = [(1 << 18) + 5, 333, 4096]
    groups = [0, 0, 1]
    ws, gs = _adam_inputs(sizes, (dtype, dtype), 29, 0)
    opt = ops.AdamW(ws, gs, bits=8, groups=groups)
    b1, b2 = 0.9, 0.999
    for step in (1, 2, 3):
        for i, x in enumerate(gs):
            x.copy_(torch.randn(x.shape, generator=_gen(10 * step + i), device=DEV) * 10.0 ** (step - 4))
        ref = Ref(opt, ws, gs, groups)
        old = {k: v.float().cpu() for k, v in opt.state().items()}
        hyper = dict(lr=1e-3, step=step, max_norm=clip, seed=5)
        opt.step(**hyper)
        ref.step(**hyper)
        g = ref.g.float().cpu()
        if clip is not None:
            factor = ((1 / (ref.norms.float().cpu() + 1e-6).double()).float() * clip).clamp(max=1)
            per = torch.repeat_interleave(torch.tensor(groups), torch.tensor([-(-n // 256) for n in sizes]))
            g = g * factor[per, None]
        m = b1 * (old["m"].view(-1, 256) * old["m_scale"][:, None]) + (1 - b1) * g
        r = (old["r"].view(-1, 256) * old["r_scale"][:, None]).square()
        r = (b2 * r + (1 - b2) * g.square()).double().sqrt().float()
        unit = torch.tensor(1 / 448)
        ms, top = m.abs().amax(1) * unit, r.amax(1)
        want = torch.where(ms[:, None] > 0, m.double() / ms.double()[:, None], 0.0).float().clamp(-448, 448).to(F8).float()
        x = torch.where(top[:, None] > 0, r * ((1 / top.double()).float() * 448)[:, None], 0.0).clamp(max=448).double()
        grid = torch.ldexp(torch.ones_like(x), torch.frexp(x)[1].clamp(min=-5) - 4)
        q = (torch.floor(x / grid + ref.unit.double().cpu()) * grid).clamp(2.0 ** -9, 448.0)
        got = {k: v.float().cpu() for k, v in opt.state().items()}
        assert torch.equal(got["m_scale"], ms) and torch.equal(got["r_scale"], top * unit)
        assert torch.equal(got["m"].view(-1, 256), want)
        assert torch.equal(got["r"].view(-1, 256), torch.where(x > 0, q, 0.0).float())


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_values_of_all_sizes(bits):
    """Blocks of zeros, of one value, of gradients over 12 decades; beta1 = 0, beta2 = 0."""
    ops = _ops()
    g = torch.zeros(256 * 6, device=DEV)
    g[256:512] = 0.25
    g[512:768] = 10.0 ** torch.linspace(-12, 0, 256, device=DEV)
    g[768] = 1e-9
    g[1024:1280] = torch.randn(256, generator=_gen(1), device=DEV) * 1e12
    w = torch.randn(g.shape, generator=_gen(2), device=DEV)
    for b1, b2 in ((0.9, 0.999), (0.0, 0.0)):
        opt = ops.AdamW([w], [g], bits=bits)
        for step in (1, 2):
            ref = Ref(opt, [w], [g], [0])
            hyper = dict(lr=1e-3, step=step, beta1=b1, beta2=b2, seed=5)
            opt.step(**hyper)
            ref.step(**hyper)
            ref.check(F32)


def test_adamw_second_moment_moves_on_average():
    """A second moment that decays by 0.1 % a step, under a step of its code: its mean over many
    elements follows 0.999^t; to nearest it would stay where it is. Bound: each step's rounding adds at
    most a variance of a quarter of a grid step squared (2^-3 relative), 200 steps, 65536 elements, 6
    standard deviations of the mean."""
    ops = _ops()
    n, steps = 65536, 200
    w, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    opt = ops.AdamW([w], [g], bits=8)
    r0 = (torch.rand(n, generator=_gen(4), device=DEV) * 200 + 50).to(F8)
    r0[::256] = 448.0  # the block's largest
    s = opt.state()
    s["r"].copy_(r0)
    s["r_scale"].fill_(1e-3)
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[::256] = False
    for step in range(1, steps + 1):
        opt.step(lr=0.0, step=step, seed=1)
    got = (s["r"].float().double().view(-1, 256) * s["r_scale"].double()[:, None]).view(-1)[keep]
    start = (r0.float().double() * 1e-3)[keep]
    ratio = (got / start).mean().item()
    want = 0.999 ** (steps / 2)
    assert abs(ratio - want) < 6 * math.sqrt(steps) * 0.5 * 2.0 ** -3 / math.sqrt(n)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_shows_gradients_that_are_not_numbers(bits, bad):
    """Without a clip they reach their own weight and (8 bits) their block's moments; no other."""
    ops = _ops()
    ws, gs = _adam_inputs([1000, 300], (F32, F32), 3, 0)
    clean, _ = _adam_inputs([1000, 300], (F32, F32), 3, 0)
    ops.AdamW(clean, gs, bits=bits).step(lr=1e-3, step=1)
    gs[0][300] = bad
    opt = ops.AdamW(ws, gs, bits=bits)
    opt.step(lr=1e-3, step=1)
    assert ws[0][300].isnan()
    ws[0][300] = clean[0][300]
    assert torch.equal(ws[0], clean[0]) and torch.equal(ws[1], clean[1])
    opt.step(lr=1e-3, step=2)
    hit = ws[0].isnan().nonzero()[:, 0].tolist()
    assert hit == (list(range(256, 512)) if bits == 8 else [300])
    assert not ws[1].isnan().any()


def test_adamw_same_steps_same_bits_and_saved_moments():
    ops = _ops()
    runs = []
    for resume in (False, True):
        ws, gs = _adam_inputs([5000, 77], (F32, F32), 8, 0)
        opt = ops.AdamW(ws, gs, bits=8, groups=[0, 1])
        for step in range(1, 6):
            if resume and step == 3:  # saved and taken up by another
                saved = {k: v.clone() for k, v in opt.state().items()}
                opt = ops.AdamW(ws, gs, bits=8, groups=[0, 1])
                for k, v in saved.items():
                    opt.state()[k].copy_(v)
            opt.step(lr=1e-3, step=step, max_norm=0.5, seed=3)
        runs.append([*ws, *(v.view(torch.uint8) for v in opt.state().values())])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_captured_with_device_lr_and_step(bits):
    ops = _ops()
    sizes = [9000, 130, 1]
    ws, gs = _adam_inputs(sizes, (F32, F32), 21, 0)
    we, _ = _adam_inputs(sizes, (F32, F32), 21, 0)
    opt, eager = ops.AdamW(ws, gs, bits=bits), ops.AdamW(we, gs, bits=bits)
    lr, step = torch.tensor([1e-2], device=DEV), torch.tensor([1], device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = opt.step(lr, step, wd=0.1, max_norm=0.02, seed=9)
    for k in range(1, 6):
        lr.fill_(1e-2 / k)
        step.fill_(k)
        for i, g in enumerate(gs):
            g.copy_(torch.randn(g.shape, generator=_gen(10 * k + i), device=DEV))
        graph.replay()
        want = eager.step(lr.item(), k, wd=0.1, max_norm=0.02, seed=9)
        torch.cuda.synchronize()
        assert torch.equal(norms, want), k
        for a, b in zip(ws, we):
            assert torch.equal(a, b), k
        for a, b in zip(opt.state().values(), eager.state().values()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), k


def test_adamw_refusals_on_the_device():
    ops = _ops()
    x = torch.zeros(1000, device=DEV)
    y = torch.zeros(1000, device=DEV)
    for bad in (dict(ws=[x, x], gs=[y, y]), dict(ws=[x[:600], x[500:]], gs=[y[:600], y[500:]]),
                dict(ws=[x[:500]], gs=[x[499:999]]), dict(ws=[x], gs=[y.cpu()]), dict(ws=[x[::2]], gs=[y[::2]])):
        with pytest.raises(ValueError):
            ops.AdamW(**bad)
    opt = ops.AdamW([x[:500], x[500:]], [y[:500], y[:500]])  # a gradient may be shared
    for bad in (dict(step=0), dict(lr=float("nan")), dict(beta1=1.0), dict(eps=-1.0)):
        with pytest.raises(RuntimeError):
            opt.step(**{"lr": 1e-3, "step": 1, **bad})
    for bad in (dict(max_norm=-1.0), dict(lr=torch.zeros(2, device=DEV)), dict(step=torch.zeros(1, device=DEV))):
        with pytest.raises(ValueError):
            opt.step(**{"lr": 1e-3, "step": 1, **bad})
    empty = ops.AdamW([x[:0]], [y[:0]])
    assert empty.step(1e-3, 1, max_norm=1.0).tolist() == [0.0]
    gaps = ops.AdamW([x[:10], x[10:20]], [y[:10], y[10:20]], groups=[1, 4])
    y[:20] = 3.0
    assert gaps.step(1e-3, 1, max_norm=1.0).tolist() == [0.0, y[:10].norm().item(), 0.0, 0.0, y[:10].norm().item()]


def test_adamw_matches_the_fp32_step():
    """32-bit moments against clip_adamw_, the framework's other step, over several groups."""
    ops = _ops()
    sizes, groups = [5000, 300, 70, 4096], [0, 0, 1, 2]
    ws, gs = _adam_inputs(sizes, (F32, F32), 31, 0)
    wc, gc = [w.clone() for w in ws], [g.clone() for g in gs]
    ms, vs = [torch.zeros_like(w) for w in ws], [torch.zeros_like(w) for w in ws]
    opt = ops.AdamW(ws, gs, bits=32, groups=groups)
    for step in (1, 2, 3):
        gc = [g.clone() for g in gs]
        opt.step(lr=1e-3, step=step, wd=0.05, max_norm=0.02)
        ops.clip_adamw_(wc, gc, ms, vs, groups, 1e-3, step, wd=0.05, max_norm=0.02)
    for a, b in zip(ws, wc):
        # 1 − beta2 is rounded from 64 bits here, taken in fp32 there: 5e-5 of v, half of it in the update
        assert (a - b).abs().max().item() < 3 * 1e-3 * 1e-4 + 8 * U32


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("loss", ["preference", "policy"])
def test_feedback_step(loss):
    """Packed ids to labels, log probabilities through the head, a loss, the rows' gradient through
    the head and the final norm, an adapter's gradient and its step: gradients against autograd in 64
    bits on the same inputs, and differences of the loss along the adapter."""
    ops = _ops()
    g = _gen(40)
    lens = [20, 31, 1, 17, 40, 25]
    n, D, V, r = sum(lens), 128, 1500, 16
    plan = ops.pack_plan(lens)
    ids = torch.randint(0, V, (n,), generator=g, device=DEV)
    labels, rows = ops.next_token_labels(ids, plan, mask=torch.rand(n, generator=g, device=DEV) < 0.7)
    W = (torch.randn(V, D, generator=g, device=DEV) * 0.3).to(BF16)
    norm = torch.ones(D, dtype=BF16, device=DEV)
    X = torch.randn(n, D, generator=g, device=DEV).to(BF16)
    A = (torch.randn(r, D, generator=g, device=DEV) * 0.1).to(BF16)
    B = torch.randn(D, r, generator=g, device=DEV) * 0.05
    ref = -torch.rand(n, generator=g, device=DEV) * 3 - 5
    adv = torch.randn(len(lens), generator=g, device=DEV)

    def forward(B):
        Z = ops.lora_skinny(X, A)
        h = ops.gemm_nt(Z, B.to(BF16), R=X)
        return Z, h, ops.rmsnorm(h, norm, 1e-5)

    def the_loss(logp, old):
        if loss == "preference":
            return ops.preference_loss(logp, ref, plan, mask=rows)
        return ops.policy_loss(logp, old, adv, plan, mask=rows, ref_logp=ref, kl_coef=0.02, reduction="sequence")

    Z, h, normed = forward(B)
    logp, other = ops.token_logprobs(normed, W, labels)
    old = logp + 0.05
    value, _, dlogp = the_loss(logp, old)
    dn = ops.token_logprobs_backward(normed, W, labels, logp, other, dlogp)
    dh = ops.rmsnorm_backward(h, dn, norm, 1e-5)
    gB = torch.empty(D, r, device=DEV)
    ops.lora_tn(Z, dh, r, True, [gB])

    # the same in 64 bits from the same rows h
    x = h.double().detach().requires_grad_()
    nx = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5)
    lp = torch.log_softmax(nx @ W.double().t(), 1)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(DEV)
    picked = torch.where(rows, lp.gather(1, labels.clamp(min=0)[:, None])[:, 0], 0.0)
    if loss == "preference":
        s = torch.zeros(len(lens), dtype=F64, device=DEV).index_add(0, seq, torch.where(rows, picked - ref, 0.0))
        exact = -torch.nn.functional.logsigmoid(0.1 * (s[0::2] - s[1::2])).mean()
    else:
        rho = torch.exp(picked - old.double())
        Ad = adv.double()[seq]
        u = ref.double() - picked
        term = -torch.minimum(rho * Ad, rho.clamp(0.8, 1.2) * Ad) + 0.02 * (torch.expm1(u) - u)
        count = torch.bincount(seq[rows], minlength=len(lens)).double()
        exact = (torch.where(rows, term, 0.0) / (count[seq].clamp(min=1) * (count > 0).sum())).sum()
    want, = torch.autograd.grad(exact, x)
    # the rows pass the norm's bf16 (2 roundings: normed, dn), q's and dh's: a share of each, in norm
    rel = (dh.double() - want).norm() / want.norm()
    assert rel < 6 * U16, rel
    wantB = want.t() @ Z.double()
    assert ((gB.double() - wantB).norm() / wantB.norm()).item() < 8 * U16

    before = B.clone()
    opt = ops.AdamW([B], [gB], bits=8)
    opt.step(lr=1e-3, step=1, max_norm=1.0)
    # a first step moves each element by lr against its gradient's sign (eps aside)
    big = gB.abs() > 1e-4 * gB.abs().max()
    moved = (before - B)[big] / gB[big].sign()
    scale = min(1.0, 1.0 / (gB.norm().item() + 1e-6))
    expect = 1e-3 * (gB[big].abs() * scale) / (gB[big].abs() * scale + 1e-8)
    assert ((moved - expect).abs() <= 64 * U32 * 1e-3 + 2 * U32 * before[big].abs()).all()
