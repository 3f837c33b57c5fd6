"""The operators for training from feedback at the ends of their ranges: labels far above the
other words, KL terms of weight 0, ratios and gradient norms past fp32. Against the formulas in 64
bits; U32 and U16 as in test_gpu_feedback."""

from __future__ import annotations

import pytest
import torch

from test_gpu_feedback import BF16, DEV, F32, U16, U32, Ref, _gen, _head_exact, _head_tol, _ops, \
    _packing, _policy_exact, _within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


# ---------------------------------------------------------------- log probabilities

def _leads(n, V, label, seed, near=None):
    """Rows whose label lies from 160 logits below to 160 above the other words (about 0 each); near:
    another word that lies that far below the label where that is above the rest."""
    D, g = 64, _gen(seed)
    W = torch.zeros(V, D, device=DEV)
    W[:, 2:] = torch.randn(V, D - 2, generator=g, device=DEV) * 0.05
    W[label, 0] = 1
    H = torch.randn(n, D, generator=g, device=DEV)
    H[:, 0] = torch.linspace(-160, 160, n, device=DEV)
    H[:, 1] = 0
    if near is not None:
        W[near[0], 1] = 1
        H[:, 1] = H[:, 0] - near[1]
    return H.to(BF16), W.to(BF16), torch.full((n,), label, device=DEV)


# label in the first, a middle and the last place; alone in the last run of 128 columns (129, 257); past
# 65536 words a narrower product takes the last ones of up to 256 rows
LEADS = [(200, 2, 0, None), (200, 2, 1, None), (200, 31, 4, None), (200, 128, 127, None), (200, 129, 128, None),
         (300, 257, 256, None), (200, 777, 5, (6, 84.0)), (200, 777, 5, (700, 60.0)), (300, 5000, 4321, (17, 92.0)),
         (130, 70001, 69999, None), (130, 70001, 40000, (41, 84.0)), (300, 70001, 3, (65900, 100.0))]


@pytest.mark.parametrize("n,V,label,near", LEADS)
def test_logprobs_of_labels_far_above_the_rest(n, V, label, near):
    """other is the plain log-sum-exp however far the label leads, and logp keeps its relative precision
    down to the smallest normal number."""
    ops = _ops()
    H, W, lab = _leads(n, V, label, V + label, near)
    logp, other = ops.token_logprobs(H, W, lab)
    e_logp, e_other, q = _head_exact(H, W, lab)
    ex, tol = _head_tol(H, W)
    _within(other, e_other, tol + 4 * U32 * e_other.abs())
    # the exponent other − x_t: both numbers' errors; and its own two halves' (256·U32)
    rel = ex + tol + (256 + 8) * U32
    _within(logp, e_logp, rel * e_logp.abs() + 2.0 ** -126)
    d = torch.ones(n, device=DEV)
    got = ops.token_logprobs_backward(H, W, lab, logp, other, d, out_dtype=F32)
    W64 = W.double()
    want = -e_logp.expm1()[:, None] * (W64[label] - q @ W64)
    spread = -e_logp.expm1()[:, None] * (q @ W64.abs() + W64[label].abs())
    _within(got, want, (2 * (U16 + ex + tol + e_other.abs() * U32 + 256 * U32) + 1024 * U32 + rel)[:, None] * spread
            + 2.0 ** -120)


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("word", [3, 100, 300])
def test_logprobs_show_words_that_are_not_numbers(n, word):
    """A NaN among the head's words is seen in every row, whether its run holds the label, leads or
    neither."""
    ops = _ops()
    H, W, lab = _leads(n, 400, 5, 1)
    W[word] = float("nan")
    logp, other = ops.token_logprobs(H, W, lab)
    assert logp.isnan().all() and other.isnan().all()


# ---------------------------------------------------------------- policy loss

@pytest.mark.parametrize("lens", [[40, 3, 61], [5000, 20, 6000]], ids=["small", "large"])
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
@pytest.mark.parametrize("kl", ["k3", "k2"])
def test_policy_loss_watches_a_kl_of_weight_0(lens, reduction, kl):
    """With kl_coef = 0 the reference enters the second statistic alone, also where its term is
    infinite."""
    ops = _ops()
    plan, seq, mask, logp, old, A = _packing(lens, 3, 3)
    logp, old = logp - 100, old - 100
    ref = logp + 0.3
    rows = mask.nonzero()[:, 0]
    ref[rows[2]] = logp[rows[2]] + 95
    kw = dict(mask=mask, reduction=reduction, kl=kl)

    def same(logp):
        loss, stats, d = ops.policy_loss(logp, old, A, plan, ref_logp=ref, **kw)
        want = ops.policy_loss(logp, old, A, plan, **kw)
        assert loss.isfinite() and d.isfinite().all()
        assert torch.equal(loss, want[0]) and torch.equal(d, want[2])
        assert torch.equal(stats[[0, 2]], want[1][[0, 2]])
        return stats[1]

    seen = same(logp)
    assert seen.isinf() if kl == "k3" else seen.isfinite() and seen > 0
    logp[rows[5]] = -float("inf")  # of probability 0
    assert same(logp).isinf()


@pytest.mark.parametrize("lens", [[64], [20000]], ids=["small", "large"])
def test_policy_loss_of_ratios_past_fp32(lens):
    """Ratios e^89 to e^120, whose product with the advantage is 0 or within fp32."""
    ops = _ops()
    n = sum(lens)
    plan, seq, mask, A = _packing(lens, 9, 1)
    logp = -torch.rand(n, generator=_gen(1), device=DEV)
    old = logp - torch.linspace(60, 120, n, device=DEV)
    A = A * 1e-20
    A[::3] = 0.0
    loss, stats, d = ops.policy_loss(logp, old, A, plan, mask=mask, reduction="sum", divisor=3.0)
    e_loss, P, K, share, e_d, (size, _), gsize = _policy_exact(
        logp, old, A, None, seq, mask, 1, 0.2, 0.2, 0.0, "k3", "sum", 3.0)
    # the ratio's argument is rounded: 2^7·U32 relative in the ratio; the rest as for other rows
    tol = (2 ** 7 + 24) * U32
    _within(loss, e_loss, tol * size + 1e-30)
    _within(d, e_d, tol * gsize + 1e-30)
    assert abs(stats[2].item() - share) <= U32


# ---------------------------------------------------------------- AdamW

@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("size", [1000, (1 << 20) + 5000])
@pytest.mark.parametrize("max_norm", [1.0, 1e20, 1e-3])
@pytest.mark.parametrize("dtypes", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)], ids=["ff", "bb", "bf", "fb"])
def test_adamw_clips_gradients_of_any_finite_size(bits, size, max_norm, dtypes):
    """Norms from 2^126 on, past fp32's range: the group is clipped to max_norm as any other, and the
    groups beside it are not touched by it."""
    ops = _ops()
    g = [torch.randn(k, generator=_gen(k), device=DEV) for k in (size, 700)]
    g[0] = (g[0].clamp(-3, 3) * 1e38)
    g = [x.to(dtypes[1]) for x in g]
    w = [torch.randn(k, generator=_gen(k + 1), device=DEV).to(dtypes[0]) for k in (size, 700)]
    w2 = w[1].clone()
    opt = ops.AdamW(w, g, bits=bits, groups=[0, 1])
    for step in (1, 2):
        ref = Ref(opt, w, g, [0, 1])
        hyper = dict(lr=1e-2, step=step, wd=0.1, max_norm=max_norm, seed=5)
        norms = opt.step(**hyper)
        ref.step(**hyper)
        assert norms[0] > 1e38 and norms[1].isfinite()
        ref.check(dtypes[0])
    alone = ops.AdamW([w2], [g[1]], bits=bits)
    for step in (1, 2):
        alone.step(lr=1e-2, step=step, wd=0.1, max_norm=max_norm, seed=5)
    if bits == 32:  # (8 bits: rounded at random by the block's number)
        assert torch.equal(w[1], w2)
