"""A decoder block's memory-bound operators at the ends of their ranges: 8-bit rows next to the largest finite
value, rotary angles of far positions against exact arithmetic."""

from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _ops():
    from deltaserve_amd import ops

    return ops


# ---------------------------------------------------------------- 8-bit rows

# the scale of the blocks whose largest magnitude may round to 2^128 (steps of 16 there in e4m3, of 1 in int8), and
# their last code below it
LAST = {"e4m3": (2.0 ** 120, 240), "int8": (2.0 ** 122, 63)}


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("w", [32, 75])
def test_finite_values_come_back_finite(w, dtype, code):
    """Values that would round to 2^128 take the code below; the others are rounded as ever, in their blocks too."""
    ops = _ops()
    one, last = LAST[code]
    top = torch.finfo(dtype).max
    x = torch.randn(7, w, generator=torch.Generator(device=DEV).manual_seed(w), device=DEV)
    x = x.clamp(-3, 3) * 2.0 ** 125  # (less than 2^127)
    x[0, 3], x[1, 5], x[1, 6] = top, -top, top
    x[2, 7] = last * one  # kept as it is
    x[3, w - 1] = -(last + 0.375) * one  # rounds to it, in bf16 to the next
    x[4, 0] = (last + (10 if code == "e4m3" else 0.625)) * one  # rounds past it
    x[5, 1] = {"e4m3": 448 * 2.0 ** 119, "int8": 127 * 2.0 ** 121}[code]  # the largest of the scale below
    x = x.to(dtype)
    q = ops.pack_rows8(x, code=code)
    scale = torch.exp2(q.scales.double() - 127).repeat_interleave(32, 1)[:, :w]
    v = x.double() / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3) if code == "e4m3" else 1.0
    want = (v / step).round() * step * scale
    past = want.abs() >= 2.0 ** 128
    assert past.sum() >= 3  # (in bf16 x[4, 0] is 127·2^121 of int8, which stays)
    want = torch.where(past, last * one * want.sign(), want)
    for got in (ops.unpack_rows8(q).double(), ops.unpack_rows8(q, F32).double()):
        assert got.isfinite().all()
        assert torch.equal(got, want)
        assert got[0, 3] == last * one and got[1, 5] == -last * one and got[5, 1] == x[5, 1]
    lost = ops.unpack_rows8(ops.pack_rows8(x.index_fill(1, torch.tensor([3], device=DEV), math.inf), code=code))
    assert lost[:, :32].isnan().all() and lost[:, 32:].isfinite().all()
    # the sum with a residual, which is finite too
    r = torch.zeros_like(x)
    same = ops.pack_rows8(x, r, code=code)
    assert torch.equal(same.codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(same.scales, q.scales)


# ---------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("n,heads,hd,ldy,hy", [(5, 4, 64, 256, 64), (5, 4, 64, 64, 320), (3, 3, 64, 212, 74),
                                               (3, 3, 64, 74, 212), (1, 4, 64, 64, 64), (5, 1, 64, 64, 64)])
def test_rotary_outputs_as_close_as_they_may_be(n, heads, hd, ldy, hy):
    ops = _ops()
    plan = ops.rotary_plan(hd, 1e4)
    x = torch.randn(n, heads, hd, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(BF16)
    pos = torch.arange(n, device=DEV) + 3
    mem = torch.full(((n - 1) * ldy + (heads - 1) * hy + hd + 8,), 7.0, device=DEV, dtype=BF16)
    out = mem.as_strided((n, heads, hd), (ldy, hy, 1))
    want = ops.rotary(x, pos, plan)
    assert torch.equal(ops.rotary(x, pos, plan, out=out), want)
    at = torch.arange(mem.numel(), device=DEV).as_strided((n, heads, hd), (ldy, hy, 1)).flatten()
    assert at.unique().numel() == at.numel() == want.numel()
    assert (mem.index_fill(0, at, 7.0) == 7).all()


PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


def _exact_cos_sin(pos, turns, rounded=False):
    """cos and sin (64 bits) of 2π·pos·turns, the product and its reduction without any rounding; rounded: the
    reduced half turns as fp32 has them."""
    ang = []
    for p in pos.tolist():
        for t in turns:
            u = p * t
            half = 2 * (u - round(u))
            ang.append(float((Fraction(float(np.float32(float(half)))) if rounded else half) * PI))
    ang = torch.tensor(ang, dtype=F64).view(len(pos), 1, len(turns)).to(DEV)
    return ang.cos(), ang.sin()


def _far(lo, hi, n=128, heads=64):
    """A plan of 8 pairs, all of them fast, positions in [lo, hi), and heads of 8 pairs."""
    g = torch.Generator().manual_seed(9)
    inv = 0.5 + 0.5 * torch.rand(8, generator=g, dtype=F64)
    inv[0] = 1.0
    plan = _ops().RotaryPlan(16, 16, False, inv.numpy(), 1.0, DEV)
    pos = torch.randint(lo, hi, (n,), generator=g).to(DEV)
    return plan, pos, torch.randn(n, heads, 16, generator=g).to(DEV)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("lo,hi", [(1, 1 << 12), (1 << 20, 1 << 21), (1 << 30, (1 << 31) - 1)])
def test_rotary_angles_are_exact_to_fp32(lo, hi, back):
    """The root mean square error of fp32 results against the angles that the plan's table stands for. In units of
    2^-24 and of the result's root mean square: a cosine or sine 0.5 (its rounding and its correction's, 0.25 each in
    root mean square, times √2 as two of them meet), a product 0.3, the sum 0.42: 0.7, 4.2e-8. An angle rounded to
    fp32 adds 4.1e-8 (2^-25 half turns in the upper half of the range, half of that in the quarter below, ...), one
    whose product with the position is rounded to 64 bits up to 1.1e-7 at 2^31: 5.8e-8 and more."""
    ops = _ops()
    plan, pos, x = _far(lo, hi)
    got = (ops.rotary_backward if back else ops.rotary)(x, pos, plan).double()
    p, q = x[..., :8].double(), x[..., 8:].double()
    for rounded in (False, True):  # (the second: what the bound does not let through)
        c, s = _exact_cos_sin(pos, [Fraction(t) for t in plan.turns.tolist()], rounded)
        s = -s if back else s
        want = torch.cat([p * c - q * s, q * c + p * s], 2)
        rms = float(((got - want) ** 2).mean().sqrt() / (want ** 2).mean().sqrt())
        assert (rms > 5e-8) if rounded else (rms < 5e-8), rms


@pytest.mark.parametrize("lo,hi", [(1 << 28, 1 << 29), (1 << 30, (1 << 31) - 1)])
def test_rotary_angles_of_far_positions(lo, hi):
    """Against the plan's frequencies: a table entry, the frequency over 2π in 64 bits, is off by 2^-52 of itself at
    most. Cosine and sine are off by 2 units of 2^-24 and their correction's rounding by 1, the products and their
    sum by 1 each of |p| + |q|."""
    ops = _ops()
    plan, pos, x = _far(lo, hi)
    c, s = _exact_cos_sin(pos, [Fraction(float(f)) / (2 * PI) for f in plan.inv_freq])
    p, q = x[..., :8].double(), x[..., 8:].double()
    off = 2.0 ** -52 * pos.double()[:, None, None] * torch.from_numpy(plan.inv_freq).to(DEV) + 5 * 2.0 ** -24
    tol = off * (p.abs() + q.abs())
    got = ops.rotary(x, pos, plan).double()
    assert ((got[..., :8] - (p * c - q * s)).abs() <= tol).all()
    assert ((got[..., 8:] - (q * c + p * s)).abs() <= tol).all()
