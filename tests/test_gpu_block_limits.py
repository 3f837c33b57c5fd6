"""A decoder block's memory-bound operators at the ends of their ranges: 8-bit rows next to the largest finite
value, rotary angles of far positions against exact arithmetic."""

from __future__ import annotations

import math

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
