"""A decoder block's memory-bound operators in large calls, whose loads and stores take other ways through the
caches than small ones' and whose offsets pass 32 bits. A row's results do not depend on the rows beside
it, so a large call equals, bit for bit, the same call on parts of its rows."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _ops():
    from deltaserve_amd import ops

    return ops


def _rand(seed, *s, dtype=BF16):
    return torch.randn(*s, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV, dtype=dtype)


def _bits(t):
    return [t.codes.view(torch.uint8), t.scales] if hasattr(t, "codes") else [t]


def _equal_parts(call, n, rows=1000, at=None):
    """call(slice) over all n rows against its parts of `rows` (those that start at `at`, or all)."""
    whole = call(slice(0, n))
    for lo in range(0, n, rows) if at is None else at:
        part = slice(lo, min(lo + rows, n))
        for i, (a, b) in enumerate(zip(whole, call(part))):
            if a is None:
                assert b is None
                continue
            for x, y in zip(_bits(a[part]), _bits(b)):
                assert torch.equal(x, y), (i, lo)


# inputs of up to 85 MB are small calls
@pytest.mark.parametrize("n", [3000, 12000, 25000])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_rows8(n, code):
    ops = _ops()
    x, r, h = _rand(1, n, 4096), _rand(2, n, 4096), _rand(3, n, 4100, dtype=F16)
    f = _rand(4, n // 2, 4096, dtype=F32)
    _equal_parts(lambda s: (ops.pack_rows8(x[s], code=code), ops.pack_rows8(x[s], r[s], code=code),
                            ops.pack_rows8(h[s], code=code)), n)
    _equal_parts(lambda s: (ops.pack_rows8(f[s], code=code),), n // 2)
    q = ops.pack_rows8(x, code=code)
    u = ops.pack_rows8(h, code=code)
    _equal_parts(lambda s: (ops.unpack_rows8(q[s]), ops.unpack_rows8(q[s], F32), ops.unpack_rows8(u[s])), n)


@pytest.mark.parametrize("n", [3000, 12000, 25000])
@pytest.mark.parametrize("code", [None, "e4m3", "int8"])
def test_norm_and_swiglu(n, code):
    ops = _ops()
    x, g, w = _rand(1, n, 4096), _rand(2, n, 4096, dtype=F32), _rand(3, 4096)
    q = x if code is None else ops.pack_rows8(x, code=code)
    if code is not None:
        _equal_parts(lambda s: (ops.rmsnorm(q[s], w, 1e-5), ops.rmsnorm_backward(q[s], g[s], w, 1e-5, resid=x[s]),
                                ops.rmsnorm_backward(q[s], x[s], w, 1e-5)), n)
    _equal_parts(lambda s: (ops.swiglu(q[s]), *ops.swiglu_backward(q[s], g[s, :2048], with_h=True),
                            ops.swiglu_backward(q[s], x[s, :2048])), n)


@pytest.mark.parametrize("n", [1500, 6000])
@pytest.mark.parametrize("gate", [None, "channel", "row", "full"])
@pytest.mark.parametrize("stream", [BF16, F32, "e4m3"])
def test_join(n, gate, stream):
    ops = _ops()
    D = 5120
    y, w, w2 = _rand(2, n, D), _rand(3, D), _rand(4, D)
    gates = {None: None, "channel": _rand(5, D), "row": _rand(5, n), "full": _rand(5, n, D)}[gate]
    part = (lambda s: gates[s]) if gate in ("row", "full") else (lambda s: gates)
    x = _rand(1, n, D, dtype=BF16 if stream == "e4m3" else stream)
    _equal_parts(lambda s: ops.residual_norm(x[s], y[s], w, 1e-5, w_out=w2, gate=part(s), scale=0.5), n)
    dn, dx = _rand(6, n, D), _rand(7, n, D, dtype=F32)
    kept, kept_y = (ops.pack_rows8(x), ops.pack_rows8(y)) if stream == "e4m3" else (x, y)
    for d in (dx, dx.to(BF16)):  # (the sums over rows are of all of them)
        _equal_parts(lambda s: ops.residual_norm_backward(
            kept[s], kept_y[s], dn[s], w, 1e-5, dx_new=d[s], w_out=w2, gate=part(s), scale=0.5,
            weight_grads=False)[:2 if gate == "channel" else 3], n)


@pytest.mark.parametrize("n", [3000, 10000, 18000])
@pytest.mark.parametrize("interleaved,rot", [(False, 128), (True, 64), (False, 62), (True, 30)])
def test_rotary(n, interleaved, rot):
    ops = _ops()
    plan = ops.rotary_plan(128, 1e6, rotary_dim=rot, interleaved=interleaved)
    pos = torch.arange(n, device=DEV)
    qkv, f = _rand(1, n, 48, 128), _rand(2, n, 20, 128, dtype=F32)
    _equal_parts(lambda s: (ops.rotary(qkv[s, :40], pos[s], plan), ops.rotary_backward(f[s], pos[s], plan)), n)
    want = ops.rotary(qkv[:, :40], pos, plan)
    kept = qkv[:, 40:].clone()
    ops.rotary(qkv[:, :40], pos, plan, out=qkv[:, :40])
    assert torch.equal(qkv[:, :40], want) and torch.equal(qkv[:, 40:], kept)


def test_offsets_past_32_bits():
    """More than 2^31 elements, 2^32 bytes: rows at the start, about the borders and at the end."""
    ops = _ops()
    n, D = 290000, 8192  # 2.4e9 elements
    at = [0, (1 << 31) // D // 2 - 8, (1 << 31) // D - 8, n - 16]
    x, w, pos = _rand(1, n, D), _rand(3, D), torch.arange(n, device=DEV)
    plan = ops.rotary_plan(128, 1e6)
    kw = dict(rows=16, at=at)
    _equal_parts(lambda s: (ops.pack_rows8(x[s]),), n, **kw)
    q = ops.pack_rows8(x)
    _equal_parts(lambda s: (ops.unpack_rows8(q[s], F32),), n, **kw)
    _equal_parts(lambda s: (ops.rmsnorm(q[s], w, 1e-5),), n, **kw)
    _equal_parts(lambda s: (ops.swiglu_backward(q[s], x[s, :D // 2]),), n, **kw)
    _equal_parts(lambda s: ops.residual_norm(x[s], x[s], w, 1e-5, w_out=w, gate=x[s]), n, **kw)
    _equal_parts(lambda s: ops.residual_norm_backward(q[s], x[s], x[s], w, 1e-5, w_out=w, gate=x[s],
                                                      weight_grads=False), n, **kw)
    _equal_parts(lambda s: (ops.rotary(x[s].view(-1, 64, 128), pos[s], plan),), n, **kw)
    src = torch.tensor([n - 1, 3], device=DEV)  # from and to rows past 2^32 bytes
    ops.pack_rows8(x, out=q, src=src, dst=torch.tensor([n - 2, 0], device=DEV))
    for to, of in ((n - 2, n - 1), (0, 3)):
        for a, b in zip(_bits(q[to:to + 1]), _bits(ops.pack_rows8(x[of:of + 1]))):
            assert torch.equal(a, b)
