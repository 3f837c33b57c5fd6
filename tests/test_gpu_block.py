"""A decoder block's memory-bound operators against their formulas in 64 bits: rows in 8 bits, the norms
and SwiGLU that read them, the join of a block with the norms around it, rotary positions, each with
its backward, and a block of all of them together. Each tolerance counts the roundings of the path, with
U32 = 2^-24 half a step of fp32 and U16 = 2^-8 half a step of bf16 (both relative)."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
U32, U16 = 2.0 ** -24, 2.0 ** -8
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}  # half a step, relative
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -149}  # and below the normal range
MOST = {"e4m3": 448.0, "int8": 127.0}
CODES = ["e4m3", "int8"]
# A row's sums: 16 terms a thread, 6 steps over a wave, 8 waves, then a few operations.
SUMS = 64


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _ops():
    from deltaserve_amd import ops

    return ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *s, dtype=F32):
    return torch.randn(*s, generator=g, device=DEV).to(dtype)


def _within(got, want, tol):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    assert not bad.any(), (int(bad.sum()), float(d[bad].max()), float((d / tol)[bad].max()))


def _strided(t, extra=8):
    """The same rows, `extra` elements further apart, with other values between them."""
    buf = torch.full((t.shape[0], t.shape[1] + extra), 9.0, device=DEV).to(t.dtype)
    buf[:, :t.shape[1]] = t
    return buf[:, :t.shape[1]]


# ---------------------------------------------------------------- rows in 8 bits

def _quantized(x, code):
    """(codes as 64-bit values, scale bytes) of the definition, for 64-bit x; NaN blocks byte 255,
    codes 0."""
    n, w = x.shape
    pad = torch.nn.functional.pad(x, (0, -w % 32)).view(n, -1, 32)
    top = pad.abs().amax(2)
    lost = ~torch.isfinite(pad).all(2)
    top = torch.where(lost, 1.0, top)
    # the least e: from log2, and one down or up where its rounding missed
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -300) / MOST[code])).clamp(min=-126)
    e = torch.where((e > -126) & (top <= MOST[code] * torch.exp2(e - 1)), e - 1, e)
    e = torch.where(top > MOST[code] * torch.exp2(e), e + 1, e)
    v = torch.where(lost[:, :, None], 0.0, pad) * torch.exp2(-e)[:, :, None]
    step = 1.0
    if code == "e4m3":
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    q = (v / step).round() * step
    bytes_ = torch.where(lost, 255.0, e + 127).to(torch.uint8)
    return q.view(n, -1)[:, :w], bytes_


def _values(q):
    """8-bit rows' values in 64 bits."""
    codes = q.codes.double()
    e = q.scales.double().repeat_interleave(32, 1)[:, :codes.shape[1]]
    return torch.where(e == 255, math.nan, codes * torch.exp2(e - 127))


def _eq(got, want):
    return bool(((got == want) | (got.isnan() & want.isnan())).all())


def _rough(g, n, w, dtype):
    """Rows of many sizes, with blocks of zeros, of tiny values and at the codes' borders."""
    x = _rand(g, n, w) * torch.exp2(torch.randint(-12, 12, (n, 1), generator=g, device=DEV).float())
    x[:, ::17] *= 30
    if n > 3 and w > 40:
        x[1, :33] = 0
        x[2, 32:41] = 448.0
        x[2, 40] = -449.0 if dtype != BF16 else -450.0
        x[3, 32:41] = 127.0
        x[3, 40] = 127.5
        x[0, :32] *= 2.0 ** (-20 if dtype == F16 else -128)
    return x.to(dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,w", [(1, 1), (3, 7), (5, 31), (4, 32), (7, 33), (5, 40), (6, 1000), (9, 4096),
                                 (4, 5001), (5, 2056), (33, 28672)])
def test_rows8_codes_are_the_definitions(n, w, dtype, code):
    ops = _ops()
    g = _gen(n * w)
    x, r = _rough(g, n, w, dtype), _rough(g, n, w, dtype)
    for a, b in ((x, None), (x, r), (_strided(x), None), (_strided(x, 3), _strided(r, 5))):
        got = ops.pack_rows8(a, b, code=code)
        want, scales = _quantized((a if b is None else a + b).double(), code)
        assert torch.equal(got.scales, scales)
        assert torch.equal(got.codes.double(), want)
        assert got.codes.stride(0) % 16 == 0 or n == 1
        assert _eq(ops.unpack_rows8(got, F32).double(), _values(got).float().double())
        assert _eq(ops.unpack_rows8(got).double(), _values(got).to(BF16).double())


@pytest.mark.parametrize("code", CODES)
def test_rows8_values_are_exact_in_bf16(code):
    """Every code times every normal scale that a saved block takes is a bf16 value."""
    ops = _ops()
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(249, 1)
    scales = torch.arange(1, 250, dtype=torch.uint8, device=DEV)[:, None].repeat(1, 8)
    q = ops.Rows8(codes.view(torch.float8_e4m3fn if code == "e4m3" else torch.int8), scales)
    want = _values(q)
    normal = (want.abs() >= 2.0 ** -126) & want.isfinite() & (want.abs() < 2.0 ** 127)
    assert torch.equal(ops.unpack_rows8(q).double()[normal], want[normal])
    assert torch.equal(ops.unpack_rows8(q, F32).double()[normal], want[normal])
    assert _eq(ops.unpack_rows8(q, F32).double(), want.float().double())


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("w", [96, 75])
def test_rows8_blocks_without_a_finite_maximum_are_nan(code, w):
    ops = _ops()
    x = _rand(_gen(1), 4, w)
    x[0, 3], x[1, 40], x[2, w - 1] = math.inf, math.nan, -math.inf
    q = ops.pack_rows8(x, code=code)
    lost = torch.zeros(4, w, dtype=torch.bool, device=DEV)
    lost[0, :32] = lost[1, 32:64] = lost[2, 64:] = True
    for dt in (BF16, F32):
        v = ops.unpack_rows8(q, dt)
        assert v[lost].isnan().all() and v[~lost].isfinite().all()
    want, scales = _quantized(x.double(), code)
    assert torch.equal(q.scales, scales) and torch.equal(q.codes.double(), want)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("w", [64, 100, 5120])
def test_save_rows_into_8_bits(w, code):
    """The save op's contract: the rows that the index pair names, no others; slots at the scratch row
    or outside are skipped."""
    from deltaserve_amd import capture

    ops = _ops()
    g = _gen(w)
    x, r = _rand(g, 40, w, dtype=BF16), _rand(g, 40, w, dtype=BF16)
    buf = ops.pack_rows8(_rand(g, 17, w), code=code)
    before = buf.codes.double().clone(), buf.scales.clone()
    src = torch.tensor([5, 39, 0, 7, 40, -1, 3, 9, 11], device=DEV)
    dst = torch.tensor([0, 15, 3, 16, 4, 5, 17, -2, 8], device=DEV)
    capture.save_rows(x, r, buf, src, dst)
    wrote = {0: 5, 15: 39, 3: 0, 8: 11}
    for row in range(17):
        if row in wrote:
            c, s = _quantized((x + r)[wrote[row]:wrote[row] + 1].double(), code)
            assert torch.equal(buf.codes[row].double(), c[0]) and torch.equal(buf.scales[row], s[0]), row
        else:
            assert torch.equal(buf.codes[row].double(), before[0][row]), row
            assert torch.equal(buf.scales[row], before[1][row]), row
    empty = torch.empty(0, dtype=torch.int64, device=DEV)
    capture.save_rows(x, None, buf, empty, empty)


def test_rows8_views_and_zeros():
    ops = _ops()
    q = ops.Rows8.zeros(6, 72, "int8")
    assert (ops.unpack_rows8(q) == 0).all() and q.codes.stride(0) == 80
    x = _rand(_gen(3), 2, 72)
    ops.pack_rows8(x, out=q[2:4])
    v = ops.unpack_rows8(q)
    assert (v[:2] == 0).all() and (v[4:] == 0).all()
    assert torch.equal(v[2:4].double(), _values(ops.pack_rows8(x, code="int8")))
    q.zero_()
    assert (ops.unpack_rows8(q) == 0).all()
    assert ops.unpack_rows8(q[:0]).shape == (0, 72)
    assert len(ops.pack_rows8(x[:0])) == 0
    assert ops.unpack_rows8(ops.pack_rows8(x[:, :0])).shape == (2, 0)


# ---------------------------------------------------------------- norms of 8-bit rows

def _norm(x, w, eps):
    """(normed, 1 / rms, x / rms) in 64 bits."""
    inv = (x.square().mean(1, keepdim=True) + eps).rsqrt()
    return x * inv * w, inv, x * inv


def _norm_back(x, gw, eps):
    """(gradient, its tolerance before the output's rounding) for the gradient gw of x / rms(x)."""
    inv = (x.square().mean(1, keepdim=True) + eps).rsqrt()
    hat = x * inv
    k = (gw * hat).mean(1, keepdim=True)
    size = (gw.abs() + hat.abs() * ((gw * hat).abs().mean(1, keepdim=True) + k.abs())) * inv
    return (gw - hat * k) * inv, SUMS * U32 * size


WIDTHS = [8, 24, 64, 520, 1024, 2048, 4096, 5120, 8192]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("n,D", [(1 + 3 * i, d) for i, d in enumerate(WIDTHS)] + [(5001, 136)])
def test_rmsnorm_of_8_bit_rows(n, D, code):
    ops = _ops()
    g = _gen(n + D)
    q = ops.pack_rows8(_rough(g, n, D, F32), code=code)
    w = (1 + 0.3 * _rand(g, D)).to(BF16)
    for eps in (1e-6, 1e-2):
        want, _, _ = _norm(_values(q), w.double(), eps)
        _within(ops.rmsnorm(q, w, eps), want, (U16 + SUMS * U32) * want.abs() + TINY[BF16])


@pytest.mark.parametrize("gdt", [BF16, F32])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("n,D", [(1 + 3 * i, d) for i, d in enumerate(WIDTHS)] + [(5001, 136)])
def test_rmsnorm_backward_of_8_bit_rows(n, D, code, gdt):
    ops = _ops()
    g = _gen(n + 2 * D)
    q = ops.pack_rows8(_rough(g, n, D, F32), code=code)
    w = (1 + 0.3 * _rand(g, D)).to(BF16)
    gr, resid = _rand(g, n, D, dtype=gdt), _rand(g, n, D, dtype=BF16)
    for r in (None, _strided(resid, 16)):
        got = ops.rmsnorm_backward(q, _strided(gr), w, 1e-5, resid=r)
        want, tol = _norm_back(_values(q), gr.double() * w.double(), 1e-5)
        if r is not None:
            want = want + r.double()
            tol = tol + 2 * U32 * r.double().abs()
        _within(got, want, tol + U16 * want.abs() + TINY[BF16])


def test_a_lost_row_stays_alone():
    """A NaN block reaches its own row of the norm and its gradient, no other."""
    ops = _ops()
    x = _rand(_gen(5), 3, 512)
    x[1, 7] = math.inf
    q = ops.pack_rows8(x)
    w = torch.ones(512, dtype=BF16, device=DEV)
    y = ops.rmsnorm(q, w, 1e-5)
    dx = ops.rmsnorm_backward(q, x.nan_to_num(posinf=1.0), w, 1e-5)
    assert y[1].isnan().all() and dx[1].isnan().all()
    assert y[[0, 2]].isfinite().all() and dx[[0, 2]].isfinite().all()


# ---------------------------------------------------------------- SwiGLU

# σ: the hardware's exponential and reciprocal, 2 units in the last place each (4·U32), of an argument
# that is rounded once (|g|·U32, and it counts with at most |g|·(1 − σ)); a product rounds once. The
# reciprocal has no subnormal results: where σ < 2^-126 it is 0, off by less than 2^-126 itself.
LEAST = 2.0 ** -126


def _glu(gu, dh=None):
    """(h, dgu, tolerances of both before their rounding) in 64 bits."""
    a, u = gu.chunk(2, 1)
    s = torch.sigmoid(a)
    off = (16 + 4 * a.abs()) * U32  # relative, of σ and of 1 − σ
    h = a * s * u
    if dh is None:
        return h, h.abs() * off + (a * u).abs() * LEAST
    dg = dh * u * s * (1 + a * (1 - s))
    du = dh * a * s
    # the bracket: 1, and a·(1 − σ) with 1 − σ off by σ's own rounding
    dtol = (dh * u).abs() * s * ((1 + a.abs() * (1 - s)) * off + a.abs() * 8 * U32)
    dtol = dtol + (dh * u).abs() * (1 + a.abs()) * LEAST
    return (h, h.abs() * off + (a * u).abs() * LEAST, torch.cat([dg, du], 1),
            torch.cat([dtol, du.abs() * off + (dh * a).abs() * LEAST], 1))


def _gate_up(g, n, I):
    x = 3 * _rand(g, n, 2 * I)
    x[:, ::7] *= 10
    return x


@pytest.mark.parametrize("kind", ["bf16"] + CODES)
@pytest.mark.parametrize("n,I", [(1, 8), (3, 24), (2, 40), (5, 1000), (7, 2048), (4, 4104), (3, 14336),
                                 (3000, 16)])
def test_swiglu_and_its_backward(n, I, kind):
    ops = _ops()
    g = _gen(n + I)
    x = _gate_up(g, n, I)
    gu = _strided(x.to(BF16)) if kind == "bf16" else ops.pack_rows8(x, code=kind)
    x = gu.double() if kind == "bf16" else _values(gu)
    want, tol = _glu(x)
    _within(ops.swiglu(gu), want, tol + U16 * want.abs() + TINY[BF16])
    for dt in (BF16, F32):
        dh = _strided(_rand(g, n, I, dtype=dt))
        want, tol, dwant, dtol = _glu(x, dh.double())
        got, h = ops.swiglu_backward(gu, dh, with_h=True)
        _within(h, want, tol + U16 * want.abs() + TINY[BF16])
        _within(got, dwant, dtol + U16 * dwant.abs() + TINY[BF16])
        assert torch.equal(h, ops.swiglu(gu))
        assert torch.equal(got, ops.swiglu_backward(gu, dh))


def test_swiglu_at_the_ends():
    """Gates far out give σ = 0 and 1, not NaN."""
    ops = _ops()
    a = torch.tensor([[-1e4, -200.0, -90.0, 0.0, 90.0, 200.0, 1e4, 1.0]], device=DEV)
    gu = torch.cat([a, torch.full_like(a, 2.0)], 1).to(BF16)
    dgu, h = ops.swiglu_backward(gu, torch.ones_like(a).to(BF16), with_h=True)
    want, tol, dwant, dtol = _glu(gu.double(), torch.ones_like(a).double())
    _within(h, want, tol + U16 * want.abs() + 2.0 ** -120)
    _within(dgu, dwant, dtol + U16 * dwant.abs() + 2.0 ** -120)


# ---------------------------------------------------------------- the join

def _join_case(seed, n, D, stream=BF16, post=True, gate="channel", spread=8):
    g = _gen(seed)
    c = dict(x=_strided(_rough(g, n, D, F32).clamp(-500, 500).to(stream), spread),
             y=_strided(_rand(g, n, D, dtype=BF16), spread), w_in=(1 + 0.3 * _rand(g, D)).to(BF16),
             w_out=(0.5 + 0.2 * _rand(g, D)).to(BF16) if post else None, scale=0.5, eps=1e-5)
    shape = {"none": None, "channel": (D,), "row": (n,), "column": (n, 1), "full": (n, D)}[gate]
    c["gate"] = None if shape is None else torch.rand(*shape, generator=g, device=DEV).to(BF16)
    if gate == "full":
        c["gate"] = _strided(c["gate"])
    return c


def _gate64(c, n, D):
    if c["gate"] is None:
        return 1.0
    g = c["gate"].double()
    return g[:, None] if g.dim() == 1 and not (len(g) == D) else g


GATES = ["none", "channel", "row", "column", "full"]


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("n,D", [(1, 8), (5, 24), (3, 520), (7, 1024), (2, 2048), (9, 4096), (3, 5120),
                                 (2, 8192), (2500, 64)])
def test_residual_norm(n, D, post, gate, stream):
    ops = _ops()
    c = _join_case(n + D, n, D, stream, post, gate)
    x, normed = ops.residual_norm(c["x"], c["y"], c["w_in"], c["eps"], w_out=c["w_out"], gate=c["gate"],
                                  scale=c["scale"])
    z = c["y"].double()
    if post:
        z = _norm(z, c["w_out"].double(), c["eps"])[0]
    z = c["scale"] * _gate64(c, n, D) * z
    want = c["x"].double() + z
    # z: its norm's sums and five products
    _within(x, want, HALF[stream] * want.abs() + SUMS * U32 * z.abs() + U32 * want.abs() + TINY[stream])
    assert x.dtype == stream and normed.dtype == BF16
    want, _, _ = _norm(x.double(), c["w_in"].double(), c["eps"])
    _within(normed, want, (U16 + SUMS * U32) * want.abs() + TINY[BF16])
    again, none = ops.residual_norm(c["x"], c["y"], None, c["eps"], w_out=c["w_out"], gate=c["gate"],
                                    scale=c["scale"])
    assert none is None and torch.equal(again, x)


def _join_back(c, x, y, dn, dxn):
    """{name: (gradient, tolerance before its rounding)} in 64 bits."""
    n, D = y.shape
    eps, a, gate = c["eps"], c["scale"], _gate64(c, n, D)
    w_in = None if c["w_in"] is None else c["w_in"].double()
    t, ttol = torch.zeros_like(y), torch.zeros_like(y)
    out = {}
    rows = (96 + n / 256) * U32  # a sum over rows: by block, then over blocks
    if dn is not None:
        t, ttol = _norm_back(x, dn * w_in, eps)
        hat = _norm(x, w_in, eps)[2]
        out["dw_in"] = ((dn * hat).sum(0), (rows + SUMS * U32) * (dn * hat).abs().sum(0))
    if dxn is not None:
        t = t + dxn
        ttol = ttol + 2 * U32 * (t.abs() + dxn.abs())
    out["dx"] = (t, ttol)
    # Σ z·t comes of three sums over a row, of terms of these sizes times |z|
    terms = torch.zeros_like(y) if dxn is None else dxn.abs()
    if dn is not None:
        xh = _norm(x, w_in, eps)[2]
        k = (dn * w_in * xh).mean(1, keepdim=True)
        kk = (dn * w_in * xh).abs().mean(1, keepdim=True) + k.abs()
        terms = terms + _norm(x, w_in, eps)[1] * ((dn * w_in).abs() + kk * xh.abs())
    dz, dztol = a * gate * t, a * gate * ttol + 4 * U32 * (a * gate * t).abs()
    z, ztol = y, 0 * y
    if c["w_out"] is None:
        out["dy"] = (dz, dztol)
    else:
        w = c["w_out"].double()
        z, j, hat = _norm(y, w, eps)
        ztol = SUMS * U32 * z.abs()
        want, tol = _norm_back(y, dz * w, eps)
        # the mean of dz·w·ŷ: each sum is off by SUMS·U32 of its terms
        m = 2 * SUMS * U32 * (a * gate * w.abs() * hat.abs() * terms).mean(1, keepdim=True)
        out["dy"] = (want, tol + j * (dztol * w.abs() + hat.abs() * m))
        out["dw_out"] = ((dz * hat).sum(0), ((rows + SUMS * U32) * (dz * hat).abs() + dztol * hat.abs()).sum(0))
    if c["gate"] is not None:
        dg, tol = a * t * z, a * (ttol * z.abs() + t.abs() * ztol) + 4 * U32 * (a * t * z).abs()
        if torch.is_tensor(gate) and gate.dim() == 1:
            dg, tol = dg.sum(0), (tol + rows * dg.abs()).sum(0)
        elif gate.shape == (n, 1) and c["gate"].shape != (n, D):
            dg = dg.sum(1, keepdim=True)
            tol = (tol + 2 * SUMS * U32 * a * z.abs() * terms).sum(1, keepdim=True)
        out["dgate"] = (dg.reshape(c["gate"].shape), tol.reshape(c["gate"].shape))
    return out


def _run_back(c, x, y, dn, dxn, **kw):
    ops = _ops()
    got = ops.residual_norm_backward(x, y, dn, c["w_in"], c["eps"], dx_new=dxn, w_out=c["w_out"],
                                     gate=c["gate"], scale=c["scale"], **kw)
    return dict(zip(("dx", "dy", "dgate", "dw_out", "dw_in"), got))


def _check_back(c, x, y, dn, dxn, got):
    d = lambda t: None if t is None else _values(t) if hasattr(t, "codes") else t.double()  # noqa: E731
    want = _join_back(c, d(x), d(y), d(dn), d(dxn))
    assert {k for k, v in got.items() if v is not None} == set(want)
    for name, (w, tol) in want.items():
        v = got[name]
        assert v.shape == w.shape, name
        _within(v, w, tol + HALF[v.dtype] * w.abs() + TINY[v.dtype] + 1e-30)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("n,D", [(1, 8), (5, 24), (3, 520), (7, 1024), (2, 2048), (9, 4096), (3, 5120),
                                 (2, 8192), (2500, 64)])
def test_residual_norm_backward(n, D, post, gate):
    c = _join_case(3 * n + D, n, D, BF16, post, gate)
    g = _gen(D)
    x_new = _strided(_rough(g, n, D, F32).clamp(-500, 500).to(BF16))
    dn, dxn = _strided(_rand(g, n, D, dtype=BF16)), _strided(_rand(g, n, D))
    got = _run_back(c, x_new, c["y"], dn, dxn)
    assert got["dx"].dtype == F32 and got["dy"].dtype == BF16
    _check_back(c, x_new, c["y"], dn, dxn, got)


@pytest.mark.parametrize("xt", ["bf16", "fp32", "e4m3", "int8"])
@pytest.mark.parametrize("yt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("gdt", [BF16, F32])
@pytest.mark.parametrize("cdt", [BF16, F32, None])
def test_residual_norm_backward_types(xt, yt, gdt, cdt):
    ops = _ops()
    n, D = 37, 264
    c = _join_case(5, n, D, BF16, True, "full")
    g = _gen(6)

    def rows(kind, v):
        if kind in CODES:
            return ops.pack_rows8(v, code=kind)
        return v.to(BF16 if kind == "bf16" else F32)

    x, y = rows(xt, _rough(g, n, D, F32).clamp(-500, 500)), rows(yt, _rand(g, n, D))
    dn = _rand(g, n, D, dtype=gdt)
    dxn = None if cdt is None else _rand(g, n, D, dtype=cdt)
    got = _run_back(c, x, y, dn, dxn)
    assert got["dx"].dtype == (cdt or gdt)
    _check_back(c, x, y, dn, dxn, got)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("post", [False, True])
def test_residual_norm_backward_without_a_norm_after(post, gate):
    n, D = 19, 136
    c = _join_case(7, n, D, BF16, post, gate)
    c["w_in"] = None
    x = _rand(_gen(1), n, D, dtype=BF16)
    dxn = _rand(_gen(2), n, D)
    _check_back(c, x, c["y"], None, dxn, _run_back(c, x, c["y"], None, dxn))


@pytest.mark.parametrize("n,D", [(511, 64), (512, 64), (513, 64), (1, 4096), (1500, 1024)])
def test_residual_norm_backward_sums_over_rows(n, D):
    """Row counts around those that one block takes more of; twice the same; without the sums the rest is
    the same."""
    c = _join_case(n, n, D, BF16, True, "channel")
    g = _gen(n)
    x, dn, dxn = _rand(g, n, D, dtype=BF16), _rand(g, n, D), _rand(g, n, D)
    got = _run_back(c, x, c["y"], dn, dxn)
    _check_back(c, x, c["y"], dn, dxn, got)
    for k, v in _run_back(c, x, c["y"], dn, dxn).items():
        assert torch.equal(v, got[k]), k
    less = _run_back(c, x, c["y"], dn, dxn, weight_grads=False)
    assert less["dw_in"] is less["dw_out"] is less["dgate"] is None
    assert torch.equal(less["dx"], got["dx"]) and torch.equal(less["dy"], got["dy"])


def test_broadcast_operands_are_refused_or_read_as_they_are():
    """A gate of one value for all rows, broadcast, has no rows of its own; rotary reads broadcast heads."""
    ops = _ops()
    x, w = _rand(_gen(1), 5, 64, dtype=BF16), torch.ones(64, dtype=BF16, device=DEV)
    from deltaserve_amd._lib import DsbError

    for kw in (dict(gate=w[:1].view(1, 1).expand(5, 1)), dict(gate=w.expand(5, 64))):
        with pytest.raises(DsbError):
            ops.residual_norm(x, x, w, 1e-5, **kw)
        with pytest.raises(DsbError):
            ops.residual_norm_backward(x, x, x, w, 1e-5, **kw)
    for bad in (w.expand(5, 64), x[:, :64].as_strided((5, 64), (32, 1))):
        with pytest.raises(DsbError):
            ops.residual_norm(bad, x, w, 1e-5)
        with pytest.raises(DsbError):
            ops.pack_rows8(bad)
    two = _rand(_gen(2), 5, 2, dtype=BF16)  # a column of a matrix is a gate by row
    got = ops.residual_norm(x, x, w, 1e-5, gate=two[:, 1:])
    for a, b in zip(got, ops.residual_norm(x, x, w, 1e-5, gate=two[:, 1].contiguous())):
        assert torch.equal(a, b)
    plan, pos = ops.rotary_plan(64, 1e4), torch.arange(5, device=DEV)
    heads = x[:, None].expand(5, 3, 64)
    assert torch.equal(ops.rotary(heads, pos, plan), ops.rotary(heads.contiguous(), pos, plan))
    with pytest.raises(DsbError):
        ops.rotary(heads, pos, plan, out=heads)


def test_residual_norm_of_no_rows():
    ops = _ops()
    x = torch.empty(0, 64, dtype=BF16, device=DEV)
    w = torch.ones(64, dtype=BF16, device=DEV)
    for gate in (None, w, x):
        new, normed = ops.residual_norm(x, x, w, 1e-5, w_out=w, gate=gate)
        assert new.shape == normed.shape == (0, 64)
        dx, dy, dgate, dw_out, dw_in = ops.residual_norm_backward(x, x, x, w, 1e-5, w_out=w, gate=gate)
        assert dx.shape == dy.shape == (0, 64)
        assert (dw_out == 0).all() and (dw_in == 0).all() and dw_in.shape == (64,)
        if gate is w:
            assert (dgate == 0).all()
    q = ops.Rows8.zeros(0, 64)
    assert ops.rmsnorm(q, w, 1e-5).shape == ops.rmsnorm_backward(q, x, w, 1e-5).shape == (0, 64)
    assert ops.swiglu(q).shape == (0, 32) and ops.swiglu_backward(q, x[:, :32]).shape == (0, 64)


def test_rows_of_zeros_and_far_sizes():
    """A row of zeros has rms sqrt(eps); rows of 1e-18 and 1e15 keep their gradients finite and right."""
    n, D = 4, 256
    c = _join_case(9, n, D, F32, True, "row")
    g = _gen(9)
    x = _rand(g, n, D) * torch.tensor([[0.0], [1e-18], [1.0], [1e15]], device=DEV)
    y = (_rand(g, n, D) * torch.tensor([[1.0], [0.0], [1e-18], [1e15]], device=DEV)).to(BF16)
    dn, dxn = _rand(g, n, D), _rand(g, n, D)
    got = _run_back(c, x, y, dn, dxn)
    assert all(v.isfinite().all() for v in got.values())
    _check_back(c, x, y, dn, dxn, got)


def test_join_gradients_against_differences():
    """Along random directions of x, y and the parameters: Σ gradient·direction is the central difference
    of the 64-bit forward (which is off by h² of its third derivative, 1e-7 here)."""
    n, D = 6, 96
    for gate in GATES:
        c = _join_case(11, n, D, F32, True, gate)
        g = _gen(12)
        x, y = _rand(g, n, D), _rand(g, n, D, dtype=BF16)
        dn, dxn = _rand(g, n, D), _rand(g, n, D)
        # the stream before the join whose x_new is x
        base = {"x": x.double(), "y": y.double(), "w_in": c["w_in"].double(), "w_out": c["w_out"].double()}
        if c["gate"] is not None:
            base["gate"] = c["gate"].double()
        z0 = c["scale"] * _gate64(c, n, D) * _norm(base["y"], base["w_out"], 1e-5)[0]
        base["x"] = base["x"] - z0

        def loss(p):
            cc = dict(c, gate=p.get("gate"))
            z = c["scale"] * _gate64(cc, n, D) * _norm(p["y"], p["w_out"], 1e-5)[0]
            new = p["x"] + z
            return float((dn.double() * _norm(new, p["w_in"], 1e-5)[0]).sum() + (dxn.double() * new).sum())

        got = _run_back(c, x, y, dn, dxn)
        want = _join_back(c, x.double(), y.double(), dn.double(), dxn.double())
        for name, key in (("dx", "x"), ("dy", "y"), ("dw_in", "w_in"), ("dw_out", "w_out"), ("dgate", "gate")):
            if key not in base:
                continue
            v = torch.randn(base[key].shape, generator=g, device=DEV, dtype=F64)
            h = 1e-4
            up, down = dict(base), dict(base)
            up[key], down[key] = base[key] + h * v, base[key] - h * v
            diff = (loss(up) - loss(down)) / (2 * h)
            grad, tol = want[name]
            tol = (tol + HALF[got[name].dtype] * grad.abs()) * v.abs()
            assert abs(float((got[name].double() * v).sum()) - diff) <= float(tol.sum()) + 1e-5 * abs(diff) + 1e-5, (gate, name)


# ---------------------------------------------------------------- rotary positions

def _turned(x, pos, plan, back=False):
    """(result, tolerance before its rounding) in 64 bits. cos and sin: the angle's fp32 part is off by
    2^-24 turns at most (2^-21 radians with 2π), the functions by 2 units in the last place, the
    factor's product by half a one; two products and a sum."""
    r = plan.rotary_dim
    inv = torch.from_numpy(plan.inv_freq).to(DEV)
    ang = pos.double()[:, None, None] * inv
    c, s = plan.factor * ang.cos(), plan.factor * ang.sin() * (-1 if back else 1)
    y, tol = x.double(), torch.zeros(x.shape, dtype=F64, device=DEV)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if plan.interleaved else (slice(0, r // 2), slice(r // 2, r))
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = p * c - q * s, q * c + p * s
    tol[..., a] = tol[..., b] = 2.0 ** -20 * plan.factor * (p.abs() + q.abs())
    return y, tol


LLAMA = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
         "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,hd,rot", [(1, 1, 2, 2), (3, 2, 6, 4), (1, 40, 128, 128), (5, 3, 80, 32),
                                            (7, 5, 64, 50), (257, 9, 96, 96), (9, 12, 256, 64), (3, 1, 1024, 1024),
                                            (2, 7, 16, 16), (2, 70, 8, 8), (33, 33, 72, 48), (4100, 2, 64, 16)])
def test_rotary(n, heads, hd, rot, interleaved, dtype):
    ops = _ops()
    g = _gen(n + hd)
    plan = ops.rotary_plan(hd, 5e5, rotary_dim=rot, interleaved=interleaved)
    x = _rand(g, n, heads, hd, dtype=dtype)
    pos = torch.randint(0, 20000, (n,), generator=g, device=DEV)
    for p, back in ((pos, False), (pos.to(torch.int32), True)):
        got = (ops.rotary_backward if back else ops.rotary)(x, p, plan)
        want, tol = _turned(x, p, plan, back)
        _within(got, want, tol + HALF[dtype] * want.abs() + TINY[dtype])
        assert torch.equal(got[..., rot:], x[..., rot:])
        # rows that hold other things beside, each head as far apart as it may be, and in place
        wide = torch.full((n, heads + 1, hd + 8), 7.0, device=DEV).to(dtype)
        view = wide[:, :heads, :hd]
        view.copy_(x)
        same = (ops.rotary_backward if back else ops.rotary)(view, p, plan)
        assert torch.equal(same, got)
        assert (ops.rotary_backward if back else ops.rotary)(view, p, plan, out=view) is view
        assert torch.equal(view, got) and (wide[:, heads:] == 7).all() and (wide[..., hd:] == 7).all()


@pytest.mark.parametrize("hd,rot", [(128, 128), (64, 36)])
def test_rotary_views_that_start_anywhere(hd, rot):
    """Heads of rows whose addresses and strides allow no wide access, or other ones in and out."""
    ops = _ops()
    g = _gen(2)
    n, heads = 11, 3
    for interleaved in (False, True):
        plan = ops.rotary_plan(hd, 1e4, rotary_dim=rot, interleaved=interleaved)
        pos = torch.arange(n, device=DEV, dtype=torch.int32)
        flat = _rand(g, n * (heads * hd + 3) + 1, dtype=BF16)
        x = flat[1:].view(n, heads * hd + 3)[:, :heads * hd].unflatten(1, (heads, hd))
        want, tol = _turned(x, pos, plan)
        got = ops.rotary(x, pos, plan)
        _within(got, want, tol + U16 * want.abs())
        out = torch.zeros(heads, n, hd, dtype=BF16, device=DEV).transpose(0, 1)
        assert torch.equal(ops.rotary(x, pos, plan, out=out), got)


@pytest.mark.parametrize("scaling", [None, LLAMA, YARN, {"rope_type": "linear", "factor": 4.0}])
def test_rotary_far_positions(scaling):
    """Angles keep fp32's precision wherever the position is."""
    ops = _ops()
    plan = ops.rotary_plan(64, 1e6, scaling)
    pos = torch.tensor([0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 31 - 1], device=DEV)
    x = _rand(_gen(4), len(pos), 4, 64)
    want, tol = _turned(x, pos, plan)
    _within(ops.rotary(x, pos, plan), want, tol + U32 * want.abs())
    back, tol2 = _turned(want, pos, plan, True)
    got = ops.rotary_backward(ops.rotary(x, pos, plan), pos, plan)
    _within(got, back, tol2 + 2 * plan.factor * (tol + U32 * want.abs()).amax(-1, keepdim=True) + U32 * back.abs())
    _within(back.float(), plan.factor ** 2 * x.double(), 2 * U32 * plan.factor ** 2 * x.double().abs() + 1e-12)


def test_rotary_of_nothing():
    ops = _ops()
    plan = ops.rotary_plan(64, 1e4)
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    assert ops.rotary(torch.empty(0, 4, 64, dtype=BF16, device=DEV), e, plan).shape == (0, 4, 64)
    p = torch.arange(3, device=DEV)
    assert ops.rotary(torch.empty(3, 0, 64, dtype=BF16, device=DEV), p, plan).shape == (3, 0, 64)


# ---------------------------------------------------------------- streams and graphs

def _every_op(s):
    """One call of each op on the tensors of s; their results."""
    ops = _ops()
    q = ops.pack_rows8(s["x"], s["y"])
    gu = ops.pack_rows8(s["x"], code="int8")
    out = [q.codes.view(torch.uint8), q.scales, ops.unpack_rows8(q), ops.rmsnorm(q, s["w"], 1e-5),
           ops.rmsnorm_backward(q, s["dn"], s["w"], 1e-5, resid=s["y"]), ops.swiglu(gu),
           *ops.swiglu_backward(gu, s["dn"][:, :s["x"].shape[1] // 2], with_h=True)]
    out += ops.residual_norm(s["x"], s["y"], s["w"], 1e-5, w_out=s["w"], gate=s["gate"], scale=0.5)
    out += ops.residual_norm_backward(q, s["y"], s["dn"], s["w"], 1e-5, dx_new=s["dx"], w_out=s["w"],
                                      gate=s["gate"], scale=0.5)
    h = s["x"].unflatten(1, (-1, 64))
    out.append(ops.rotary_backward(ops.rotary(h, s["pos"], s["plan"]), s["pos"], s["plan"]))
    return out


def _state(seed, n=700, D=1024):
    g = _gen(seed)
    return dict(x=_rand(g, n, D, dtype=BF16), y=_rand(g, n, D, dtype=BF16), dn=_rand(g, n, D, dtype=BF16),
                dx=_rand(g, n, D), w=_rand(g, D, dtype=BF16), gate=_rand(g, D, dtype=BF16),
                pos=torch.arange(n, device=DEV) + seed, plan=_ops().rotary_plan(64, 1e4, interleaved=True))


def test_two_graphs_replayed_with_new_inputs():
    """All ops in one graph, and again in a second, replayed in turn with eager work between."""
    states = [_state(1), _state(2, 300, 512)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for s in states:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            outs.append(_every_op(s))
        graphs.append(graph)
    for rep in range(3):
        for s, graph, out in zip(states, graphs, outs):
            new = _state(10 + rep, *s["x"].shape)
            for k, v in new.items():
                if torch.is_tensor(v):
                    s[k].copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            for i, (got, want) in enumerate(zip(out, _every_op(s))):
                assert torch.equal(got, want), (rep, i)


def test_ops_run_on_the_current_stream():
    s = _state(3)
    want = _every_op(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = torch.randn(2048, 2048, device=DEV)
        for _ in range(20):  # work that the ops' inputs wait behind
            a = a @ a / 50
        late = {k: v.clone() if torch.is_tensor(v) else v for k, v in s.items()}
        got = _every_op(late)
    side.synchronize()
    for i, (g, w) in enumerate(zip(got, want)):
        assert torch.equal(g, w), i


# ---------------------------------------------------------------- a block

class _Exact:
    """The block's operators in 64 bits; rounding: to the kernels' types where they store."""

    def __init__(self, rounding):
        self.r = (lambda t, dt=BF16: t.to(dt).double()) if rounding else (lambda t, dt=BF16: t)

    def mm(self, a, b):
        return self.r(a @ b.t())

    def mm_back(self, g, b):
        return g @ b  # fp32 out

    def norm(self, x, w):
        return self.r(_norm(x, w, 1e-5)[0])

    def join(self, x, y, w_in, w_out, gate):
        new = self.r(x + 0.5 * gate * _norm(y, w_out, 1e-5)[0])
        return new, None if w_in is None else self.norm(new, w_in)

    def join_back(self, x, y, dn, dx, w_in, w_out, gate):
        c = dict(eps=1e-5, scale=0.5, gate=gate, w_in=w_in, w_out=w_out)
        out = {k: v[0] for k, v in _join_back(c, x, y, dn, dx).items()}
        return out["dx"], self.r(out["dy"]), out

    def norm_back(self, x, g, w, resid):
        return _norm_back(x, g * w, 1e-5)[0] + resid

    def swiglu(self, gu):
        return self.r(_glu(gu)[0])

    def swiglu_back(self, gu, dh):
        return self.r(_glu(gu, dh)[2])

    def turn(self, x, pos, plan, back=False):
        return self.r(_turned(x, pos, plan, back)[0])

    def _heads(self, qk, v, lens):
        for n0, n1 in zip([0, *torch.tensor(lens).cumsum(0).tolist()], torch.tensor(lens).cumsum(0).tolist()):
            q, k, w = (t[n0:n1].transpose(0, 1) for t in (qk[:, :4], qk[:, 4:], v))
            p = (q.unflatten(0, (2, 2)) @ k[:, None].transpose(-1, -2)) / math.sqrt(q.shape[-1])
            p = p.masked_fill(~torch.ones(n1 - n0, n1 - n0, dtype=torch.bool, device=DEV).tril(), -math.inf)
            yield n0, n1, q, k, w, p.softmax(-1)

    def attn(self, qk, v, lens):
        out = torch.zeros(qk.shape[0], 4, qk.shape[2], dtype=F64, device=DEV)
        for n0, n1, _, _, w, p in self._heads(qk, v, lens):
            out[n0:n1] = (p @ w[:, None]).flatten(0, 1).transpose(0, 1)
        return self.r(out.flatten(1))

    def attn_back(self, qk, v, dout, lens):
        dqk, dv = torch.zeros_like(qk), torch.zeros_like(v)
        for n0, n1, q, k, w, p in self._heads(qk, v, lens):
            d = dout[n0:n1].unflatten(1, (4, -1)).transpose(0, 1).unflatten(0, (2, 2))
            dp = d @ w[:, None].transpose(-1, -2)
            ds = p * (dp - (dp * p).sum(-1, keepdim=True)) / math.sqrt(q.shape[-1])
            dqk[n0:n1, :4] = (ds @ k[:, None]).flatten(0, 1).transpose(0, 1)
            dqk[n0:n1, 4:] = (ds.transpose(-1, -2) @ q.unflatten(0, (2, 2))).sum(1).transpose(0, 1)
            dv[n0:n1] = (p.transpose(-1, -2) @ d).sum(1).transpose(0, 1)
        return self.r(dqk), self.r(dv)


class _Kernels:
    def __init__(self):
        self.ops = _ops()

    def mm(self, a, b):
        return self.ops.gemm_nt(a, b)

    def mm_back(self, g, b):
        return self.ops.gemm_nt(g, b, out_dtype=F32, b_kn=True)

    def norm(self, x, w):
        return self.ops.rmsnorm(x, w, 1e-5)

    def join(self, x, y, w_in, w_out, gate):
        return self.ops.residual_norm(x, y, w_in, 1e-5, w_out=w_out, gate=gate, scale=0.5)

    def join_back(self, x, y, dn, dx, w_in, w_out, gate):
        dx, dy, dgate, dw_out, dw_in = self.ops.residual_norm_backward(
            x, y, dn, w_in, 1e-5, dx_new=dx, w_out=w_out, gate=gate, scale=0.5)
        return dx, dy, dict(dgate=dgate, dw_out=dw_out, dw_in=dw_in)

    def norm_back(self, x, g, w, resid):
        # (a join's backward without a block would do; the framework's norm op takes a bf16 residual)
        return self.ops.rmsnorm_backward(x, g, w, 1e-5, resid=resid.to(BF16))

    def swiglu(self, gu):
        return self.ops.swiglu(gu)

    def swiglu_back(self, gu, dh):
        return self.ops.swiglu_backward(gu, dh)

    def turn(self, x, pos, plan, back=False):
        return (self.ops.rotary_backward if back else self.ops.rotary)(x, pos, plan)

    def attn(self, qk, v, lens):
        self.saved = self.ops.attn_forward(qk[:, :4].flatten(1), qk[:, 4:].flatten(1), v.flatten(1), lens, 4, 2, 64)
        return self.saved[0]

    def attn_back(self, qk, v, dout, lens):
        _, o32, lse = self.ops.attn_forward(qk[:, :4].flatten(1), qk[:, 4:].flatten(1), v.flatten(1), lens, 4, 2, 64)
        dq, dk, dv = self.ops.attn_backward(qk[:, :4].flatten(1), qk[:, 4:].flatten(1), v.flatten(1), o32,
                                            lse, dout, lens, 4, 2, 64)
        return torch.cat([dq, dk], 1).unflatten(1, (6, 64)), dv.unflatten(1, (2, 64))


def _block(k, m, x, dout, pos, plan, lens, keep):
    """A block forward and backward: norm, attention, join, MLP, join. ``keep`` is what happens to an
    activation between the two (name, rows)."""
    normed = k.norm(x, m["w1"])
    qkv = k.mm(normed, m["qkv"]).unflatten(1, (8, 64))
    qk, v = k.turn(qkv[:, :6], pos, plan), qkv[:, 6:].contiguous()
    ctx = k.attn(qk, v, lens)
    y1 = k.mm(ctx, m["o"])
    x1, n1 = k.join(x, y1, m["w2"], m["p1"], m["g1"])
    gu = k.mm(n1, m["gu"])
    y2 = k.mm(k.swiglu(gu), m["down"])
    x2, _ = k.join(x1, y2, None, m["p2"], m["g2"])
    x_, y1, x1, gu, y2 = (keep(name, t) for name, t in (("x", x), ("y1", y1), ("x1", x1), ("gu", gu), ("y2", y2)))
    # backward
    dx, dy, g2 = k.join_back(x1, y2, None, dout, None, m["p2"], m["g2"])
    dgu = k.swiglu_back(gu, k.mm_back(dy, m["down"]))
    dx, dy, g1 = k.join_back(x1, y1, k.mm_back(dgu, m["gu"]), dx, m["w2"], m["p1"], m["g1"])
    dctx = k.mm_back(dy, m["o"])
    dctx = dctx.to(BF16) if dctx.dtype == F32 else k.r(dctx)
    dqk, dv = k.attn_back(qk, v, dctx, lens)
    dqkv = torch.cat([k.turn(dqk, pos, plan, True).flatten(1), dv.flatten(1)], 1)
    dx = k.norm_back(x_, k.mm_back(dqkv, m["qkv"]), m["w1"], dx)
    return dict(x2=x2, dx=dx, **{"a_" + n: t for n, t in g1.items() if n in ("dgate", "dw_out", "dw_in")},
                **{"b_" + n: t for n, t in g2.items() if n in ("dgate", "dw_out")})


@pytest.mark.parametrize("code", [None, "e4m3", "int8"])
@pytest.mark.parametrize("interleaved,rot", [(False, 64), (True, 32)])
def test_a_block_forward_and_backward(code, interleaved, rot):
    """Every result of a block's kernels is at most twice as far from the block in 64 bits (in
    norm) as 64-bit arithmetic is that rounds where the kernels store; its activations are kept in 8
    bits between forward and backward, the same ones on all sides."""
    ops = _ops()
    lens, D = [70, 1, 129], 256
    n = sum(lens)
    g = _gen(21)
    w = lambda *s: (_rand(g, *s) / math.sqrt(s[-1])).to(BF16)  # noqa: E731
    v = lambda: (1 + 0.2 * _rand(g, D)).to(BF16)  # noqa: E731
    m = dict(qkv=w(512, D), o=w(D, D), gu=w(1024, D), down=w(D, 512), w1=v(), w2=v(), p1=v(), p2=v(),
             g1=v(), g2=v())
    x, dout = _rand(g, n, D, dtype=BF16), _rand(g, n, D)
    pos = torch.cat([torch.arange(k, device=DEV) for k in lens]).to(torch.int32) + 1000
    plan = ops.rotary_plan(64, 1e4, rotary_dim=rot, interleaved=interleaved)
    kept = {}

    def keep(name, t):
        kept[name] = t if code is None else ops.pack_rows8(t, code=code)
        return kept[name]

    got = _block(_Kernels(), m, x, dout, pos, plan, lens, keep)
    again = lambda name, t: kept[name].double() if code is None else _values(kept[name])  # noqa: E731
    m64 = {k: t.double() for k, t in m.items()}
    exact, rounded = (_block(_Exact(r), m64, x.double(), dout.double(), pos, plan, lens, again)
                      for r in (False, True))
    assert set(got) == set(exact)
    for name, want in exact.items():
        own = float((got[name].double() - want).norm() / want.norm())
        far = float((rounded[name] - want).norm() / want.norm())
        out = HALF[got[name].dtype]
        # and fp32's own roundings of sums over rows: (96 + SUMS)·U32 of the terms' sizes, which for
        # terms of random signs come to sqrt(n) times their sum
        sums = (96 + SUMS) * U32 * math.sqrt(n)
        assert own <= 2 * far + 2 * out + sums, (name, own, far)
