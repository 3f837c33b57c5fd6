"""A decoder block's memory-bound operators without a GPU: the frequencies of rotary plans and the
refusals, which come before any device call."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


def _lib():
    from deltaserve_amd import _lib as L

    return L, L.load()


def _refused(name, args, part):
    L, lib = _lib()
    assert getattr(lib, name)(*args) == -1
    assert part in L.last_error(), L.last_error()


A = 1 << 20  # an address, aligned; the calls below are refused before they use it


# ---------------------------------------------------------------- 8-bit rows

def test_rows8_of_other_tensors_are_refused():
    from deltaserve_amd.rows8 import Rows8

    codes, scales = torch.zeros(3, 40, dtype=torch.int8), torch.ones(3, 2, dtype=torch.uint8)
    q = Rows8(codes, scales)
    assert q.code == "int8" and q.shape == (3, 40) and len(q[1:]) == 2 and q.nbytes == 126
    assert Rows8.zeros(2, 33, "e4m3", "cpu").codes.stride(0) == 48
    for c, s in ((codes.to(torch.uint8), scales), (codes[0], scales), (codes, scales[:, :1]),
                 (codes, scales.to(torch.int8)), (codes, scales[:2]), (codes.t().contiguous().t(), scales)):
        with pytest.raises(ValueError):
            Rows8(c, s)
    with pytest.raises(ValueError):
        Rows8.zeros(1, 1, "int4", "cpu")
    with pytest.raises(TypeError):
        q[0]


def test_cpu_tensors_are_refused():
    from deltaserve_amd import capture, ops
    from deltaserve_amd.rows8 import Rows8

    x = torch.zeros(2, 64, dtype=BF16)
    w = torch.ones(64, dtype=BF16)
    q = Rows8.zeros(2, 64, device="cpu")
    i = torch.zeros(1, dtype=torch.int64)
    plan = ops.RotaryPlan(32, 32, False, np.ones(16), 1.0, "cpu")
    for call in (lambda: ops.pack_rows8(x), lambda: ops.unpack_rows8(q), lambda: ops.rmsnorm(q, w, 1e-5),
                 lambda: ops.rmsnorm_backward(q, x, w, 1e-5), lambda: ops.swiglu(q), lambda: ops.swiglu(x),
                 lambda: ops.swiglu_backward(x, x[:, :32].contiguous()),
                 lambda: ops.residual_norm(x, x, w, 1e-5),
                 lambda: ops.residual_norm_backward(x, x, x, w, 1e-5),
                 lambda: capture.save_rows(x, None, q, i, i),
                 lambda: ops.rotary(x.view(2, 2, 32), i.expand(2).contiguous(), plan),
                 lambda: ops.rotary_plan(64, 1e4, device="cpu")):
        with pytest.raises(ValueError):
            call()


def test_save_rows8_refusals():
    good = [A, 64, None, 0, 10, 0, A, A, 4, 64, A, 64, A, 2, 3, 10, None]

    def bad(part, **at):
        args = list(good)
        for i, v in at.items():
            args[int(i[1:])] = v
        _refused("dsb_save_rows8", args, part)

    bad("bf16, fp16 or fp32", _5=3)
    bad("e4m3 or int8", _14=2)
    bad("bad sizes", _8=-1)
    bad("bad sizes", _8=1 << 24)
    bad("bad sizes", _9=-1)
    bad("bad sizes", _4=-1)
    bad("together", _6=None)
    bad("past the rows", _6=None, _7=None, _8=11)
    bad("null", _0=None)
    bad("null", _10=None)
    bad("null", _12=None)
    bad("aligned", _0=A + 1)
    bad("stride", _1=63)
    bad("stride", _2=A, _3=63)
    bad("stride", _11=63)
    bad("stride", _13=1)


def test_restore_rows8_refusals():
    good = [A, 64, A, 2, 3, 4, 64, A, 64, 0, None]
    for part, at in (("e4m3 or int8", {4: 0}), ("bad sizes", {5: -1}), ("bad sizes", {5: 1 << 24}),
                     ("bad sizes", {6: -1}), ("null", {0: None}), ("null", {2: None}), ("null", {7: None}),
                     ("stride", {1: 63}), ("stride", {8: 63}), ("stride", {3: 1}), ("aligned", {7: A + 1})):
        args = [at.get(i, v) for i, v in enumerate(good)]
        _refused("dsb_op_restore_rows8", args, part)


# ---------------------------------------------------------------- SwiGLU

def test_swiglu_refusals():
    good = [A, 128, A, 4, 3, 4, 64, A, 64, 0, A, 128, A, 64, None]
    for part, at in (("multiple of 8", {6: 60}), ("multiple of 8", {6: 0}), ("2^24", {5: 1 << 24}),
                     ("type", {4: 1}), ("type", {4: 2}), ("type", {4: 9}), ("null", {0: None}), ("scale byte", {2: None}),
                     ("scale byte", {3: 3}), ("codes must be", {0: A + 4}), ("codes must be", {1: 132}),
                     ("stride", {1: 120}), ("null", {7: None}), ("16-byte", {7: A + 8}), ("16-byte", {8: 68}),
                     ("null", {10: None}), ("stride", {11: 120}), ("16-byte", {11: 132}), ("16-byte", {12: A + 2}),
                     ("stride", {13: 56})):
        _refused("dsb_op_swiglu_bwd", [at.get(i, v) for i, v in enumerate(good)], part)
    good = [A, 128, None, 0, 0, 4, 64, A, 64, None]
    for part, at in (("multiple of 8", {6: 12}), ("type", {4: 2}), ("16-byte", {0: A + 8}), ("null", {7: None})):
        _refused("dsb_op_swiglu", [at.get(i, v) for i, v in enumerate(good)], part)
    from deltaserve_amd import ops

    with pytest.raises(ValueError, match="multiple of 8"):
        ops.swiglu(torch.zeros(2, 24, dtype=BF16))
    with pytest.raises(ValueError, match="dh"):
        ops.swiglu_backward(torch.zeros(2, 32, dtype=BF16), torch.zeros(2, 32, dtype=BF16))


# ---------------------------------------------------------------- the join

def test_norm_join_refusals():
    good = dict(x=A, ldx=64, xs=None, ldxs=0, xt=0, y=A, ldy=64, w_out=A, w_in=A, gate=A, ldg=64, kind=3,
                scale=1.0, eps=1e-5, rows=4, D=64, x_new=A, ldxn=64, normed=A, ldn=64, stream=None)

    def bad(part, **at):
        _refused("dsb_op_norm_join", list({**good, **at}.values()), part)

    bad("multiple of 8", D=60)
    bad("multiple of 8", D=8200)
    bad("2^24", rows=1 << 24)
    bad("2^24", rows=-1)
    for v in (math.nan, math.inf, -1.0):
        bad("eps", eps=v)
    bad("scale", scale=math.inf)
    bad("kind of gate", kind=4)
    bad("do not match", kind=0)
    bad("do not match", gate=None)
    bad("block's", x_new=None)
    bad("type", xt=3, xs=A, ldxs=2)
    bad("type", xt=1)
    bad("null", x=None)
    bad("null", y=None)
    bad("together", w_in=None)
    bad("together", normed=None)
    bad("is null", x_new=None, w_out=None, gate=None, kind=0)
    bad("stride", ldy=56)
    bad("16-byte", ldy=68)
    bad("16-byte", x_new=A + 8)
    bad("weights", w_out=A + 8)
    bad("gate", kind=1, gate=A + 8)
    bad("bad gate", kind=2, ldg=0)
    bad("stride", kind=3, ldg=8)
    bad("16-byte", ldn=65)


def test_norm_join_backward_refusals():
    good = dict(x=A, ldx=64, xs=A, ldxs=2, xt=3, y=A, ldy=64, ys=A, ldys=2, yt=4, dn=A, lddn=64, dnf=0,
                dxn=A, lddxn=64, dxnf=1, w_out=A, w_in=A, gate=A, ldg=0, kind=1, scale=1.0, eps=1e-5,
                rows=4, D=64, dx=A, lddx=64, dxf=1, dy=A, lddy=64, dgate=A, lddg=64, dw_out=A, dw_in=A,
                work=A, bytes=1 << 20, stream=None)

    def bad(part, **at):
        _refused("dsb_op_norm_join_bwd", list({**good, **at}.values()), part)

    bad("multiple of 8", D=4)
    bad("eps", eps=-1.0)
    bad("type", xt=1)
    bad("type", yt=2)
    bad("scale byte", xs=None)
    bad("scale byte", ldys=1)
    bad("codes must be", y=A + 4)
    bad("together", dn=None)
    bad("together", w_in=None, dw_in=None)
    bad("no gradient", dn=None, w_in=None, dw_in=None, dxn=None)
    bad("without the weight", w_out=None)
    bad("without the weight", w_in=None)
    bad("without a gate", gate=None, kind=0)
    bad("block's", dy=None)
    alone = dict(dy=None, w_out=None, dw_out=None, gate=None, kind=0, dgate=None)
    bad("dy is null", **alone, dw_in=None)
    bad("comes with a block", **alone)
    bad("neither a block nor a norm", **alone, y=None, dn=None, w_in=None, dw_in=None)
    bad("null", kind=3, ldg=64, dgate=None)
    bad("null", dx=None)
    bad("null", y=None)
    bad("stride", lddx=56)
    bad("16-byte", lddxn=66)
    bad("16-byte", kind=3, ldg=64, lddg=68)
    bad("vectors", dw_in=A + 4)
    bad("vectors", dgate=A + 4)
    bad("too small", bytes=8 * 4 * 64 - 1)
    bad("too small", work=None)
    bad("workspace must", work=A + 4)


def test_norm_join_workspace():
    L, lib = _lib()
    b = ctypes.c_int64(-1)
    for rows, D, sums, want in ((0, 64, 1, 0), (4, 64, 1, 8 * 4 * 64), (4, 64, 0, 0)):
        assert lib.dsb_op_norm_join_workspace(rows, D, sums, ctypes.byref(b)) == 0 and b.value == want
    for args in ((-1, 64, 1, ctypes.byref(b)), (1, 65, 1, ctypes.byref(b)), (1, 64, 1, None)):
        _refused("dsb_op_norm_join_workspace", args, "bad argument")


def test_join_arguments_are_checked():
    from deltaserve_amd import ops
    from deltaserve_amd.rows8 import Rows8

    x, w = torch.zeros(3, 64, dtype=BF16), torch.ones(64, dtype=BF16)
    q = Rows8.zeros(3, 64, device="cpu")
    for call in (lambda: ops.residual_norm(q, x, w, 1e-5),
                 lambda: ops.residual_norm(x, x.float(), w, 1e-5),
                 lambda: ops.residual_norm(x, x[:2], w, 1e-5),
                 lambda: ops.residual_norm(x.half(), x, w, 1e-5),
                 lambda: ops.residual_norm(x, x, w.float(), 1e-5),
                 lambda: ops.residual_norm(x, x, w[:32], 1e-5),
                 lambda: ops.residual_norm(x, x, w, 1e-5, gate=w[:5]),
                 lambda: ops.residual_norm(x, x, w, 1e-5, gate=w.float()),
                 lambda: ops.residual_norm(x, x, w, 1e-5, gate=torch.zeros(3, 1)),
                 lambda: ops.residual_norm(x, x, w, 1e-5, gate=x.float()),
                 lambda: ops.residual_norm(x.t().contiguous().t(), x, w, 1e-5),
                 lambda: ops.residual_norm_backward(x, x, None, w, 1e-5, dx_new=x),
                 lambda: ops.residual_norm_backward(x, x, x, None, 1e-5),
                 lambda: ops.residual_norm_backward(x, x, None, None, 1e-5),
                 lambda: ops.residual_norm_backward(x[:2], x, x, w, 1e-5),
                 lambda: ops.residual_norm_backward(x, x, x.half(), w, 1e-5),
                 lambda: ops.residual_norm_backward(x, x, x, w, 1e-5, dx_new=x[:, :32])):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- rotary positions

def _freq(d, theta, scaling=None, seq_len=None):
    from deltaserve_amd.ops import _rotary_frequencies

    return _rotary_frequencies(d, theta, scaling, seq_len)


def test_rotary_frequencies():
    i = np.arange(32)
    inv = 1e4 ** (-2 * i / 64)
    plain, f = _freq(64, 1e4)
    assert f == 1 and np.allclose(plain, inv, rtol=1e-14)
    lin, f = _freq(64, 1e4, {"rope_type": "linear", "factor": 4})
    assert f == 1 and np.allclose(lin, inv / 4, rtol=1e-14)
    # as the cycle has llama3, whose arithmetic is fp32
    from deltaserve_amd import ops

    rs = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    ll, f = _freq(64, 5e5, rs)
    assert f == 1 and np.allclose(ll, ops.rope_inv_freq(64, 5e5, rs).numpy(), rtol=4e-6)
    # dynamic: theta so that position now·... turns as the original's length did: unscaled within it
    dyn = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}
    assert np.allclose(_freq(64, 1e4, dyn)[0], inv) and np.allclose(_freq(64, 1e4, dyn, 1000)[0], inv)
    far = _freq(64, 1e4, dyn, 4096)[0]
    assert far[0] == 1 and np.allclose(far[-1], inv[-1] / 3, rtol=1e-12)  # by s·now/length − (s − 1)
    # yarn: pairs that turn often keep their frequency, those that turn less than once are divided
    yarn = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    y, f = _freq(64, 1e4, yarn)
    assert f == pytest.approx(0.1 * math.log(16) + 1)
    turns = 4096 * inv / (2 * math.pi)
    # (borders are whole pairs: one either way is left out)
    assert np.allclose(y[turns > 32 * 1e4 ** (2 / 64)], inv[turns > 32 * 1e4 ** (2 / 64)])
    assert np.allclose(y[turns < 1e4 ** (-2 / 64)], inv[turns < 1e4 ** (-2 / 64)] / 16)
    assert (np.diff(y) < 0).all() and (y <= inv).all() and (y >= inv / 16).all()
    assert _freq(64, 1e4, {**yarn, "attention_factor": 1.5})[1] == 1.5
    for above, below in ((1.0, 0.0), (0.707, 0.707), (1.0, 0.5), (0.0, 0.5), (2.0, None)):
        f = _freq(64, 1e4, {**yarn, "mscale": above, "mscale_all_dim": below})[1]
        grow = 0.1 * math.log(16)
        assert f == pytest.approx((above * grow + 1) / ((below or 0) * grow + 1), rel=1e-14)
    assert _freq(64, 1e4, {**yarn, "factor": 0.5, "mscale": 2.0})[1] == 1
    # borders between pairs: the share that is divided is the pair's place between them, exactly
    cut = _freq(64, 1e4, {**yarn, "truncate": False})[0]
    at = [64 * math.log(4096 / (b * 2 * math.pi)) / (2 * math.log(1e4)) for b in (32, 1)]
    share = np.clip((i - at[0]) / (at[1] - at[0]), 0, 1)
    assert np.allclose(cut, inv * (1 - share * (1 - 1 / 16)), rtol=1e-12) and not np.allclose(cut, y, rtol=1e-3)
    lr = {"rope_type": "longrope", "factor": 4.0, "original_max_position_embeddings": 4096,
          "short_factor": [1.0] * 32, "long_factor": list(range(1, 33))}
    assert np.allclose(_freq(64, 1e4, lr, 4096)[0], inv)
    far, f = _freq(64, 1e4, lr, 4097)
    assert np.allclose(far, inv / np.arange(1, 33)) and f == pytest.approx(math.sqrt(1 + math.log(4) / math.log(4096)))


def test_rotary_plans_are_checked():
    from deltaserve_amd import ops

    for args, kw in (((64, 1e4), dict(rotary_dim=63)), ((64, 1e4), dict(rotary_dim=66)), ((64, 1e4), dict(rotary_dim=0)),
                     ((2048, 1e4), {}), ((63, 1e4), {}), ((64, 1.0), {}), ((64, math.nan), {}),
                     ((64, 1e4, {"rope_type": "linear"}), {}), ((64, 1e4, {"rope_type": "linear", "factor": 0}), {}),
                     ((64, math.inf), {}), ((64, 1e4, {"rope_type": "yarn", "factor": 2}), {}),
                     ((64, 1e4, {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 64,
                                 "mscale": -1.0}), {}),
                     ((64, 1e4, {"rope_type": "llama3", "factor": 2, "original_max_position_embeddings": 64,
                                 "low_freq_factor": 4, "high_freq_factor": 4}), {}),
                     ((64, 1e4, {"rope_type": "longrope", "factor": 2, "original_max_position_embeddings": 64,
                                 "short_factor": [1.0] * 31}), {}),
                     ((2, 1e4, {"rope_type": "dynamic", "factor": 2, "original_max_position_embeddings": 64}), {})):
        with pytest.raises(ValueError):
            ops.rotary_plan(*args, device="cpu", **kw)
    with pytest.raises(NotImplementedError):
        ops.rotary_plan(64, 1e4, {"rope_type": "su"}, device="cpu")


def test_rotary_refusals():
    good = dict(x=A, ldx=256, hx=64, y=2 * A, ldy=256, hy=64, dt=0, pos=A, p64=0, turns=A, factor=1.0, n=4,
                heads=4, hd=64, rot=64, inter=0, inv=0, stream=None)

    def bad(part, **at):
        _refused("dsb_op_rotary", list({**good, **at}.values()), part)

    bad("bf16, fp16 or fp32", dt=3)
    bad("even", rot=63)
    bad("even", rot=0)
    bad("even", rot=66)
    bad("1024", hd=1026, rot=64)
    bad("2^24", n=1 << 24)
    bad("2^20", heads=1 << 15)
    bad("2^24", n=-1)
    bad("overlap", hy=63)
    bad("overlap", ldy=0)
    bad("factor", factor=math.nan)
    bad("null", x=None)
    bad("null", turns=None)
    bad("null", pos=None)
    bad("aligned", x=A + 1)
    bad("aligned", pos=A + 4, p64=1)
    bad("aligned", turns=A + 4)
    bad("in place", y=A, ldy=512)
    from deltaserve_amd import ops

    plan = ops.RotaryPlan(64, 64, False, np.ones(32), 1.0, "cpu")
    x, p = torch.zeros(2, 3, 64, dtype=BF16), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.rotary(x[..., :32], p, plan), lambda: ops.rotary(x.double(), p, plan),
                 lambda: ops.rotary(x[0], p, plan), lambda: ops.rotary(x, p[:1], plan),
                 lambda: ops.rotary(x, p.float(), plan)):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- the store in 8 bits, around the cycle

def test_rows8_go_between_processes_and_are_fingerprinted_and_wiped():
    import pickle

    from deltaserve_amd import integrity
    from deltaserve_amd.bwd_services.base import BackwardService
    from deltaserve_amd.rows8 import Rows8

    q = Rows8.zeros(5, 40, "int8", "cpu")
    q.codes.copy_(torch.arange(200, dtype=torch.int8).view(5, 40))
    q.scales.fill_(120)
    p = pickle.loads(pickle.dumps(q))
    assert type(p) is Rows8 and torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    assert (p.type, p.shape, p.ld_scales) == (q.type, q.shape, q.ld_scales)
    acts = {"layer_in": [q, p], "concat_input_ids": torch.arange(5)}
    rep = integrity.activation_hash_report(acts, 4)
    assert rep["layer_in_first"] == rep["layer_in_last"] != integrity.tensor_digest(q[:3])
    p.scales[0, 0] = 121
    assert integrity.activation_hash_report(acts, 4)["layer_in_last"] != rep["layer_in_last"]
    svc = BackwardService.__new__(BackwardService)
    svc.activations = acts
    svc._wipe_activations()
    assert (q.codes == 0).all() and (q.scales == 1).all() and (acts["concat_input_ids"] == 0).all()


def test_a_store_in_8_bits_on_the_host():
    from deltaserve_amd.capture import ActivationStore
    from deltaserve_amd.rows8 import Rows8

    s = ActivationStore(2, 64, 10, device="cpu", intermediate_size=96, code="e4m3")
    assert all(isinstance(b, Rows8) and b.shape == (11, 64) for b in s.layer_in)
    assert all(b.shape == (11, 192) for b in s.mlp_gate_up) and torch.is_tensor(s.final_in)
    s.layer_in[0].codes.view(torch.uint8).fill_(9)
    s.zero_offset_range(3, 4)
    rows = s.layer_in[0].codes.view(torch.uint8)[:, 0]
    assert rows.tolist() == [9] * 3 + [0] * 4 + [9] * 4
    with pytest.raises(ValueError):
        ActivationStore(2, 64, 10, device="cpu", code="int4")


def test_rows8_struct_matches_header(tmp_path):
    import os
    import subprocess

    from harness import ROOT

    L, _ = _lib()
    src = tmp_path / "p.c"
    names = [f for f, _ in L.DsbRows8._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dsb.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu ", offsetof(dsb_rows8, {f}));\n' for f in names)
                   + 'printf("%zu", sizeof(dsb_rows8)); return 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src),
                    "-o", str(tmp_path / "p")], check=True)
    got = subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == [*(getattr(L.DsbRows8, f).offset for f in names), ctypes.sizeof(L.DsbRows8)]
