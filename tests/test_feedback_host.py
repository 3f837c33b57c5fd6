"""The operators for training from feedback without a GPU: packing plans against a plain
construction, the C structs' layouts, and the refusals, which come before any device call."""

from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from harness import ROOT


def _lib():
    from deltaserve_amd import _lib as L

    return L, L.load()


def _plan(lens):
    """(struct, tables as a list of arrays) with device_base 0: its pointers are byte offsets."""
    L, lib = _lib()
    arr = L.i32_array(lens)
    c, elems = L.DsbPackPlan(), ctypes.c_int64()
    assert lib.dsb_plan_sizes(arr, len(lens), ctypes.byref(c), ctypes.byref(elems)) == 0
    host = np.full(elems.value, -7, dtype=np.int32)
    base = 1 << 20
    assert lib.dsb_plan_fill(arr, ctypes.byref(c), host.ctypes.data, base) == 0
    at = [((getattr(c, k) or 0) - base) // 4 for k in ("tiles", "seq_tile", "starts", "chunk_seq")]
    assert all(a % 4 == 0 for a in at)
    chunks = -(-c.n // 4096) + 1
    sizes = [4 * c.ntiles, c.nseq + 1, c.nseq + 1, chunks]
    assert at[-1] + sizes[-1] <= elems.value
    return c, [host[a:a + s] for a, s in zip(at, sizes)]


@pytest.mark.parametrize("lens", [[], [0], [1], [5, 0, 3], [0, 0, 4096, 0], [4097, 1, 0, 8192],
                                  [1] * 9000, [20000], list(range(200))])
def test_plan_tables(lens):
    c, (tiles, seq_tile, starts, chunk) = _plan(lens)
    n = sum(lens)
    assert (c.n, c.nseq, c.npred, c.nonempty) == (n, len(lens), sum(max(x - 1, 0) for x in lens),
                                                  sum(x > 1 for x in lens))
    assert c.longest == max(lens, default=0)
    want = np.concatenate([[0], np.cumsum(lens)]).astype(int)
    assert starts.tolist() == want.tolist()
    tiles = tiles.reshape(-1, 4)
    seq = np.full(n, -1)
    for i, (r0, r1, s, z) in enumerate(tiles.tolist()):
        assert 0 < r1 - r0 <= 4096 and z == 0 and seq_tile[s] <= i < seq_tile[s + 1]
        assert want[s] <= r0 and r1 <= want[s + 1] and (seq[r0:r1] == -1).all()
        seq[r0:r1] = s
    assert (seq >= 0).all() and seq_tile[-1] == len(tiles)
    assert [seq[4096 * i] for i in range(len(chunk) - 1)] == chunk[:-1].tolist()
    assert chunk[-1] == max(len(lens) - 1, 0)


def test_plan_refusals():
    L, lib = _lib()
    c, e = L.DsbPackPlan(), ctypes.c_int64()
    ref = ctypes.byref
    assert lib.dsb_plan_sizes(L.i32_array([3, -1]), 2, ref(c), ref(e)) != 0
    assert "negative" in L.last_error()
    assert lib.dsb_plan_sizes(L.i32_array([2**31 - 1, 2]), 2, ref(c), ref(e)) != 0
    assert lib.dsb_plan_sizes(None, 1, ref(c), ref(e)) != 0
    assert lib.dsb_plan_sizes(L.i32_array([3, 4]), 2, ref(c), ref(e)) == 0
    host = (ctypes.c_int32 * e.value)()
    assert lib.dsb_plan_fill(L.i32_array([3, 5]), ref(c), host, None) != 0  # other lengths
    assert lib.dsb_plan_fill(L.i32_array([3, 3]), ref(c), host, None) != 0
    from deltaserve_amd import ops

    with pytest.raises(ValueError):
        ops.pack_plan([3, -1])
    with pytest.raises(ValueError):
        ops.pack_plan([3], device="cpu")


def test_struct_layouts(tmp_path):
    L, _ = _lib()
    structs = {"dsb_pack_plan": L.DsbPackPlan, "dsb_adam_chunk": L.DsbAdamChunk}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dsb.h"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'  printf("%zu", sizeof({name}));')
        lines += [f'  printf(" %zu", offsetof({name}, {f}));' for f, _ in cls._fields_]
        lines.append('  printf("\\n");')
    src = tmp_path / "p.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src),
                    "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout
    for line, cls in zip(out.splitlines(), structs.values()):
        assert [int(x) for x in line.split()] == [ctypes.sizeof(cls)] + [
            getattr(cls, f).offset for f, _ in cls._fields_]


FAKE = 1 << 20  # an aligned stand-in for an address; the refused calls never read it
BIG = 1 << 40


def _lp(lib, **kw):
    a = dict(h=FAKE, ld=64, w=FAKE, lab=FAKE, n=4, D=64, V=100, logp=FAKE, other=FAKE, work=FAKE,
             nbytes=BIG)
    a.update(kw)
    return lib.dsb_op_token_logprobs(*[a[k] for k in ("h", "ld", "w", "lab", "n", "D", "V", "logp",
                                                      "other", "work", "nbytes")], None)


@pytest.mark.parametrize("bad", [dict(ld=63), dict(ld=60), dict(D=60), dict(D=0), dict(V=1), dict(n=-1),
                                 dict(h=FAKE + 2), dict(w=FAKE + 8), dict(lab=None), dict(logp=None),
                                 dict(work=None), dict(nbytes=100), dict(work=FAKE + 16),
                                 dict(V=(1 << 24) + 1), dict(n=(1 << 30) + 1)])
def test_logprob_refusals(bad):
    L, lib = _lib()
    assert _lp(lib, **bad) != 0 and L.last_error()


def test_logprob_empty_is_nothing_to_do():
    _, lib = _lib()
    assert _lp(lib, n=0, h=None, w=None, lab=None, work=None, nbytes=0) == 0


@pytest.mark.parametrize("bad", [dict(ldd=60), dict(dh=FAKE + 4), dict(g=None), dict(nbytes=64)])
def test_logprob_backward_refusals(bad):
    L, lib = _lib()
    a = dict(g=FAKE, dh=FAKE, ldd=64, nbytes=BIG)
    a.update(bad)
    rc = lib.dsb_op_token_logprobs_bwd(FAKE, 64, FAKE, FAKE, 4, 64, 100, FAKE, FAKE, a["g"], a["dh"],
                                       a["ldd"], 0, FAKE, a["nbytes"], None)
    assert rc != 0 and L.last_error()


def _losses(lib, L, lens):
    c, _ = _plan(lens)

    def pref(**kw):
        a = dict(logp=FAKE, ref=FAKE, mask=FAKE, plan=ctypes.byref(c), kind=0, beta=0.1, smooth=0.0,
                 margin=0.0, average=0, scale=1.0, loss=FAKE, rewards=FAKE, d=FAKE, work=FAKE, nbytes=BIG)
        a.update(kw)
        return lib.dsb_op_preference_loss(*a.values(), None)

    def policy(**kw):
        a = dict(logp=FAKE, old=FAKE, ref=FAKE, adv=FAKE, rows=1, mask=FAKE, plan=ctypes.byref(c), low=0.2,
                 high=0.2, coef=0.1, kl=0, red=0, div=1.0, scale=1.0, out=FAKE, d=FAKE, work=FAKE,
                 nbytes=BIG)
        a.update(kw)
        return lib.dsb_op_policy_loss(*a.values(), None)

    return c, pref, policy


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("bad", [dict(kind=3), dict(kind=-1), dict(beta=0.0), dict(beta=NAN),
                                 dict(beta=INF), dict(smooth=-0.1), dict(smooth=1.5), dict(margin=INF),
                                 dict(kind=1, smooth=0.1), dict(kind=2, margin=0.1), dict(logp=None),
                                 dict(logp=FAKE + 2), dict(loss=None), dict(rewards=None), dict(d=None),
                                 dict(work=None), dict(nbytes=1), dict(plan=None)])
def test_preference_refusals(bad):
    L, lib = _lib()
    c, pref, _ = _losses(lib, L, [4000, 5000])
    assert pref(**bad) != 0 and L.last_error()


@pytest.mark.parametrize("lens", [[], [4], [4, 5, 6]])
def test_preference_needs_pairs(lens):
    L, lib = _lib()
    c, pref, _ = _losses(lib, L, lens)
    assert pref() != 0 and "pairs" in L.last_error()


@pytest.mark.parametrize("bad", [dict(low=-0.1), dict(low=1.1), dict(high=-0.1), dict(high=NAN), dict(kl=2),
                                 dict(red=3), dict(ref=None), dict(coef=INF), dict(red=2, div=0.0),
                                 dict(red=2, div=NAN), dict(adv=None), dict(old=None), dict(out=None),
                                 dict(d=None), dict(adv=FAKE + 1), dict(nbytes=1), dict(plan=None)])
def test_policy_refusals(bad):
    L, lib = _lib()
    c, _, policy = _losses(lib, L, [4000, 5000])
    assert policy(**bad) != 0 and L.last_error()


@pytest.mark.parametrize("bad", [dict(bits=4), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0),
                                 dict(eps=INF), dict(lr=NAN), dict(wd=INF), dict(step=0), dict(maxn=NAN),
                                 dict(maxn=1.0, norms=None), dict(m=None), dict(v=FAKE + 4),
                                 dict(ms=None), dict(chunks=None), dict(ngroups=0), dict(nbytes=8),
                                 dict(work=FAKE + 8), dict(nchunks=-1), dict(most=2),
                                 dict(most=-1)])
def test_adam_refusals(bad):
    L, lib = _lib()
    a = dict(chunks=FAKE, nchunks=1, gc=FAKE, ngroups=1, most=1, m=FAKE, v=FAKE, ms=FAKE, rs=FAKE,
             bits=8, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.0, maxn=-1.0, step=1, seed=0,
             lrd=None, stepd=None, norms=FAKE, work=FAKE, nbytes=BIG)
    a.update(bad)
    assert lib.dsb_op_adam_step(*a.values(), None) != 0 and L.last_error()


def test_front_end_refusals():
    from deltaserve_amd import ops

    f, b = torch.zeros(4), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.token_logprobs(b, b, torch.zeros(4, dtype=torch.int64))  # host tensors
    for lens in ([1.5, 2.0], [3, -1], [1 << 31], ["3"], [True]):
        with pytest.raises(ValueError):
            ops.pack_plan(lens)
    with pytest.raises(ValueError):
        ops.token_logprobs(b.float(), b, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.token_logprobs(b, b[:, :4], torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.token_logprobs(b, b, torch.zeros(4, dtype=torch.int32))
    for bad in (dict(ws=[], gs=[]), dict(ws=[f], gs=[f, f]), dict(ws=[f], gs=[f], bits=16),
                dict(ws=[f], gs=[f[:2]]), dict(ws=[f.half()], gs=[f]), dict(ws=[f], gs=[f], groups=[-1]),
                dict(ws=[f, f.clone()], gs=[f, f], groups=[1, 0]), dict(ws=[f, f[1:]], gs=[f, f[1:]]),
                dict(ws=[f], gs=[f], groups=[1 << 20]), dict(ws=[b.t()], gs=[b.t()]), dict(ws=[f], gs=[f])):
        with pytest.raises(ValueError):
            ops.AdamW(**bad)


def _mix(x):
    x = x & 0xffffffff
    x = x ^ (x >> 16)
    x = (x * 0x6a09e667) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0xbb67ae85) & 0xffffffff
    return x ^ (x >> 16)


def test_rounding_numbers_are_even():
    """The numbers that round the second moments, over neighbouring steps and blocks: each of 16
    bits set half the time, neighbours uncorrelated, the mean over an element's steps near a half. The
    bounds are 6 standard deviations of independent fair draws."""
    steps, blocks = torch.arange(1, 65), torch.arange(64)
    key = _mix(torch.tensor(3) + steps * 0x9e3779b9)
    key = _mix(key[:, None] ^ _mix(blocks)[None])
    x = _mix(key[..., None] + torch.arange(128) * 0x9e3779b9)
    n = x.numel()
    for bit in range(32):
        share = ((x >> bit) & 1).double().mean().item()
        assert abs(share - 0.5) < 6 * 0.5 / n ** 0.5, bit
    u = torch.stack([x & 0xffff, x >> 16], 3).double().add(0.5).div(65536)
    c = (u - 0.5) * 12 ** 0.5
    for dim in range(4):
        a, b = c.narrow(dim, 0, c.shape[dim] - 1), c.narrow(dim, 1, c.shape[dim] - 1)
        assert abs((a * b).mean().item()) < 6 / a.numel() ** 0.5, dim
    per = u.mean(0)  # over the 64 steps of each of 16384 elements
    assert (per - 0.5).abs().max().item() < 6 * (1 / 12) ** 0.5 / 8
