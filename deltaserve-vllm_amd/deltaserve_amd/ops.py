"""Torch-tensor front end of libdsb's single-op entry points.

Each function mirrors one op of the reference's ``bwd_services/common``
modules (cited per function; paths under ``deltaserve-plugin/deltaserve/``)
and runs the HIP kernel on the current torch stream. Inputs are bf16 CUDA
tensors with a contiguous last dimension (row strides are passed through);
nothing here falls back to a PyTorch implementation.
"""

from __future__ import annotations

import contextlib
import ctypes
from ctypes import byref, c_float, c_int, c_int32, c_int64, c_void_p

import numpy as np
import torch

from . import _lib as L

BF16 = torch.bfloat16


def _stream():
    return c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t):
    return None if t is None else c_void_p(t.data_ptr())


def _ld(t):
    assert t.stride(-1) == 1, "last dimension must be contiguous"
    return t.stride(0) if t.dim() > 1 else t.shape[0]


def _dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("deltaserve_amd ops take CUDA (HIP) tensors")


def release_workspaces():
    """Free the scratch memory the ops keep between calls (the next call
    allocates again)."""
    L.check(L.load().dsb_release_workspaces(), what="dsb_release_workspaces")


# ---------------------------------------------------------------- integer packing

def pack(seq_lens):
    """trainer.py:510-518, head.py:63-72 via libdsb: (positions, pred, n_valid)."""
    lib = L.load()
    n = int(sum(int(s) for s in seq_lens))
    arr = L.i32_array(seq_lens)
    pos = (c_int32 * max(n, 1))()
    pred = (c_int32 * max(n, 1))()
    nv = lib.dsb_pack(arr, len(seq_lens), n, pos, pred)
    if nv < 0:
        raise ValueError("seq_lens must be non-negative")
    return list(pos)[:n], list(pred)[:n], nv


def rope_inv_freq(head_dim, theta, rope_scaling=None):
    """ops.py:26-57 via libdsb (host), as a CPU float32 tensor."""
    lib = L.load()
    rs = rope_scaling or {}
    rtype = rs.get("rope_type", "default") or "default"
    code = {"default": L.ROPE_DEFAULT, "linear": L.ROPE_LINEAR, "llama3": L.ROPE_LLAMA3}.get(rtype)
    if code is None:
        raise NotImplementedError(f"RoPE type {rtype!r} is not supported")
    out = (c_float * (head_dim // 2))()
    L.check(lib.dsb_rope_inv_freq(head_dim, float(theta), code, float(rs.get("factor", 1.0)),
                                  float(rs.get("low_freq_factor", 1.0)),
                                  float(rs.get("high_freq_factor", 1.0)),
                                  float(rs.get("original_max_position_embeddings", 1.0)), out))
    return torch.tensor(list(out), dtype=torch.float32)


# ---------------------------------------------------------------- dense products

def gemm_plan(M, N, K, out_bytes):
    """(tile, K slices) that a product takes by the cost model; ``out_bytes``
    read and written per output element."""
    tile, slices = c_int(), c_int()
    L.check(L.load().dsb_gemm_plan(M, N, K, float(out_bytes), byref(tile), byref(slices)),
            what="dsb_gemm_plan")
    return tile.value, slices.value


def gemm_nt(A, B, A2=None, B2=None, out_dtype=BF16, R=None, out=None, accumulate=False, cfg=-1,
            b_kn=False, slices=0):
    """C = A·Bᵀ (+ A2·B2ᵀ) (+ R) — the projection products of ops.py:103-146.
    b_kn: B [K1, N] and B2 [K2, N] (C = A·B + A2·B2, the backward's dY·W with W
    in its own layout). ``slices`` 2 to 16: tile ``cfg`` (0 to 4) in that many K
    slices instead of the cost model's choice."""
    _dev(A, B, A2, B2, R)
    M, K1 = A.shape
    N = B.shape[1] if b_kn else B.shape[0]
    K2 = 0 if A2 is None else A2.shape[1]
    f32 = out_dtype == torch.float32
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=A.device)
    args = (_p(A), _ld(A), _p(B), _ld(B), _p(A2), 0 if A2 is None else _ld(A2),
            _p(B2), 0 if B2 is None else _ld(B2), M, N, K1, K2, _p(out),
            _ld(out), int(f32), int(accumulate), _p(R),
            0 if R is None else _ld(R), int(bool(b_kn)), int(cfg))
    if slices:
        L.check(L.load().dsb_op_gemm_split(*args, int(slices), _stream()), what="dsb_op_gemm_split")
    else:
        L.check(L.load().dsb_op_gemm(*args, _stream()), what="dsb_op_gemm")
    return out


def gemm_glu(A, B, A2=None, B2=None, with_h=True):
    """Gate‖up product with the SwiGLU forward fused (ffn.py:25-26, silu as
    ffn.py:40-41): returns (GU [M, 2I] = bf16(A·Bᵀ (+ A2·B2ᵀ)) with B = gate
    rows then up rows, H [M, I] = bf16(silu(gate)·up) or None)."""
    _dev(A, B, A2, B2)
    M, K1 = A.shape
    I = B.shape[0] // 2
    K2 = 0 if A2 is None else A2.shape[1]
    GU = torch.empty(M, 2 * I, dtype=BF16, device=A.device)
    H = torch.empty(M, I, dtype=BF16, device=A.device) if with_h else None
    L.check(L.load().dsb_op_gemm_glu(_p(A), _ld(A), _p(B), _ld(B), _p(A2),
                                     0 if A2 is None else _ld(A2), _p(B2),
                                     0 if B2 is None else _ld(B2), M, I, K1, K2, _p(GU), _ld(GU),
                                     _p(H), 0 if H is None else _ld(H), _stream()),
            what="dsb_op_gemm_glu")
    return GU, H


# ---------------------------------------------------------------- norms / rope

def rmsnorm(x, w, eps):
    """ops.py:84-88 (bf16 in/out, fp32 internals)."""
    _dev(x, w)
    y = torch.empty(x.shape, dtype=BF16, device=x.device)
    L.check(L.load().dsb_op_rmsnorm(_p(x), _ld(x), _p(w), _p(y), _ld(y), x.shape[0], x.shape[1],
                                    float(eps), _stream()), what="dsb_op_rmsnorm")
    return y


def rmsnorm_backward(x, g, w, eps, resid=None):
    """ops.py:91-100 (+ bf16 residual add, llama3.py:205); bf16 out. An fp32 g
    [parts, n, D] is added up in order first."""
    _dev(x, g, w, resid)
    out = torch.empty(x.shape, dtype=BF16, device=x.device)
    if g.dim() == 3:
        assert g.dtype == torch.float32 and g.stride(2) == 1
        L.check(L.load().dsb_op_rmsnorm_bwd_parts(
            _p(x), _ld(x), _p(g), g.stride(1), g.shape[0], g.stride(0), _p(w), _p(resid),
            0 if resid is None else _ld(resid), _p(out), _ld(out), x.shape[0], x.shape[1],
            float(eps), _stream()), what="dsb_op_rmsnorm_bwd_parts")
        return out
    L.check(L.load().dsb_op_rmsnorm_bwd(_p(x), _ld(x), _p(g), int(g.dtype == torch.float32),
                                        _ld(g), _p(w), _p(resid), 0 if resid is None else _ld(resid),
                                        _p(out), _ld(out), x.shape[0], x.shape[1], float(eps),
                                        _stream()), what="dsb_op_rmsnorm_bwd")
    return out


def rope_cos_sin(positions, inv_freq):
    """ops.py:60-65: cos, sin [n, Hd/2] fp32 from int32 positions (CUDA)."""
    _dev(positions, inv_freq)
    n, half = positions.shape[0], inv_freq.shape[0]
    c = torch.empty(n, half, dtype=torch.float32, device=positions.device)
    s = torch.empty_like(c)
    L.check(L.load().dsb_op_rope_table(_p(positions), n, _p(inv_freq), half, _p(c), _p(s),
                                       _stream()), what="dsb_op_rope_table")
    return c, s


def apply_rope(qkv_pre, Hq, Hkv, cos, sin, q_norm=None, k_norm=None, eps=1e-6):
    """ops.py:68-73 (+ qwen3.py:96-107): rotated [q | k] of a [n, q+2kv] row block
    (head_dim = 2·cos.shape[1]: 128 or 64)."""
    _dev(qkv_pre, cos, sin)
    n, hd = qkv_pre.shape[0], 2 * cos.shape[1]
    out = torch.empty(n, (Hq + Hkv) * hd, dtype=BF16, device=qkv_pre.device)
    L.check(L.load().dsb_op_rope(_p(qkv_pre), _ld(qkv_pre), _p(out), _ld(out), _p(cos), _p(sin),
                                 n, Hq, Hkv, hd, _p(q_norm), _p(k_norm), float(eps), _stream()),
            what="dsb_op_rope")
    return out


def rope_backward_(g, qkv_pre, Hq, Hkv, cos, sin, q_norm=None, k_norm=None, eps=1e-6):
    """ops.py:76-81 (+ qwen3.py:133-144), in place on g's [q | k] columns."""
    _dev(g, qkv_pre, cos, sin)
    L.check(L.load().dsb_op_rope_bwd(_p(g), _ld(g), _p(qkv_pre), _ld(qkv_pre), _p(cos), _p(sin),
                                     g.shape[0], Hq, Hkv, 2 * cos.shape[1], _p(q_norm),
                                     _p(k_norm), float(eps), _stream()), what="dsb_op_rope_bwd")
    return g


# ---------------------------------------------------------------- attention

def attn_forward(q, k, v, seq_lens, Hq, Hkv, head_dim=None):
    """attention.py:20-45 over packed rows: (ctx bf16, o32 fp32, lse [Hq, n] log2);
    head_dim (128 or 64) defaults to q's width over Hq."""
    _dev(q, k, v)
    n = q.shape[0]
    hd = head_dim or q.shape[1] // Hq
    ctx = torch.empty(n, Hq * hd, dtype=BF16, device=q.device)
    o32 = torch.empty(n, Hq * hd, dtype=torch.float32, device=q.device)
    lse = torch.empty(Hq, max(n, 1), dtype=torch.float32, device=q.device)
    L.check(L.load().dsb_op_attn_fwd(_p(q), _ld(q), _p(k), _ld(k), _p(v), _ld(v), _p(ctx),
                                     _ld(ctx), _p(o32), _p(lse), L.i32_array(seq_lens),
                                     len(seq_lens), Hq, Hkv, hd, _stream()),
            what="dsb_op_attn_fwd")
    return ctx, o32, lse


def attn_backward(q, k, v, o32, lse, dout, seq_lens, Hq, Hkv, head_dim=None):
    """attention.py:48-112: (dq, dk, dv) bf16 in [n, H*head_dim]."""
    _dev(q, k, v, o32, lse, dout)
    n = q.shape[0]
    hd = head_dim or q.shape[1] // Hq
    dq = torch.empty(n, Hq * hd, dtype=BF16, device=q.device)
    dk = torch.empty(n, Hkv * hd, dtype=BF16, device=q.device)
    dv = torch.empty(n, Hkv * hd, dtype=BF16, device=q.device)
    L.check(L.load().dsb_op_attn_bwd(_p(q), _ld(q), _p(k), _ld(k), _p(v), _ld(v), _p(o32),
                                     _p(lse), _p(dout), _ld(dout), _p(dq), _ld(dq), _p(dk),
                                     _ld(dk), _p(dv), _ld(dv), L.i32_array(seq_lens),
                                     len(seq_lens), Hq, Hkv, hd, _stream()),
            what="dsb_op_attn_bwd")
    return dq, dk, dv


# ---------------------------------------------------------------- head

def head_backward(normed, lm_w, ids, seq_lens, vocab_chunk=0):
    """head.py:42-100 from the normed rows: (loss, n_valid, dH fp32 [n, D]),
    streaming the vocabulary in chunks of ``vocab_chunk`` columns (0: 16384)."""
    _dev(normed, lm_w, ids)
    n, D = normed.shape
    V = lm_w.shape[0]
    dH = torch.empty(n, D, dtype=torch.float32, device=normed.device)
    loss = c_float(0.0)
    nv = c_int(0)
    L.check(L.load().dsb_op_head(_p(normed), _ld(normed), _p(lm_w), _p(ids), L.i32_array(seq_lens),
                                 len(seq_lens), n, D, V, int(vocab_chunk), _p(dH), byref(loss),
                                 byref(nv), _stream()),
            what="dsb_op_head")
    return loss.value, nv.value, dH


# ---------------------------------------------------------------- LoRA grads / optimizer

def lora_tn(P, X, rg, transpose_out, outs, scale=1.0):
    """ops.py:143-144: scale · Pᵀ·X over rows (grad_A, or grad_B when
    transpose_out); P bf16 [n, R]."""
    _dev(P, X, *outs)
    n, R = P.shape
    C = X.shape[1]
    o = list(outs) + [None] * (3 - len(outs))
    L.check(L.load().dsb_op_lora_tn(_p(P), _ld(P), _p(X), _ld(X), n, R, C, float(scale), _p(o[0]),
                                    _p(o[1]), _p(o[2]), rg, int(transpose_out), _stream()),
            what="dsb_op_lora_tn")
    return outs


def lora_skinny(X, B):
    """ops.py:141-142: bf16(X·Bᵀ) for a rank-r factor B [R, K]."""
    _dev(X, B)
    n, K = X.shape
    R = B.shape[0]
    Z = torch.empty(n, R, dtype=BF16, device=X.device)
    L.check(L.load().dsb_op_lora_skinny(_p(X), _ld(X), _p(B), _ld(B), n, R, K, _p(Z), _ld(Z),
                                        _stream()), what="dsb_op_lora_skinny")
    return Z


def _dual_passes(passes):
    arr = (L.DsbDualPass * len(passes))()
    for i, (G, Z, BT, gZ, gB, scale, tr) in enumerate(passes):
        _dev(G, Z, BT, gZ, gB)
        arr[i] = L.DsbDualPass(G.data_ptr(), _ld(G), Z.data_ptr(), _ld(Z), BT.data_ptr(), _ld(BT),
                               G.shape[1], float(scale), gZ.data_ptr(), _ld(gZ), gB.data_ptr(),
                               int(tr))
    return arr


def lora_dual_batch(passes, n, n_alloc=None, entry="dsb_op_lora_dual"):
    """One launch over 1-3 passes ``(G, Z, BT, gZ_out, gB_out, scale,
    transpose_out)`` of the same rank over the first ``n`` rows (the row
    count read from device memory, partials laid out for ``n_alloc``): per
    pass gZ_out[:n] = bf16(G·BTᵀ) and gB_out = scale·Gᵀ·Z (ops.py:142, :144)."""
    r = passes[0][2].shape[0]
    arr = _dual_passes(passes)
    L.check(getattr(L.load(), entry)(arr, len(passes), int(n), int(n_alloc or n), int(r),
                                     _stream()), what=entry)


def lora_dual(G, Z, BT, scale=1.0, transpose_out=True):
    """ops.py:142 and :144 from one pass over G [n, C]: returns
    (bf16(G·BTᵀ) [n, r], scale·Gᵀ·Z fp32 [C, r] (or [r, C])) for BT = (s·B)ᵀ
    [r, C]; with G = xin, BT = A, Z = grad_Z it gives Z and grad_A."""
    n, C = G.shape
    r = BT.shape[0]
    gZ = torch.empty(n, r, dtype=BF16, device=G.device)
    shape = (C, r) if transpose_out else (r, C)
    gB = torch.empty(*shape, dtype=torch.float32, device=G.device)
    lora_dual_batch([(G, Z, BT, gZ, gB, scale, transpose_out)], n)
    return gZ, gB


def clip_adamw_(ws, gs, ms, vs, groups, lr, step, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.0,
                max_norm=1.0, clip=True):
    """trainer.py:624-636 + :668 over fp32 CUDA tensors (in place)."""
    _dev(*ws, *gs, *ms, *vs)
    k = len(ws)
    arr = lambda ts: (c_void_p * k)(*[t.data_ptr() for t in ts])  # noqa: E731
    L.check(L.load().dsb_op_clip_adamw(arr(ws), arr(gs), arr(ms), arr(vs),
                                       L.i32_array([t.numel() for t in ws]), L.i32_array(groups),
                                       k, max(groups) + 1, float(lr), float(beta1), float(beta2),
                                       float(eps), float(wd), int(step), float(max_norm),
                                       int(clip), _stream()), what="dsb_op_clip_adamw")


# ---------------------------------------------------------------- training from feedback
#
# These ops only enqueue on the current stream of their tensors' device (which need not be
# the current device): no synchronisation, scratch memory from torch's caching allocator, so
# they can be captured into a graph. The reference has no counterpart of them.

_HERE = contextlib.nullcontext()


def _on(what, *ts):
    """A context in which the device that holds all tensors (None: left out) is the current one."""
    dev = -1
    for t in ts:
        if t is not None:
            d = t.get_device()  # -1: not on a device
            if d != dev:
                if d < 0:
                    raise ValueError(f"{what}: takes CUDA (HIP) tensors")
                if dev >= 0:
                    raise ValueError(f"{what}: the tensors are on different devices")
                dev = d
    if dev < 0:
        raise ValueError(f"{what}: takes CUDA (HIP) tensors")
    return _HERE if torch.cuda.current_device() == dev else torch.cuda.device(dev)


def _vec(what, name, t, n, *dtypes):
    """A contiguous vector of n elements of one of the dtypes."""
    if t.dtype not in dtypes or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous vector of {n} elements of "
                         f"{' or '.join(str(d) for d in dtypes)}")


def _at(t):
    """A tensor's address for ctypes (None for None)."""
    return None if t is None else t.data_ptr()


def _now():
    # (torch.cuda.current_stream() builds a stream object: 2.8 µs, this 0.1)
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _work(nbytes, device):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


class PackPlan:
    """Sequences packed row after row: their tables on the device, built once per packing by
    :func:`pack_plan` and read by the losses. ``n`` rows, ``nseq`` sequences."""

    __slots__ = ("n", "nseq", "device", "c", "ref", "tables", "loss_bytes")

    def __init__(self, seq_lens, device):
        lib = L.load()
        lens = np.asarray(seq_lens).reshape(-1)
        if lens.size and (lens.dtype.kind not in "iu" or lens.min() < 0 or lens.max() > 0x7fffffff):
            raise ValueError("pack_plan: lengths must be whole numbers in [0, 2^31)")
        lens = np.ascontiguousarray(lens, dtype=np.int32)
        p = lens.ctypes.data_as(ctypes.POINTER(c_int32))
        c, elems, nbytes = L.DsbPackPlan(), c_int64(), c_int64()
        L.check(lib.dsb_plan_sizes(p, lens.size, byref(c), byref(elems)), what="dsb_plan_sizes")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("pack_plan: the plan's device must be CUDA (HIP)")
        host = torch.empty(max(elems.value, 4), dtype=torch.int32)
        self.tables = torch.empty(host.shape, dtype=torch.int32, device=self.device)
        self.device = self.tables.device
        L.check(lib.dsb_plan_fill(p, byref(c), _p(host), _p(self.tables)), what="dsb_plan_fill")
        self.tables.copy_(host)
        L.check(lib.dsb_op_loss_workspace(byref(c), byref(nbytes)), what="dsb_op_loss_workspace")
        self.c, self.n, self.nseq, self.loss_bytes = c, c.n, c.nseq, nbytes.value
        self.ref = byref(c)


def pack_plan(seq_lens, device="cuda"):
    """The :class:`PackPlan` of packed sequences of these lengths (zeros allowed)."""
    return PackPlan(seq_lens, device)


def _mask(what, mask, n):
    if mask is not None:
        _vec(what, "mask", mask, n, torch.bool, torch.uint8)


def next_token_labels(ids, plan, mask=None):
    """(labels int64 [n], rows bool [n]) of packed token ids [n] int64: the label of a row is its
    sequence's next token, -1 where there is none or ``mask`` (by token: the tokens to score) is
    not set there; ``rows`` marks the rows with a label."""
    what = "next_token_labels"
    _vec(what, "ids", ids, plan.n, torch.int64)
    _mask(what, mask, plan.n)
    with _on(what, ids, mask, plan.tables):
        labels = torch.empty_like(ids)
        rows = torch.empty(plan.n, dtype=torch.bool, device=ids.device)
        L.check(L.load().dsb_op_next_token_labels(_at(ids), _at(mask), plan.ref, _at(labels),
                                                  _at(rows), _now()),
                what="dsb_op_next_token_labels")
    return labels, rows


def _head_args(what, normed, lm_w, labels):
    if normed.dtype != BF16 or lm_w.dtype != BF16 or normed.dim() != 2 or lm_w.dim() != 2:
        raise ValueError(f"{what}: normed and lm_w must be bf16 matrices")
    n, D = normed.shape
    if max(n, D, lm_w.shape[0]) >= 1 << 31:
        raise ValueError(f"{what}: a dimension is too large")
    if lm_w.shape[1] != D or not lm_w.is_contiguous():
        raise ValueError(f"{what}: lm_w must be a contiguous [V, {D}]")
    if n and D > 1 and normed.stride(1) != 1:
        raise ValueError(f"{what}: normed's last dimension must be contiguous")
    _vec(what, "labels", labels, n, torch.int64)
    # the row stride of a single row is any number
    return n, D, lm_w.shape[0], normed.stride(0) if n > 1 else D


def _logprob_work(n, D, V, backward, device):
    nbytes = c_int64()
    L.check(L.load().dsb_op_logprob_workspace(n, D, V, backward, byref(nbytes)),
            what="dsb_op_logprob_workspace")
    return _work(nbytes.value, device), max(nbytes.value, 256)


def token_logprobs(normed, lm_w, labels):
    """Log probabilities of labels through the LM head: normed bf16 [n, D] (final-norm rows, row
    stride a multiple of 8), lm_w bf16 [V, D], labels int64 [n], a negative one unscored. Returns
    fp32 (logp [n] = log softmax(normed·lm_wᵀ)[label], other [n] = the log-sum-exp of the other
    words' logits, which :func:`token_logprobs_backward` takes); 0 on unscored rows, NaN where a
    label is past the vocabulary. Only scored rows cost a product. n and (n / 256)·(V / 256) are below
    2^24."""
    what = "token_logprobs"
    n, D, V, ld = _head_args(what, normed, lm_w, labels)
    with _on(what, normed, lm_w, labels):
        logp = torch.empty(n, dtype=torch.float32, device=normed.device)
        other = torch.empty_like(logp)
        work, nbytes = _logprob_work(n, D, V, 0, normed.device)
        L.check(L.load().dsb_op_token_logprobs(_at(normed), ld, _at(lm_w), _at(labels), n, D, V,
                                               _at(logp), _at(other), _at(work), nbytes, _now()),
                what="dsb_op_token_logprobs")
    return logp, other


def token_logprobs_backward(normed, lm_w, labels, logp, other, dlogp, out_dtype=BF16):
    """The rows' gradient [n, D] (bf16 or fp32) of Σ dlogp·logp, from the forward's logp and other;
    zeros on unscored rows and where dlogp is 0, which cost no product. The probabilities that multiply
    the head are bf16 (2^-9 relative on average, their common part divided out) and the sums fp32, also
    where the result is fp32."""
    what = "token_logprobs_backward"
    n, D, V, ld = _head_args(what, normed, lm_w, labels)
    for name, t in (("logp", logp), ("other", other), ("dlogp", dlogp)):
        _vec(what, name, t, n, torch.float32)
    if out_dtype not in (BF16, torch.float32):
        raise ValueError(f"{what}: out_dtype is bfloat16 or float32")
    with _on(what, normed, lm_w, labels, logp, other, dlogp):
        dH = torch.empty(n, D, dtype=out_dtype, device=normed.device)
        work, nbytes = _logprob_work(n, D, V, 1, normed.device)
        L.check(L.load().dsb_op_token_logprobs_bwd(
            _at(normed), ld, _at(lm_w), _at(labels), n, D, V, _at(logp), _at(other), _at(dlogp),
            _at(dH), D, int(out_dtype == torch.float32), _at(work), nbytes, _now()),
            what="dsb_op_token_logprobs_bwd")
    return dH


def preference_loss(logp, ref_logp, plan, mask=None, kind="sigmoid", beta=0.1, label_smoothing=0.0,
                    margin=0.0, average=False, grad_scale=1.0):
    """Preference loss over pairs and its gradient: sequence 2i of the plan is preferred to 2i + 1.

    logp, ref_logp (or None: 0): fp32 [n] log probabilities by row; mask (bool or uint8 [n]): the
    scored rows, by default every row but the last of its sequence. With s = Σ (logp − ref_logp)
    over a sequence's scored rows (their mean with ``average``) and z = beta·(s_2i − s_2i+1) −
    margin, ``kind`` is "sigmoid" −(1 − ε)·log σ(z) − ε·log σ(−z) with ε ``label_smoothing``,
    "hinge" max(0, 1 − z) or "ipo" (s_2i − s_2i+1 − 1/(2·beta))². Returns fp32 (loss, the mean over
    pairs; rewards [nseq] = beta·s; dlogp [n] = grad_scale·dloss/dlogp)."""
    what = "preference_loss"
    if kind not in L.PREF_KINDS:
        raise ValueError(f"{what}: kind is one of {', '.join(L.PREF_KINDS)}")
    _vec(what, "logp", logp, plan.n, torch.float32)
    if ref_logp is not None:
        _vec(what, "ref_logp", ref_logp, plan.n, torch.float32)
    _mask(what, mask, plan.n)
    with _on(what, logp, ref_logp, mask, plan.tables):
        dlogp = torch.empty_like(logp)
        loss = torch.empty((), dtype=torch.float32, device=logp.device)
        rewards = torch.empty(plan.nseq, dtype=torch.float32, device=logp.device)
        work = _work(plan.loss_bytes, logp.device) if plan.loss_bytes else None
        L.check(L.load().dsb_op_preference_loss(
            _at(logp), _at(ref_logp), _at(mask), plan.ref, L.PREF_KINDS[kind], beta, label_smoothing,
            margin, average, grad_scale, _at(loss), _at(rewards), _at(dlogp), _at(work),
            plan.loss_bytes, _now()), what="dsb_op_preference_loss")
    return loss, rewards, dlogp


def policy_loss(logp, old_logp, adv, plan, mask=None, ref_logp=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, kl="k3", reduction="token", divisor=1.0, grad_scale=1.0):
    """Clipped policy loss with a KL term, and its gradient.

    logp, old_logp, ref_logp (or None): fp32 [n] by row; adv: fp32 advantages by row [n] or by
    sequence [nseq] (n = nseq: by row); mask as in :func:`preference_loss`. With ρ = exp(logp −
    old_logp) a scored row's policy term is −min(ρ·A, clamp(ρ, 1 − clip_low, 1 + clip_high)·A), its
    KL term with u = ref_logp − logp is e^u − 1 − u ("k3") or u²/2 ("k2"). ``reduction``: "token"
    (mean over scored rows), "sequence" (mean over the sequences that have some, of their rows'
    mean) or "sum" (sum / divisor). Returns fp32 (loss = policy + kl_coef·kl; stats [3] = policy, kl,
    the share of scored rows whose ratio is clipped; dlogp [n] = grad_scale·dloss/dlogp). Without
    scored rows all are 0. With kl_coef = 0 ref_logp enters the KL statistic alone, also where its term
    is infinite. As the formula has it, an infinite ratio with an advantage of 0 gives NaN."""
    what = "policy_loss"
    if kl not in L.KL_KINDS:
        raise ValueError(f"{what}: kl is one of {', '.join(L.KL_KINDS)}")
    if reduction not in L.REDUCTIONS:
        raise ValueError(f"{what}: reduction is one of {', '.join(L.REDUCTIONS)}")
    _vec(what, "logp", logp, plan.n, torch.float32)
    _vec(what, "old_logp", old_logp, plan.n, torch.float32)
    if ref_logp is not None:
        _vec(what, "ref_logp", ref_logp, plan.n, torch.float32)
    by_row = adv.dim() == 1 and adv.shape[0] == plan.n
    _vec(what, "adv", adv, plan.n if by_row else plan.nseq, torch.float32)
    _mask(what, mask, plan.n)
    with _on(what, logp, old_logp, adv, ref_logp, mask, plan.tables):
        dlogp = torch.empty_like(logp)
        out = torch.empty(4, dtype=torch.float32, device=logp.device)
        work = _work(plan.loss_bytes, logp.device) if plan.loss_bytes else None
        L.check(L.load().dsb_op_policy_loss(
            _at(logp), _at(old_logp), _at(ref_logp), _at(adv), by_row, _at(mask), plan.ref, clip_low,
            clip_high, kl_coef, L.KL_KINDS[kl], L.REDUCTIONS[reduction], divisor, grad_scale,
            _at(out), _at(dlogp), _at(work), plan.loss_bytes, _now()), what="dsb_op_policy_loss")
    return out[0], out[1:], dlogp


class AdamW:
    """AdamW over many tensors in one launch, with gradient clipping by group and moments in 8 or
    32 bits (:func:`clip_adamw_` keeps fp32 moments of the caller's).

    ws, gs: weights and their gradient buffers, fp32 or bf16 each, contiguous, on one device, no
    weight overlapping another or a gradient; they are bound: each step reads the gradients from, and writes the
    weights to, the memory that these tensors had here (which is kept alive). groups:
    non-decreasing group numbers from 0 (default: one group).

    The moments start at zero, in blocks of 256 elements, each tensor from a block of its own.
    :meth:`state` names them: ``m`` and ``v`` fp32 with bits=32; with bits=8 ``m`` and ``r`` in
    float8_e4m3fn with a scale per block, ``m_scale`` and ``r_scale`` fp32: the first moment is
    m·m_scale, the second (r·r_scale)². They may be saved and copied back."""

    def __init__(self, ws, gs, bits=8, groups=None):
        what = "AdamW"
        ws, gs = list(ws), list(gs)
        groups = [0] * len(ws) if groups is None else [int(g) for g in groups]
        if bits not in (8, 32):
            raise ValueError(f"{what}: bits is 8 or 32")
        if not ws or len(gs) != len(ws) or len(groups) != len(ws):
            raise ValueError(f"{what}: takes as many gradients and groups as weights, at least one")
        if groups[0] < 0 or groups[-1] >= 1 << 20 or any(b < a for a, b in zip(groups, groups[1:])):
            raise ValueError(f"{what}: groups must be non-decreasing numbers below 2^20")
        code = {BF16: L.DT_BF16, torch.float32: L.DT_F32}
        for w, g in zip(ws, gs):
            if w.dtype not in code or g.dtype not in code:
                raise ValueError(f"{what}: weights and gradients are fp32 or bf16")
            if w.shape != g.shape or not w.is_contiguous() or not g.is_contiguous():
                raise ValueError(f"{what}: a weight and its gradient are contiguous, of one shape")
        # by address: each weight's end before the next weight and the next gradient begin, and each
        # gradient's before the next weight (gradients may be shared)
        span = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size(), k)
                      for k, xs in enumerate((ws, gs)) for x in xs if x.numel())
        end = [0, 0]
        for a, b, k in span:
            if a < end[0] or (k == 0 and a < end[1]):
                raise ValueError(f"{what}: a weight overlaps another weight or a gradient in memory")
            end[k] = max(end[k], b)
        with _on(what, *ws, *gs):
            self.device, self.bits, self.ngroups = ws[0].device, bits, groups[-1] + 1
            numel = np.array([w.numel() for w in ws], dtype=np.int64)
            blocks = -(-numel // L.ADAM_BLOCK)
            chunks = -(-numel // L.ADAM_CHUNK)
            block0 = np.cumsum(blocks) - blocks
            self.nblocks, self.nchunks = int(blocks.sum()), int(chunks.sum())
            if self.nchunks >= 1 << 24:  # (a launch's blocks)
                raise ValueError(f"{what}: too many elements")
            # a record per chunk: one table to read, no second one behind it
            t = np.repeat(np.arange(len(ws)), chunks)
            at = (np.arange(self.nchunks) - (np.cumsum(chunks) - chunks)[t]) * L.ADAM_CHUNK
            table = np.zeros(self.nchunks, dtype=np.dtype(L.DsbAdamChunk))
            for name, ts in (("w", ws), ("g", gs)):
                base = np.array([x.data_ptr() for x in ts], dtype=np.uint64)
                size = np.array([x.element_size() for x in ts], dtype=np.int64)
                table[name] = base[t] + (at * size[t]).astype(np.uint64)
            table["block"] = block0[t] + at // L.ADAM_BLOCK
            table["count"] = np.minimum(numel[t] - at, L.ADAM_CHUNK)
            table["dtypes"] = np.array([code[w.dtype] + 256 * code[g.dtype] for w, g in zip(ws, gs)])[t]
            per = np.bincount(np.array(groups), weights=chunks, minlength=self.ngroups)
            most = int(per.max())
            ends = np.concatenate([[0], np.cumsum(per)]).astype(np.int32)
            table["group"] = group = np.array(groups)[t]
            table["c0"], table["c1"] = ends[group], ends[group + 1]

            def dev(a):
                raw = np.frombuffer(a.tobytes(), dtype=np.uint8).copy()
                return torch.from_numpy(raw).to(self.device) if raw.size else _work(0, self.device)

            self._chunks, self._ends = dev(table), dev(ends)
            self._kept = [t.untyped_storage() for t in (*ws, *gs)]
            nbytes = c_int64()
            L.check(L.load().dsb_op_adam_workspace(self.nchunks, self.ngroups, byref(nbytes)),
                    what="dsb_op_adam_workspace")
            self._bytes = nbytes.value
            n = self.nblocks * L.ADAM_BLOCK
            zeros = lambda k, dt: torch.zeros(k, dtype=dt, device=self.device)  # noqa: E731
            if bits == 8:
                f8 = torch.float8_e4m3fn
                self._state = {"m": zeros(n, torch.uint8).view(f8),
                               "m_scale": zeros(self.nblocks, torch.float32),
                               "r": zeros(n, torch.uint8).view(f8),
                               "r_scale": zeros(self.nblocks, torch.float32)}
            else:
                self._state = {"m": zeros(n, torch.float32), "v": zeros(n, torch.float32)}
            s = self._state
            self._args = (_at(self._chunks), self.nchunks, _at(self._ends), self.ngroups, most,
                          _at(s["m"]), _at(s["r" if bits == 8 else "v"]), _at(s.get("m_scale")),
                          _at(s.get("r_scale")), bits)

    def state(self):
        """The moments by name (the optimizer's own tensors)."""
        return dict(self._state)

    def step(self, lr, step, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.0, max_norm=None, seed=0):
        """One step, the step-th (from 1), in place on the weights and the moments. max_norm: clip
        each group's gradient to this norm (the gradients stay as they are) and return the norms
        before the clip, fp32 [ngroups]; None: no clip, returns None. 8-bit second moments are
        rounded at random by ``seed`` and step, the same way for the same two. For a step that is
        captured into a graph, lr (fp32) and step (int64) may be one-element tensors on the device,
        read when it runs; numbers are baked in. A NaN or infinite gradient reaches the weights that
        it reaches in the formula, and with 8 bits its block's moments. A finite one of 2^64 or more
        (after the clip) has an infinite square in fp32: with 32 bits its weight stays where it is, with
        8 bits its block's moments are lost."""
        what = "AdamW.step"
        lr_t = lr if isinstance(lr, torch.Tensor) else None
        step_t = step if isinstance(step, torch.Tensor) else None
        for name, t, dt in (("lr", lr_t, torch.float32), ("step", step_t, torch.int64)):
            if t is not None and (t.numel() != 1 or t.dtype != dt):
                raise ValueError(f"{what}: a {name} tensor holds one element of {dt}")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"{what}: max_norm must not be negative")
        with _on(what, self._chunks, lr_t, step_t):
            norms = None
            if max_norm is not None:
                norms = torch.empty(self.ngroups, dtype=torch.float32, device=self.device)
            work = _work(self._bytes, self.device)
            L.check(L.load().dsb_op_adam_step(
                *self._args, 0.0 if lr_t is not None else lr, beta1, beta2, eps, wd,
                -1.0 if max_norm is None else max_norm, 0 if step_t is not None else step,
                seed & 0xffffffff, _at(lr_t), _at(step_t), _at(norms), _at(work), self._bytes, _now()),
                what="dsb_op_adam_step")
        return norms
