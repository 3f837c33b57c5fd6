"""The backward cycle on an activation store that keeps layer inputs and gate‖up in 8 bits: it is the
cycle on a bf16 store that holds the same values, bit for bit (a value in 8 bits is exact in bf16),
however the cycle is run, and the store is filled by the save op."""

from __future__ import annotations

import pytest
import torch

from harness import O, bf16_round_acts, build_service, gpu_activations, tiny_meta

pytestmark = pytest.mark.gpu

SEQ = [37, 128, 1, 200, 64]
N = sum(SEQ)


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _setup(family="llama3", gate_up=True, L=3, **meta):
    meta = {**tiny_meta(family=family, L=L), **meta}
    model = O.make_model(meta, seed=6, w_std=0.05, b_std=0.02, norm_jitter=0.2)
    ids = torch.randint(0, meta["vocab_size"], (N,), generator=torch.Generator().manual_seed(6))
    acts = bf16_round_acts(O.forward_capture(model, ids, SEQ, save_gate_up=gate_up))
    return meta, model, gpu_activations(acts, meta["max_saved_finetuning_tokens"])


def _both(acts, code, points):
    """(the store with these points in 8 bits, a bf16 store of its values)."""
    from deltaserve_amd import ops

    small, plain = dict(acts), dict(acts)
    for name in points:
        small[name] = [ops.pack_rows8(t, code=code) for t in acts[name]]
        plain[name] = [ops.unpack_rows8(q) for q in small[name]]
    return small, plain


def _state(svc):
    return {(i, p, ab): (t.detach().clone(), t.grad.detach().clone())
            for i, d in svc.lora.items() for p, dd in d.items() for ab, t in dd.items()}


def _same(a, b, what):
    sa, sb = _state(a), _state(b)
    assert sa.keys() == sb.keys()
    for k in sa:
        for x, y in zip(sa[k], sb[k]):
            assert torch.equal(x, y), (what, k)


@pytest.mark.parametrize("family", ["llama3", "qwen3"])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("points", [("layer_in",), ("mlp_gate_up",), ("layer_in", "mlp_gate_up")])
def test_cycle_on_8_bits_equals_the_cycle_on_their_values(family, code, points):
    _, model, acts = _setup(family)
    small, plain = _both(acts, code, points)
    a, b = build_service(model, family), build_service(model, family)
    try:
        for epoch in range(3):  # the captured graph, replayed
            assert a.process_backward(small, SEQ, N, epoch) == b.process_backward(plain, SEQ, N, epoch)
            _same(a, b, epoch)
        # and on fewer rows, then on the bf16 store (rebound), then back
        assert a.process_backward(small, SEQ[:2], 165, 3) == b.process_backward(plain, SEQ[:2], 165, 3)
        assert a.process_backward(plain, SEQ, N, 4) == b.process_backward(small, SEQ, N, 4)
        assert a.process_backward(small, SEQ, N, 5) == b.process_backward(plain, SEQ, N, 5)
        _same(a, b, "rebound")
    finally:
        a.close()
        b.close()


def test_the_same_memory_with_another_code():
    """Buffers that come back at the same addresses with another code or stride are bound again."""
    from deltaserve_amd import ops

    _, model, acts = _setup()
    rows, D = acts["layer_in"][0].shape
    codes = [torch.zeros(rows, D + 32, dtype=torch.uint8, device="cuda") for _ in range(3)]
    scales = [torch.zeros(rows, D // 32 + 1, dtype=torch.uint8, device="cuda") for _ in range(3)]
    a, b = build_service(model, "llama3"), build_service(model, "llama3")
    try:
        for epoch, (code, ld, lds) in enumerate([("e4m3", D, D // 32), ("int8", D, D // 32), ("int8", D + 32, D // 32),
                                                 ("int8", D + 32, D // 32 + 1), ("e4m3", D + 32, D // 32 + 1)]):
            kind = torch.float8_e4m3fn if code == "e4m3" else torch.int8
            small, plain = dict(acts), dict(acts)
            small["layer_in"] = [
                ops.pack_rows8(t, out=ops.Rows8(c.flatten()[:rows * ld].view(rows, ld)[:, :D].view(kind),
                                                s.flatten()[:rows * lds].view(rows, lds)[:, :D // 32]))
                for t, c, s in zip(acts["layer_in"], codes, scales)]
            plain["layer_in"] = [ops.unpack_rows8(q) for q in small["layer_in"]]
            assert a.process_backward(small, SEQ, N, epoch) == b.process_backward(plain, SEQ, N, epoch)
            _same(a, b, (code, ld, lds))
    finally:
        a.close()
        b.close()


@pytest.mark.parametrize("meta", [dict(backward_serial_layers=True), dict(backward_hip_graph=False),
                                  dict(backward_pause_boundaries=True, backward_run_ahead_boundaries=1)])
def test_cycle_orders_agree_on_8_bits(meta):
    _, model, acts = _setup()
    _, other, _ = _setup(**meta)
    small, _ = _both(acts, "e4m3", ("layer_in", "mlp_gate_up"))
    a, b = build_service(model, "llama3"), build_service(other, "llama3")
    try:
        for epoch in range(2):
            assert a.process_backward(small, SEQ, N, epoch) == b.process_backward(small, SEQ, N, epoch)
            _same(a, b, epoch)
    finally:
        a.close()
        b.close()


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_a_store_in_8_bits_filled_by_the_save_op(code):
    from deltaserve_amd import capture as C, ops

    meta, model, acts = _setup()
    S, D, inter = meta["max_saved_finetuning_tokens"], meta["hidden_size"], meta["intermediate_size"]
    store = C.ActivationStore(3, D, S, intermediate_size=inter, code=code)
    half = 200
    for lo, hi in ((0, half), (half, N)):  # two steps
        st = store.arm_op_step(list(range(hi - lo)), hi - lo, lo)
        with C.active_state(st):
            for i in range(3):
                C.dserve_save_rows(acts["layer_in"][i][lo:hi].contiguous(), None, store.marker, store.slot(i))
                C.dserve_save_rows(acts["mlp_gate_up"][i][lo:hi].contiguous(), None, store.marker,
                                   store.slot(i, C.SLOT_GATE_UP))
            C.dserve_save_rows(acts["final_in"][lo:hi].contiguous(), None, store.marker, store.final_slot)
        store.save_final_ids(acts["concat_input_ids"][lo:hi].contiguous(), st)
    small, _ = _both(acts, code, ("layer_in", "mlp_gate_up"))
    for name in ("layer_in", "mlp_gate_up"):
        for got, want in zip(store.activations()[name], small[name]):
            assert torch.equal(got.scales[:N], want.scales[:N])
            assert torch.equal(got.codes.view(torch.uint8)[:N], want.codes.view(torch.uint8)[:N])
            assert (ops.unpack_rows8(got[N:]) == 0).all()
    one, two = build_service(model, "llama3"), build_service(model, "llama3")
    try:
        assert one.process_backward(store.activations(), SEQ, N, 0) == two.process_backward(small, SEQ, N, 0)
        _same(one, two, "store")
    finally:
        one.close()
        two.close()
    store.zero_offset_range(half, N)
    assert (ops.unpack_rows8(store.layer_in[0])[half:] == 0).all()
    assert (ops.unpack_rows8(store.layer_in[0])[:half] != 0).any()


def test_stores_that_do_not_fit_are_refused():
    from deltaserve_amd import ops

    meta, model, acts = _setup()
    svc = build_service(model, "llama3")
    small, plain = _both(acts, "e4m3", ("layer_in", "mlp_gate_up"))
    try:
        mixed = dict(small, layer_in=[*small["layer_in"][:2], plain["layer_in"][2]])
        narrow = dict(small, layer_in=[ops.pack_rows8(t[:, :128]) for t in plain["layer_in"]])
        for bad, err in ((mixed, TypeError), (narrow, TypeError),
                         (dict(small, mlp_gate_up=[q[:N] for q in small["mlp_gate_up"]]), ValueError)):
            with pytest.raises(err):
                svc.process_backward(bad, SEQ, N, 0)
        svc.process_backward(small, SEQ, N, 0)
    finally:
        svc.close()
