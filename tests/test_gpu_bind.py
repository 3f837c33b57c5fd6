"""Binds of activation buffers that are refused: the cycle goes on with the buffers bound before."""

from __future__ import annotations

import ctypes

import pytest
import torch

from harness import O, bf16_round_acts, build_service, gpu_activations, tiny_meta

pytestmark = pytest.mark.gpu

SEQ = [37, 128, 1, 64]
N = sum(SEQ)


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_a_refused_bind_leaves_the_one_before_it(graph, eight):
    from deltaserve_amd import _lib as L, ops

    meta = {**tiny_meta(L=3), "backward_hip_graph": graph}
    model = O.make_model(meta, seed=7, w_std=0.05, b_std=0.02, norm_jitter=0.2)
    ids = torch.randint(0, meta["vocab_size"], (N,), generator=torch.Generator().manual_seed(7))
    acts = gpu_activations(bf16_round_acts(O.forward_capture(model, ids, SEQ)), meta["max_saved_finetuning_tokens"])
    if eight:
        acts["layer_in"] = [ops.pack_rows8(t) for t in acts["layer_in"]]
    other = gpu_activations({"layer_in": [torch.ones(N, 256)] * 3, "final_in": torch.ones(N, 256),
                             "concat_input_ids": ids}, meta["max_saved_finetuning_tokens"])
    a, b = build_service(model), build_service(model)
    try:
        assert a.process_backward(acts, SEQ, N, 0) == b.process_backward(acts, SEQ, N, 0)
        ptrs = (ctypes.c_void_p * 3)(*[t.data_ptr() for t in other["layer_in"]])
        ptrs[1] = None
        bad = L.DsbActivations(layer_in=ctypes.cast(ptrs, ctypes.POINTER(ctypes.c_void_p)), ld=256,
                               final_in=other["final_in"].data_ptr(),
                               input_ids=other["concat_input_ids"].data_ptr())
        assert L.load().dsb_bind_activations(a._h, ctypes.byref(bad)) == -1
        assert "null layer_in" in L.last_error(a._h)
        for epoch in (1, 2):
            assert a.process_backward(acts, SEQ, N, epoch) == b.process_backward(acts, SEQ, N, epoch)
            for i, d in a.lora.items():
                for p, dd in d.items():
                    for ab, t in dd.items():
                        assert torch.equal(t, b.lora[i][p][ab]) and torch.equal(t.grad, b.lora[i][p][ab].grad)
    finally:
        a.close()
        b.close()
