"""Binding of activation buffers on the host: libdsb.so against a HIP runtime of a few functions whose
allocations can be made to fail, and the trainer's checks of the buffers that it is given."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

from harness import ROOT

HIP = r"""
#include <stdlib.h>
/* bytes that are held, and the allocation of these to come that fails, with all after it (0: none) */
long held_bytes = 0, fail_at = 0;
static struct { void* p; size_t n; } blocks[4096];
static int nblocks = 0;
int hipMalloc(void** p, size_t n) {
  if (fail_at == 1) return 2;
  if (fail_at) --fail_at;
  *p = aligned_alloc(256, 256);
  blocks[nblocks].p = *p;
  blocks[nblocks++].n = n;
  held_bytes += (long)n;
  return 0;
}
int hipFree(void* p) {
  for (int i = 0; i < nblocks; ++i)
    if (blocks[i].p == p) {
      held_bytes -= (long)blocks[i].n;
      blocks[i] = blocks[--nblocks];
      free(p);
      break;
    }
  return 0;
}
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipGetLastError(void) { return 0; }
const char* hipGetErrorString(int e) { return e == 2 ? "out of memory" : "?"; }
int hipStreamCreateWithFlags(void** s, unsigned f) { *s = (void*)1; return 0; }
int hipStreamSynchronize(void* s) { return 0; }
int hipStreamDestroy(void* s) { return 0; }
int hipEventCreateWithFlags(void** e, unsigned f) { *e = (void*)1; return 0; }
int hipEventCreate(void** e) { *e = (void*)1; return 0; }
int hipEventDestroy(void* e) { return 0; }
"""

MAIN = r"""
import ctypes, sys

hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # before libdsb.so, whose calls go to it
sys.path.insert(0, sys.argv[2])
from deltaserve_amd import _lib as L

lib = L.load()
held, fail_at = (ctypes.c_long.in_dll(hip, n) for n in ("held_bytes", "fail_at"))
S, D, LAYERS = 500, 64, 3


def handle(flags):
    d = L.DsbDesc(abi_version=L.ABI_VERSION, family=0, n_layers=LAYERS, hidden=D, n_heads=2, n_kv_heads=1,
                  head_dim=64, intermediate=128, vocab=100, lora_rank=8, s_max=S, max_seqs=4, flags=flags)
    h = ctypes.c_void_p()
    assert lib.dsb_create(ctypes.byref(d), ctypes.byref(h)) == 0, L.last_error()
    return h


A = 1 << 20  # an address; nothing reads it here
a = L.DsbActivations(final_in=A, input_ids=A, ld=D)
rows = (L.DsbRows8 * LAYERS)(*[L.DsbRows8(A, A, D, D // 32, L.DT_E4M3)] * LAYERS)
bind = lambda h: lib.dsb_bind_activations8(h, ctypes.byref(a), rows, None)  # noqa: E731
set_bytes = 2 * S * D  # a recompute set's restored rows, bf16
for flags, sets in ((0, 2), (L.FLAG_SERIAL_LAYERS, 1)):
    for nth in (1, 2):
        h, before = handle(flags), held.value
        fail_at.value = nth
        if bind(h) != 0:
            assert "hipMalloc" in L.last_error(), L.last_error()
            once = held.value
            for _ in range(3):  # as a cycle after a cycle that keeps failing
                fail_at.value = nth
                assert bind(h) != 0
                assert held.value == once, "a failed bind keeps more memory every time"
        fail_at.value = 0
        assert bind(h) == 0, L.last_error()
        got = held.value - before
        assert got >= sets * set_bytes, f"{sets} sets of rows need {sets * set_bytes} bytes, {got} are held"
        assert bind(h) == 0 and held.value - before == got
        lib.dsb_destroy(h)
        assert held.value == before
print("ok")
"""


def test_restored_rows_of_overlapped_layers_are_two_buffers_after_a_failed_allocation(tmp_path):
    """A layer's recompute restores its input while the layer after still reads its own: each of the two
    has a buffer, also where an earlier bind ran out of memory."""
    (tmp_path / "hip.c").write_text(HIP)
    (tmp_path / "main.py").write_text(MAIN)
    subprocess.run(["gcc", "-shared", "-fPIC", str(tmp_path / "hip.c"), "-o", str(tmp_path / "hip.so")], check=True)
    r = subprocess.run([sys.executable, str(tmp_path / "main.py"), str(tmp_path / "hip.so"),
                        os.path.join(ROOT, "deltaserve-vllm_amd")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


# ---------------------------------------------------------------- the trainer's checks

def _trainer():
    from types import SimpleNamespace

    from deltaserve_amd.bwd_services.common.trainer import LoraSftTrainerService

    svc = LoraSftTrainerService.__new__(LoraSftTrainerService)
    svc.L, svc.D, svc.inter, svc.q_size, svc.kv_size, svc._s_max = 2, 64, 96, 64, 32, 4
    svc.shared = {"meta": {"save_attn_qkv": True, "save_resid_mid": True}}
    svc.family = SimpleNamespace(supports_saved_qkv=True)
    return svc


@pytest.mark.parametrize("name,width", [("final_in", 64), ("concat_input_ids", 64), ("attn_ctx", 64), ("attn_qh", 64),
                                        ("attn_kh", 32), ("attn_vh", 32), ("resid_mid", 64)])
def test_8_bit_rows_where_the_cycle_takes_bf16_are_a_type_error(name, width, monkeypatch):
    from deltaserve_amd.rows8 import Rows8

    # (the checks ask of a tensor only whether it is on the device)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))

    def rows(w):
        return torch.zeros(5, w, dtype=torch.bfloat16)

    acts = {"layer_in": [rows(64)] * 2, "final_in": rows(64), "concat_input_ids": torch.zeros(4, dtype=torch.int64),
            "attn_ctx": [rows(64)] * 2, "attn_qh": [rows(64)] * 2, "attn_kh": [rows(32)] * 2,
            "attn_vh": [rows(32)] * 2, "resid_mid": [rows(64)] * 2}
    small = Rows8.zeros(5, width, device="cpu")
    for bad in ([small, small], [rows(width), small], [small, rows(width)]):
        acts[name] = bad if isinstance(acts[name], list) else small
        with pytest.raises(TypeError):
            _trainer()._bind_activations(acts)
