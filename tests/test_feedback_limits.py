"""Sizes past what one launch holds (2^32 threads) are refused by the operators for training from
feedback before anything is enqueued, with a message; without a GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from test_feedback_host import BIG, FAKE, _lib, _lp


@pytest.mark.parametrize("n,V,ok", [((1 << 24) - 1, 256, True), (1 << 24, 256, False), (1 << 30, 2, False),
                                    (1 << 20, 1 << 20, False), (1 << 20, (1 << 20) - 256, True)])
def test_rows_of_a_head_product(n, V, ok):
    L, lib = _lib()
    nbytes = ctypes.c_int64(-1)
    for backward in (0, 1):
        rc = lib.dsb_op_logprob_workspace(n, 8, V, backward, ctypes.byref(nbytes))
        assert (rc == 0) == ok and (not ok or nbytes.value > 0)
    if not ok:
        assert _lp(lib, n=n, V=V, D=8, ld=8) != 0 and "2^24" in L.last_error()
        assert lib.dsb_op_token_logprobs_bwd(FAKE, 8, FAKE, FAKE, n, 8, V, FAKE, FAKE, FAKE, FAKE, 8, 0, FAKE,
                                             BIG, None) != 0


@pytest.mark.parametrize("length", [0, 1])
def test_sequences_of_a_plan(length):
    L, lib = _lib()
    lens = np.full((1 << 26) - 11, length, dtype=np.int32)
    p = lens.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
    plan, elems = L.DsbPackPlan(), ctypes.c_int64()
    assert lib.dsb_plan_sizes(p, len(lens), ctypes.byref(plan), ctypes.byref(elems)) != 0
    assert "too many sequences" in L.last_error()
    assert lib.dsb_plan_sizes(p, len(lens) - 1, ctypes.byref(plan), ctypes.byref(elems)) == 0
    # of few sequences the rows' own bound is the first
    lens = np.array([(1 << 31) - 4097 - 5, 5], dtype=np.int32)
    p = lens.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
    assert lib.dsb_plan_sizes(p, 2, ctypes.byref(plan), ctypes.byref(elems)) == 0
    lens[1] = 6
    assert lib.dsb_plan_sizes(p, 2, ctypes.byref(plan), ctypes.byref(elems)) != 0


def test_chunks_of_an_optimizer_step():
    L, lib = _lib()
    nbytes = ctypes.c_int64()
    for n, ok in (((1 << 24) - 1, True), (1 << 24, False)):
        assert (lib.dsb_op_adam_workspace(n, 1, ctypes.byref(nbytes)) == 0) == ok
    assert lib.dsb_op_adam_step(FAKE, 1 << 24, FAKE, 1, 1, FAKE, FAKE, FAKE, FAKE, 8, 1e-3, 0.9, 0.999, 1e-8, 0.0,
                                -1.0, 1, 0, None, None, FAKE, FAKE, BIG, None) != 0
    assert "sizes" in L.last_error()
