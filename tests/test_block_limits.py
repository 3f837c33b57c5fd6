"""Calls of a decoder block's memory-bound operators that are refused before any device call, beyond those of
test_block_host.py."""

from __future__ import annotations

import pytest

A = 1 << 20  # an address, aligned


def _lib():
    from deltaserve_amd import _lib as L

    return L, L.load()


def _rotary(n, heads, hd, ldy, hy, place):
    """dsb_op_rotary's answer to a y of these strides."""
    L, lib = _lib()
    x = (A, ldy, hy) if place else (A, heads * hd, hd)
    r = lib.dsb_op_rotary(*x, A if place else 1 << 40, ldy, hy, 0, A, 0, A, 1.0, n, heads, hd, hd, 0, 0, None)
    return r, L.last_error()


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("n,heads,ldy,hy", [
    (2, 2, 64, 64),            # row t, head h + 1 is row t + 1, head h
    (5, 4, 64, 64), (5, 4, 128, 64), (5, 4, 255, 64),  # rows that begin inside the row before
    (5, 4, 64, 319 - 64), (5, 4, 64, 128),             # heads first: a head's rows run into the next head
    (3, 2, 1 << 62, 63), (2, 3, 63, 1 << 62),
    (1 << 20, 2, 64, (1 << 26) - 1),
])
def test_rotary_outputs_that_overlap_themselves_are_refused(n, heads, ldy, hy, place):
    r, err = _rotary(n, heads, 64, ldy, hy, place)
    assert r == -1 and "overlap" in err, err
