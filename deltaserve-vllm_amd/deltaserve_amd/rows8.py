"""Rows of activations in 8 bits.

``Rows8`` holds codes (e4m3 or int8) and a byte per 32 columns of a row, the exponent of their scale
+ 127: a value is code·2^(byte − 127); byte 0 makes 0, byte 255 (codes 0: a lost block) NaN.
``capture.save_rows`` fills one from the serving step's rows, ``ops.pack_rows8`` from a matrix;
``ops.rmsnorm``, ``rmsnorm_backward``, ``swiglu``, ``swiglu_backward`` and ``residual_norm_backward``
read it in place of bf16 rows, ``ops.unpack_rows8`` gives bf16 or fp32 ones. The reference keeps activations in bf16 and has no counterpart.

Which code: int8 is off by at most 1/254 to 1/127 of its block's largest magnitude, whatever the value;
e4m3 by 2^-4 of the value itself down to 2^-14 of the largest. The values of a Gaussian block come back
0.8 % off (root mean square) in int8 and 2.7 % in e4m3; beside a value a hundred times as large, 29 %
and 2.7 %."""

from __future__ import annotations

import torch

from . import _lib as L

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_TYPE = {torch.float8_e4m3fn: L.DT_E4M3, torch.int8: L.DT_INT8}


class Rows8:
    """codes [rows, width] (``torch.float8_e4m3fn`` or ``torch.int8``) and scales uint8 [rows,
    ceil(width / 32)], on one device, each row contiguous. Slices of rows share their memory."""

    __slots__ = ("codes", "scales", "type", "ld", "ld_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype not in _TYPE or codes.dim() != 2:
            raise ValueError("Rows8: codes must be a matrix of float8_e4m3fn or int8")
        n, w = codes.shape
        if scales.dtype != torch.uint8 or scales.shape != (n, -(-w // L.ROWS8_BLOCK)):
            raise ValueError("Rows8: scales must be uint8, one for every 32 columns of a row")
        if codes.device != scales.device:
            raise ValueError("Rows8: codes and scales are on different devices")
        for t in (codes, scales):
            if t.numel() and t.shape[1] > 1 and t.stride(1) != 1:
                raise ValueError("Rows8: rows must be contiguous")
        self.codes, self.scales, self.type = codes, scales, _TYPE[codes.dtype]
        # (the row stride of a single row is any number)
        self.ld = codes.stride(0) if n > 1 else -(-w // 8) * 8
        self.ld_scales = scales.stride(0) if n > 1 else scales.shape[1]

    @classmethod
    def zeros(cls, rows: int, width: int, code: str = "e4m3", device="cuda") -> "Rows8":
        """Rows of zeros. Their codes lie a multiple of 16 bytes apart, so that every op takes them
        (widths of a multiple of 8)."""
        if code not in CODES:
            raise ValueError(f"Rows8: code is one of {', '.join(CODES)}")
        codes = torch.zeros(rows, -(-width // 16) * 16, dtype=torch.uint8, device=device)[:, :width]
        scales = torch.ones(rows, -(-width // L.ROWS8_BLOCK), dtype=torch.uint8, device=device)
        return cls(codes.view(CODES[code]), scales)

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def code(self) -> str:
        return "e4m3" if self.type == L.DT_E4M3 else "int8"

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    def data_ptr(self) -> int:
        return self.codes.data_ptr()

    def __len__(self) -> int:
        return self.codes.shape[0]

    def __getitem__(self, rows: slice) -> "Rows8":
        if not isinstance(rows, slice):
            raise TypeError("Rows8: takes slices of rows")
        return Rows8(self.codes[rows], self.scales[rows])

    def zero_(self) -> "Rows8":
        self.codes.view(torch.uint8).zero_()
        self.scales.fill_(1)
        return self

    def __repr__(self) -> str:
        return f"Rows8({len(self)} x {self.shape[1]}, {self.code}, {self.device})"
