"""8-bit activation checkpoints: what a backward pass needs of an activation, in
1 + 1/32 bytes per value.

Blocks of 32 values along a row share a power of two ``2^e`` with
``e = floor(log2(max |x|)) - 6`` (at least -126; -24 for float16); a value is
kept as ``x * 2^-e`` rounded half to even and clamped to -127..127, and stands
for ``code * 2^e``. Every step but that rounding is exact, and the value a code
stands for is exact in float32, bfloat16 and float16, so a gradient computed
from a checkpoint sees the checkpoint's own values. A block that holds an
infinity or a NaN stands for NaN.

``layer_norm_forward(..., checkpoint8=True)`` and
``linear_forward(..., save="8bit")`` write checkpoints in the pass that has the
values at hand; ``layer_norm_backward`` and ``linear_backward`` take an
:class:`Act8` wherever they take the tensor it stands for. The reference keeps
nothing for a backward pass and has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _layers as L

BLOCK = 32


class Act8:
    """A tensor's 8-bit checkpoint: ``codes`` int8 of the tensor's shape,
    ``exponents`` uint8 ``(..., ceil(cols / 32))`` holding e + 127 (255: the block
    stands for NaN), and the ``dtype`` the tensor had."""

    __slots__ = ("codes", "exponents", "dtype")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype = torch.float32):
        if codes.dtype != torch.int8 or exponents.dtype != torch.uint8:
            raise ValueError(f"Act8: codes must be int8 and exponents uint8, got {codes.dtype} and {exponents.dtype}")
        if dtype not in L.DTYPES:
            raise ValueError(f"Act8: dtype must be float32, bfloat16 or float16, got {dtype}")
        if codes.dim() < 1 or codes.shape[-1] < 1:
            raise ValueError(f"Act8: codes need a last axis, got shape {tuple(codes.shape)}")
        want = (*codes.shape[:-1], -(-codes.shape[-1] // BLOCK))
        if tuple(exponents.shape) != want:
            raise ValueError(f"Act8: exponents must be {want}, got {tuple(exponents.shape)}")
        if codes.device != exponents.device:
            raise ValueError("Act8: codes and exponents must be on the same device")
        if not codes.is_contiguous() or not exponents.is_contiguous():
            raise ValueError("Act8: codes and exponents must be contiguous")
        self.codes, self.exponents, self.dtype = codes, exponents, dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    def __repr__(self):
        return f"Act8({tuple(self.shape)}, {self.dtype}, {self.device})"


def _wrap(codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype) -> Act8:
    """An Act8 of tensors the library just wrote."""
    a = object.__new__(Act8)
    a.codes, a.exponents, a.dtype = codes, exponents, dtype
    return a


def pack_act8(x: torch.Tensor) -> Act8:
    """The 8-bit checkpoint of ``x`` (..., cols), a float32, bfloat16 or float16
    CUDA tensor."""
    return _wrap(*L.ext().act8_pack(x), x.dtype)


def unpack_act8(a: Act8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values ``a`` stands for, as ``dtype`` (default: the packed tensor's).
    Exact, but that another dtype than the packed tensor's may round or overflow."""
    return L.ext().act8_unpack(a.codes, a.exponents, a.dtype if dtype is None else dtype)


__all__ = ["Act8", "pack_act8", "unpack_act8"]
