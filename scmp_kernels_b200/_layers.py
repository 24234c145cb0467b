"""What the layers' Python functions share: argument checks, row views, the
device guard and the call into the library."""
from __future__ import annotations

import contextlib
import functools

import torch

from . import _lib

DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_NO_GUARD = contextlib.nullcontext()


def need_cuda(who: str, name: str, t: torch.Tensor) -> None:
    if t.device.type != "cuda":
        _lib.require_cuda()
        raise ValueError(f"{who}: {name} must be a CUDA tensor, got one on {t.device}")


def dtype_code(who: str, name: str, t: torch.Tensor) -> int:
    """The library's number of ``t``'s dtype; ``t`` is a CUDA tensor."""
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{who}: {name} must be float32, bfloat16 or float16, got {t.dtype}")
    need_cuda(who, name, t)
    return code


def same_place(who: str, x: torch.Tensor, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{who}: {name} is on {t.device}, x on {x.device}")


def parameter(who: str, name: str, p, x_dtype: torch.dtype, n: int):
    """A vector of ``n`` values, float32 or of x's type, contiguous (None stays None)."""
    if p is None:
        return None
    if p.dim() != 1 or p.shape[0] != n:
        raise ValueError(f"{who}: {name} must be ({n},), got {tuple(p.shape)}")
    if p.dtype != x_dtype and p.dtype != torch.float32:
        raise ValueError(f"{who}: {name} must be float32 or {x_dtype}, got {p.dtype}")
    return p if p.is_contiguous() else p.contiguous()


def rows_of(t: torch.Tensor):
    """(tensor, rows, pitch): ``t`` (..., cols) as rows at a fixed pitch, without a
    copy where its strides allow it."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // cols, cols
    # a 2D view with neighbouring columns and rows that do not overlap
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= cols:
        return t, t.shape[0], t.stride(0)
    if t.dim() > 2 and t.stride(-1) == 1 and t.stride(-2) >= cols and all(
            t.stride(i) == t.stride(i + 1) * t.shape[i + 1] for i in range(t.dim() - 2)):
        return t, t.numel() // cols, t.stride(-2)
    t = t.contiguous()
    return t, t.numel() // cols, cols


def on(device: torch.device):
    """Makes ``device`` current for a call; free when it already is."""
    return _NO_GUARD if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    return getattr(_lib.lib(), name)


def call(name: str, *args) -> None:
    status = _entry(name)(*args)
    if status:
        _lib.check(status, name[5:])


@functools.lru_cache(maxsize=4096)
def workspace_bytes(name: str, *sizes: int) -> int:
    """Answer of a host-only ``*_workspace_size`` entry point: a function of sizes
    and types alone."""
    n = _lib.c_size_t()
    _lib.check(getattr(_lib.lib(), name)(*sizes, _lib.ctypes.byref(n)), name)
    return n.value


def workspace(device: torch.device, name: str, *sizes: int):
    """(pointer, bytes, owner): scratch for one call, from the caching allocator on
    the current stream."""
    n = workspace_bytes(name, *sizes)
    if n == 0:
        return None, 0, None
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws.data_ptr(), n, ws


def unaligned(flag: int, t, pitch: int) -> int:
    """``flag`` when the library has to copy ``t``'s rows before it can multiply
    them (they do not start and step by 16 bytes), else 0."""
    return flag if t is not None and (t.data_ptr() | pitch * t.element_size()) & 15 else 0


def ptr(t):
    return None if t is None else t.data_ptr()
