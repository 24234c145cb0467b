"""The exact linear layer, forward and backward.

``y = act(x @ weight.T + bias) + residual`` with the operands' layout of
``sc_matmul`` (x (..., D) as a, weight (M, D) as b): the layers that a
mixed-precision model keeps exact, and the product whose gradient an SC layer
trains with (a straight-through estimate: ``sc_matmul`` forward,
:func:`linear_backward` backward). The reference leaves both to its callers.

x, weight and residual share one dtype (float32, bfloat16 or float16); the bias
may also be float32. Sums and epilogues are float32, rounded once; float32
products keep float32 accuracy.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _layers as L
from . import _lib
from .act8 import Act8, _empty


def _activation(who: str, activation) -> int:
    code = _lib.ACTIVATIONS.get(activation)
    if code is None:
        names = ", ".join(repr(k) for k in _lib.ACTIVATIONS)
        raise ValueError(f"{who}: unknown activation '{activation}'. Expected one of {names}.")
    return code


def _weight(who: str, weight: torch.Tensor, dtype: torch.dtype, d: Optional[int], m: Optional[int]):
    if weight.dim() != 2:
        raise ValueError(f"{who}: weight must be 2D (M, D), got {weight.dim()}D")
    if weight.dtype != dtype:
        raise ValueError(f"{who}: weight is {weight.dtype}, expected {dtype}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{who}: weight has no values: {tuple(weight.shape)}")
    if (d is not None and weight.shape[1] != d) or (m is not None and weight.shape[0] != m):
        raise ValueError(f"{who}: inner dimension mismatch: weight is {tuple(weight.shape)}, "
                         f"expected ({'M' if m is None else m}, {'D' if d is None else d})")


@torch.no_grad()
def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                   activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                   save: Optional[str] = None):
    """``act(x @ weight.T + bias) + residual`` in one pass over the product.

    activation: None, "relu", "gelu" (erf), "gelu_tanh" or "silu". save: "exact"
    also returns the pre-activation ``x @ weight.T + bias`` (x's dtype), "8bit" its
    :class:`Act8`, written by the same pass: ``(y, pre)`` instead of ``y``.
    """
    who = "linear_forward"
    dt = L.dtype_code(who, "x", x)
    act = _activation(who, activation)
    if save not in (None, "exact", "8bit"):
        raise ValueError(f"{who}: unknown save '{save}'. Expected None, 'exact' or '8bit'.")
    if x.dim() < 1:
        raise ValueError(f"{who}: x needs a last axis")
    d = x.shape[-1]
    _weight(who, weight, x.dtype, d, None)
    m = weight.shape[0]
    shape = (*x.shape[:-1], m)
    bias = L.parameter(who, "bias", bias, x.dtype, m)
    if residual is not None and (residual.dtype != x.dtype or tuple(residual.shape) != shape):
        raise ValueError(f"{who}: residual must be {x.dtype} {shape}, got {residual.dtype} {tuple(residual.shape)}")
    L.same_place(who, x, weight=weight, bias=bias, residual=residual)
    dev = x.device
    with L.on(dev):
        x2, rows, ldx = L.rows_of(x)
        w2, _, ldw = L.rows_of(weight)
        r2, _, ldr = (None, 0, 0) if residual is None else L.rows_of(residual)
        y = torch.empty(shape, dtype=x.dtype, device=dev)
        pre = torch.empty(shape, dtype=x.dtype, device=dev) if save == "exact" else \
            _empty(shape, x.dtype, dev) if save == "8bit" else None
        ws, nbytes, keep = L.workspace(dev, "scmp_linear_forward_workspace_size", dt, rows, d, m,
                                       L.unaligned(1, x2, ldx) | L.unaligned(2, w2, ldw))
        L.call("scmp_linear_forward", x2.data_ptr(), ldx, w2.data_ptr(), ldw, L.ptr(bias),
               dt if bias is None else L.DTYPES[bias.dtype], L.ptr(r2), ldr, dt, rows, d, m, act, y.data_ptr(),
               pre.data_ptr() if save == "exact" else None, pre.codes.data_ptr() if save == "8bit" else None,
               pre.exponents.data_ptr() if save == "8bit" else None, ws, nbytes, L.stream(dev))
    return y if save is None else (y, pre)


@torch.no_grad()
def linear_backward(dy: torch.Tensor, x: Union[torch.Tensor, Act8, None], weight: Optional[torch.Tensor], *,
                    activation: Optional[str] = None, pre: Union[torch.Tensor, Act8, None] = None,
                    with_bias: bool = True, bias_dtype: Optional[torch.dtype] = None, need_dx: bool = True,
                    need_dweight: bool = True):
    """``(dx, dweight, dbias)`` of :func:`linear_forward`; the residual's gradient is
    dy itself.

    x and pre (the pre-activation, needed with an activation) are tensors or
    their :class:`Act8`. x may be None with ``need_dweight=False``, weight with
    ``need_dx=False``; what is not asked for is None. dbias has ``bias_dtype``
    (default: dy's; or float32). The gradient of the pre-activation that the two
    products share is rounded to dy's dtype once; dbias is summed before that
    rounding.
    """
    who = "linear_backward"
    dt = L.dtype_code(who, "dy", dy)
    act = _activation(who, activation)
    if dy.dim() < 1 or dy.shape[-1] < 1:
        raise ValueError(f"{who}: dy needs a last axis, got shape {tuple(dy.shape)}")
    m, lead, dev = dy.shape[-1], tuple(dy.shape[:-1]), dy.device
    bias_dtype = dy.dtype if bias_dtype is None else bias_dtype
    if bias_dtype != dy.dtype and bias_dtype != torch.float32:
        raise ValueError(f"{who}: bias_dtype must be float32 or {dy.dtype}, got {bias_dtype}")
    if need_dx and weight is None:
        raise ValueError(f"{who}: dx needs the weight")
    if need_dweight and x is None:
        raise ValueError(f"{who}: dweight needs x")
    d = None
    if x is not None:
        if x.dtype != dy.dtype:
            raise ValueError(f"{who}: dy is {dy.dtype}, x {x.dtype}")
        if tuple(x.shape[:-1]) != lead or x.shape[-1] < 1:
            raise ValueError(f"{who}: dy has shape {tuple(dy.shape)}, x {tuple(x.shape)}")
        d = x.shape[-1]
    if weight is not None:
        _weight(who, weight, dy.dtype, d, m)
        d = weight.shape[1]
    if act:
        if pre is None:
            raise ValueError(f"{who}: activation '{activation}' needs pre, the pre-activation")
        if pre.dtype != dy.dtype or tuple(pre.shape) != tuple(dy.shape):
            raise ValueError(f"{who}: pre must be {dy.dtype} {tuple(dy.shape)}, got {pre.dtype} {tuple(pre.shape)}")
    else:
        pre = None
    for name, t in (("x", x), ("weight", weight), ("pre", pre)):
        if t is not None and t.device != dev:
            raise ValueError(f"{who}: {name} is on {t.device}, dy on {dev}")
    x8 = x if isinstance(x, Act8) and need_dweight else None
    p8 = pre if isinstance(pre, Act8) else None
    with L.on(dev):
        dy2, rows, ldy = L.rows_of(dy)
        x2, _, ldx = L.rows_of(x) if need_dweight and x8 is None else (None, 0, 0)
        w2, _, ldw = L.rows_of(weight) if need_dx else (None, 0, 0)
        p2, _, ldp = L.rows_of(pre) if pre is not None and p8 is None else (None, 0, 0)
        dx = torch.empty((*lead, d), dtype=dy.dtype, device=dev) if need_dx else None
        dw = torch.empty((m, d), dtype=dy.dtype, device=dev) if need_dweight else None
        db = torch.empty(m, dtype=bias_dtype, device=dev) if with_bias else None
        parts = int(need_dx) | 2 * int(need_dweight) | 4 * int(with_bias)
        if not parts:
            return None, None, None
        d = 1 if d is None else d
        ws, nbytes, keep = L.workspace(dev, "scmp_linear_backward_workspace_size", dt, rows, d, m, act,
                                       int(x8 is not None), parts,
                                       L.unaligned(4, dy2, ldy) | L.unaligned(1, x2, ldx) | L.unaligned(2, w2, ldw))
        L.call("scmp_linear_backward", dy2.data_ptr(), ldy, L.ptr(x2), ldx, x8.codes.data_ptr() if x8 is not None else None,
               x8.exponents.data_ptr() if x8 is not None else None, L.ptr(w2), ldw, L.ptr(p2), ldp,
               p8.codes.data_ptr() if p8 is not None else None, p8.exponents.data_ptr() if p8 is not None else None, dt,
               rows, d, m, act, L.ptr(dx), L.ptr(dw), L.ptr(db), L.DTYPES[bias_dtype], ws, nbytes, L.stream(dev))
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, checkpoint):
        eight = checkpoint == "8bit"
        need_w = ctx.needs_input_grad[1]
        need_pre = activation is not None and any(ctx.needs_input_grad[:3])
        out = linear_forward(x, weight, bias, activation=activation, residual=residual,
                             save=("8bit" if eight else "exact") if need_pre else None)
        y, pre = out if need_pre else (out, None)
        kept = []
        if not need_w:
            kept += [None, None]
        elif eight:
            from .act8 import pack_act8
            x8 = pack_act8(x)
            kept += [x8.codes, x8.exponents]
        else:
            kept += [x, None]
        if pre is None:
            kept += [None, None]
        elif eight:
            kept += [pre.codes, pre.exponents]
        else:
            kept += [pre, None]
        ctx.save_for_backward(weight, *kept)
        ctx.activation, ctx.dtype = activation, x.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        weight, x, xe, pre, pe = ctx.saved_tensors
        x = Act8(x, xe, ctx.dtype) if xe is not None else x
        pre = Act8(pre, pe, ctx.dtype) if pe is not None else pre
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            dx, dw, db = linear_backward(dy, x, weight, activation=ctx.activation, pre=pre, with_bias=need_b,
                                         bias_dtype=ctx.bias_dtype, need_dx=need_x, need_dweight=need_w)
        return dx, dw, db, dy if need_r else None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           checkpoint: str = "exact") -> torch.Tensor:
    """Differentiable ``act(x @ weight.T + bias) + residual``. ``checkpoint="8bit"``
    keeps x and the pre-activation for the backward pass in 8 bits."""
    if checkpoint not in ("exact", "8bit"):
        raise ValueError(f"linear: unknown checkpoint '{checkpoint}'. Expected 'exact' or '8bit'.")
    return _Linear.apply(x, weight, bias, residual, activation, checkpoint)


__all__ = ["linear", "linear_forward", "linear_backward"]
