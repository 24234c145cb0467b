"""Layer norm over the last axis, forward and backward.

``y = (x - mean) * rstd * weight + bias`` with ``rstd = 1 / sqrt(var + eps)``,
the layer before an (SC) product in a transformer block; the reference leaves
it to its callers' model code. x is float32, bfloat16 or float16, weight and
bias float32 or x's type; statistics, sums and the weight's gradient are
float32 and rounded once.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _layers as L
from .act8 import Act8, _empty


def _check_x(who, x):
    dt = L.dtype_code(who, "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{who}: x needs a last axis, got shape {tuple(x.shape)}")
    return dt


@torch.no_grad()
def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                       eps: float = 1e-5, checkpoint8: bool = False):
    """``(y, mean, rstd)``; with ``checkpoint8`` ``(y, mean, rstd, x8)`` where x8 is
    the 8-bit checkpoint of x, written in the same pass.

    x: (..., D). mean and rstd are float32 of x's leading shape. weight and bias:
    (D,), of one dtype, or None.
    """
    who = "layer_norm_forward"
    dt = _check_x(who, x)
    cols = x.shape[-1]
    weight, bias = L.parameter(who, "weight", weight, x.dtype, cols), L.parameter(who, "bias", bias, x.dtype, cols)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{who}: weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    L.same_place(who, x, weight=weight, bias=bias)
    p = weight if weight is not None else bias
    dev = x.device
    with L.on(dev):
        x2, rows, ld = L.rows_of(x)
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        mean, rstd = torch.empty((2, *x.shape[:-1]), dtype=torch.float32, device=dev).unbind(0)
        x8 = _empty(x.shape, x.dtype, dev) if checkpoint8 else None
        L.call("scmp_layer_norm_forward", x2.data_ptr(), dt, rows, cols, ld, L.ptr(weight), L.ptr(bias),
               dt if p is None else L.DTYPES[p.dtype], eps, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
               x8.codes.data_ptr() if checkpoint8 else None, x8.exponents.data_ptr() if checkpoint8 else None,
               L.stream(dev))
    return (y, mean, rstd, x8) if checkpoint8 else (y, mean, rstd)


@torch.no_grad()
def layer_norm_backward(dy: torch.Tensor, x: Union[torch.Tensor, Act8], mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, *, with_bias: bool = True):
    """``(dx, dweight, dbias)`` of :func:`layer_norm_forward`.

    x: the forward pass's input or its :class:`Act8`. dx has dy's shape and dtype
    (x's); dweight and dbias have weight's dtype. Without a weight dweight is None
    and dbias has x's dtype; ``with_bias=False`` leaves dbias out (None).
    """
    who = "layer_norm_backward"
    packed = isinstance(x, Act8)
    dt = L.dtype_code(who, "dy", dy)
    if tuple(x.shape) != tuple(dy.shape):
        raise ValueError(f"{who}: dy has shape {tuple(dy.shape)}, x {tuple(x.shape)}")
    if dy.dim() < 1 or dy.shape[-1] < 1:
        raise ValueError(f"{who}: dy needs a last axis, got shape {tuple(dy.shape)}")
    if x.dtype != dy.dtype:
        raise ValueError(f"{who}: dy is {dy.dtype}, x {x.dtype}")
    for name, s in (("mean", mean), ("rstd", rstd)):
        if s.dtype != torch.float32 or tuple(s.shape) != tuple(dy.shape[:-1]):
            raise ValueError(f"{who}: {name} must be float32 {tuple(dy.shape[:-1])}, got {s.dtype} {tuple(s.shape)}")
    cols = dy.shape[-1]
    weight = L.parameter(who, "weight", weight, dy.dtype, cols)
    dev = dy.device
    for name, t in (("x", x), ("mean", mean), ("rstd", rstd), ("weight", weight)):
        if t is not None and t.device != dev:
            raise ValueError(f"{who}: {name} is on {t.device}, dy on {dev}")
    with L.on(dev):
        dy2, rows, ldy = L.rows_of(dy)
        x2, _, ldx = (None, 0, 0) if packed else L.rows_of(x)
        mean, rstd = mean.contiguous(), rstd.contiguous()
        wdtype = dy.dtype if weight is None else weight.dtype
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dev)
        dw = torch.empty(cols, dtype=wdtype, device=dev) if weight is not None else None
        db = torch.empty(cols, dtype=wdtype, device=dev) if with_bias else None
        ws = nbytes = None
        if dw is not None or db is not None:
            ws, nbytes, keep = L.workspace(dev, "scmp_layer_norm_backward_workspace_size", rows, cols)
        L.call("scmp_layer_norm_backward", dy2.data_ptr(), ldy, L.ptr(x2), ldx,
               x.codes.data_ptr() if packed else None, x.exponents.data_ptr() if packed else None, dt, rows, cols,
               mean.data_ptr(), rstd.data_ptr(), L.ptr(weight), L.DTYPES[wdtype], dx.data_ptr(), L.ptr(dw), L.ptr(db),
               ws, nbytes or 0, L.stream(dev))
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint):
        out = layer_norm_forward(x, weight, bias, eps=eps, checkpoint8=checkpoint == "8bit")
        y, mean, rstd = out[:3]
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.dtype = x.dtype
        if checkpoint == "8bit":
            ctx.save_for_backward(out[3].codes, out[3].exponents, mean, rstd, weight)
        else:
            ctx.save_for_backward(x, None, mean, rstd, weight)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, exps, mean, rstd, weight = ctx.saved_tensors
        if exps is not None:
            x = Act8(x, exps, ctx.dtype)
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, with_bias=ctx.bias_dtype is not None)
        if db is not None and db.dtype != ctx.bias_dtype:  # a float32 bias without a weight
            db = db.to(ctx.bias_dtype)
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5, checkpoint: str = "exact") -> torch.Tensor:
    """Differentiable layer norm over the last axis. ``checkpoint="8bit"`` keeps x
    for the backward pass in 8 bits instead of holding on to the tensor."""
    if checkpoint not in ("exact", "8bit"):
        raise ValueError(f"layer_norm: unknown checkpoint '{checkpoint}'. Expected 'exact' or '8bit'.")
    return _LayerNorm.apply(x, weight, bias, eps, checkpoint)


__all__ = ["layer_norm", "layer_norm_forward", "layer_norm_backward"]
