"""Fine-tune a transformer MLP block whose second product runs on stochastic computing.

    python examples/finetune_mlp.py [--steps 40] [--rows 788] [--width 768] [--hidden 1536]

The block is ``x + W2 gelu(W1 norm(x) + b1) + b2``. W1 stays exact (``linear``
with bias and GELU in its epilogue), W2 is an SC layer: ``sc_matmul`` forward
and, as a straight-through estimate, the exact product's gradient backward
(``linear_backward``). Everything the backward pass needs of the activations is
kept in 8 bits: the block input by ``layer_norm``, the input and
pre-activation of W1 by ``linear``, the input of W2 by ``pack_act8``. A teacher
block in exact arithmetic supplies the targets, and the student starts from
the teacher's weights plus noise, so the loss shows the SC layer being tuned.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import scmp_kernels_b200 as S  # noqa: E402


class SCLinear(torch.autograd.Function):
    """``sc_matmul(x, weight)`` with the gradient of ``x @ weight.T``."""

    @staticmethod
    def forward(ctx, x, weight, sc_prec, stoc_len):
        x8 = S.pack_act8(x)
        ctx.save_for_backward(x8.codes, x8.exponents, weight)
        return S.sc_matmul(x, weight, "per_row", sc_prec=sc_prec, stoc_len=stoc_len, rng_levels=stoc_len)

    @staticmethod
    def backward(ctx, dy):
        codes, exponents, weight = ctx.saved_tensors
        dx, dw, _ = S.linear_backward(dy, S.Act8(codes, exponents, torch.float32), weight, with_bias=False)
        return dx, dw, None, None


class Block(torch.nn.Module):
    def __init__(self, width: int, hidden: int, sc_len: int | None, generator: torch.Generator):
        super().__init__()

        def randn(*shape, scale=1.0):
            return torch.nn.Parameter(torch.randn(*shape, generator=generator, device=generator.device) * scale)
        self.sc_len = sc_len
        self.norm_w = torch.nn.Parameter(torch.ones(width, device=generator.device))
        self.norm_b = torch.nn.Parameter(torch.zeros(width, device=generator.device))
        self.w1, self.b1 = randn(hidden, width, scale=width ** -0.5), randn(hidden, scale=0.1)
        self.w2, self.b2 = randn(width, hidden, scale=hidden ** -0.5), randn(width, scale=0.1)

    def forward(self, x):
        if self.sc_len is None:  # the teacher: exact throughout, the residual in the epilogue
            h = S.layer_norm(x, self.norm_w, self.norm_b)
            h = S.linear(h, self.w1, self.b1, activation="gelu")
            return S.linear(h, self.w2, self.b2, residual=x)
        h = S.layer_norm(x, self.norm_w, self.norm_b, checkpoint="8bit")
        h = S.linear(h, self.w1, self.b1, activation="gelu", checkpoint="8bit")
        return SCLinear.apply(h, self.w2, 8, self.sc_len) + self.b2 + x


def run(steps: int = 40, rows: int = 788, width: int = 768, hidden: int = 1536, sc_len: int = 128,
        device: str = "cuda", seed: int = 0, log=print):
    """Mean squared error of the student against the teacher before every step and
    after the last."""
    g = torch.Generator(device=device).manual_seed(seed)
    teacher = Block(width, hidden, None, g)
    student = Block(width, hidden, sc_len, g)
    with torch.no_grad():
        for p, q in zip(student.parameters(), teacher.parameters()):
            p.copy_(q + 0.1 * q.std().nan_to_num(0.0) * torch.randn(q.shape, generator=g, device=device))
    opt = torch.optim.Adam(student.parameters(), lr=1e-3)
    x = torch.randn(rows, width, generator=g, device=device)
    with torch.no_grad():
        target = teacher(x)
    losses = []
    for step in range(steps + 1):
        loss = (student(x) - target).square().mean()
        losses.append(float(loss.detach()))
        if step == steps:
            break
        if step % 10 == 0:
            log(f"step {step:3d}  mse {losses[-1]:.5f}")
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
    log(f"step {steps:3d}  mse {losses[-1]:.5f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("steps", 40), ("rows", 788), ("width", 768), ("hidden", 1536), ("sc_len", 128)):
        ap.add_argument("--" + name.replace("_", "-"), type=int, default=value)
    run(**vars(ap.parse_args()))
