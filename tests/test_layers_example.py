"""The fine-tuning example runs, and its straight-through gradients are those of
the exact block at the SC block's activations."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

spec = importlib.util.spec_from_file_location("finetune_mlp", os.path.join(REPO, "examples", "finetune_mlp.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def test_the_example_learns():
    losses = example.run(steps=15, rows=96, width=128, hidden=200, log=lambda *_: None)
    assert len(losses) == 16 and all(l == l for l in losses)
    assert losses[-1] < 0.7 * losses[0]


def test_straight_through_gradient():
    import scmp_kernels_b200 as S
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(40, 96, generator=g, device="cuda", requires_grad=True)
    w = (torch.randn(64, 96, generator=g, device="cuda") * 0.1).requires_grad_()
    dy = torch.randn(40, 64, generator=g, device="cuda")
    y = example.SCLinear.apply(x, w, 8, 128)
    assert torch.equal(y, S.sc_matmul(x.detach(), w.detach(), "per_row", sc_prec=8, stoc_len=128, rng_levels=128))
    y.backward(dy)
    dx, dw, _ = S.linear_backward(dy, S.pack_act8(x.detach()), w.detach(), with_bias=False)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
