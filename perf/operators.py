"""Cases of the layers next to ``sc_matmul``: layer norm, the exact linear layer
and 8-bit activation checkpoints, each forward and backward.

The layers round a stochastic-computing model trains through: the layer norm
before a product, the products a mixed-precision model keeps exact (with bias,
activation and residual in one pass) and that give an SC layer its straight-through
gradient, and the activations kept between the passes in 8 bits (``Act8``: blocks
of 32 values along a row share a power of two, see ``_pack``).

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once at the end) or, where ``own`` is true, through the package's
public functions. ``exact`` restates every case in 64 bits, apart from both.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 32          # values of a row that share one power of two in an 8-bit checkpoint
EPS = 1e-5


def listed():
    return [
        # layer norm of one decoded token at the 4096-wide residual stream: latency
        dict(name="norm token", op="norm", rows=1, d=4096, dtype="bf16"),
        # a batch of 64 images of 197 patches at width 768, in float32 as sc_matmul takes it
        dict(name="norm images fp32", op="norm", rows=12608, d=768, dtype="fp32"),
        # its gradient in half precision at a ragged batch and an odd width
        dict(name="norm grad odd fp16", op="norm_grad", rows=1001, d=1023, dtype="fp16", ckpt="exact"),
        # the gradient of 8192 tokens at width 8192, the input kept in 8 bits
        dict(name="norm grad 8bit", op="norm_grad", rows=8192, d=8192, dtype="bf16", ckpt="8bit"),
        # one decoded token through the 4096 -> 11008 up-projection: the weight's bytes
        dict(name="linear token", op="linear", rows=1, d=4096, m=11008, dtype="bf16", act="silu",
             bias=True, residual=False, save="none"),
        # a float32 layer of one 197-patch image at odd widths, everything in the epilogue
        dict(name="linear odd fp32", op="linear", rows=197, d=1111, m=1001, dtype="fp32", act="gelu",
             bias=True, residual=True, save="none"),
        # the attention's output projection of the image batch, added to the residual stream
        dict(name="linear images fp16", op="linear", rows=12608, d=768, m=768, dtype="fp16", act="none",
             bias=True, residual=True, save="none"),
        # the up-projection of 4096 tokens in training: the pre-activation kept in 8 bits
        dict(name="linear up 8bit", op="linear", rows=4096, d=4096, m=11008, dtype="bf16", act="gelu",
             bias=True, residual=False, save="8bit"),
        # the gradients of a small float32 layer of two 197-patch images
        dict(name="linear grad fp32", op="linear_grad", rows=394, d=520, m=1000, dtype="fp32", act="gelu",
             ckpt="exact"),
        # the gradients of the up-projection, input and pre-activation kept in 8 bits
        dict(name="linear grad up 8bit", op="linear_grad", rows=4096, d=4096, m=11008, dtype="bf16",
             act="gelu", ckpt="8bit"),
        # a checkpoint of a few tokens: latency
        dict(name="act8 tokens", op="act8", rows=16, d=4096, dtype="bf16"),
        # a checkpoint of 8192 tokens at width 8192
        dict(name="act8 long fp32", op="act8", rows=8192, d=8192, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "linear", "linear", "linear_grad", "linear_grad", "act8"])
    c = dict(op=op, rows=_log(rng, 1, 12608), d=_log(rng, 32, 8192), dtype=rng.choice(list(DTYPES)))
    if op in ("linear", "linear_grad"):
        c["m"] = _log(rng, 32, 11008)
        if rng.random() < 0.5:  # half of them at widths that models use
            c["d"], c["m"] = -(-c["d"] // 64) * 64, -(-c["m"] // 64) * 64
        most = 4096 * 4096 * 11008 // (2 if c["dtype"] == "fp32" else 1)
        c["rows"] = max(1, min(c["rows"], most // (c["d"] * c["m"])))
        c["act"] = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    elif rng.random() < 0.5:
        c["d"] = -(-c["d"] // 64) * 64
    if op == "linear":
        c["bias"], c["residual"] = rng.random() < 0.7, rng.random() < 0.5
        # a float32 checkpoint of a computed value may differ by a whole code between any two
        # right kernels (a tie on either side), so it is drawn for the 16-bit types
        c["save"] = rng.choice(["none", "exact"] + ([] if c["dtype"] == "fp32" else ["8bit"]))
    if op in ("norm_grad", "linear_grad"):
        c["ckpt"] = rng.choice(["exact", "8bit"])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(g, rows, d, dtype):
    """N(0,1) with one channel in a hundred scaled by 20, as activations of large models are."""
    x = torch.randn(rows, d, generator=g, device="cuda")
    n = max(1, d // 100)
    x[:, torch.randperm(d, generator=g, device="cuda")[:n]] *= 20.0
    return x.to(dtype)


def prepare(case, seed):
    c = dict(case)
    t = DTYPES[c["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(t)

    r, d = c["rows"], c["d"]
    s = {"case": c, "x": _activations(g, r, d, t)}
    if c["op"] in ("norm", "norm_grad"):
        s["weight"], s["bias"] = randn(d, scale=0.1, shift=1.0), randn(d, scale=0.1)
    if c["op"] == "norm_grad":
        x = s["x"].float()
        mu = x.mean(-1)
        s["mean"], s["rstd"] = mu, 1.0 / torch.sqrt((x - mu[:, None]).square().mean(-1) + EPS)
        s["dy"] = randn(r, d, scale=0.01)
    if c["op"] in ("linear", "linear_grad"):
        s["weight"] = randn(c["m"], d, scale=0.02)
    if c["op"] == "linear":
        s["bias"] = randn(c["m"], scale=0.1) if c["bias"] else None
        s["residual"] = randn(r, c["m"]) if c["residual"] else None
    if c["op"] == "linear_grad":
        s["dy"] = randn(r, c["m"], scale=0.01)
        s["pre"] = randn(r, c["m"], scale=1.5) if c["act"] != "none" else None
    if c.get("ckpt") == "8bit":  # what the forward pass left
        s["x8"] = _pack(s.pop("x"), t)
        if s.get("pre") is not None:
            s["pre8"] = _pack(s.pop("pre"), t)
    return s


# ---------------------------------------------------------------------------
# plain form: 32 bits, elementary operations
# ---------------------------------------------------------------------------
def _pack(x, dtype):
    """(codes int8 (r, d), exponents uint8 (r, ceil(d/32))): code * 2^(exponent - 127).

    The exponent of a block is floor(log2(largest magnitude)) - 6, so that the codes
    fill -127..127 (128 saturates), at least -126 (-24 for half precision, whose
    smallest step that is); codes round half to even. A block that holds an
    infinity or a NaN has exponent byte 255 and stands for NaN.
    """
    r, d = x.shape
    nb = -(-d // BLOCK)
    v = torch.zeros(r, nb * BLOCK, dtype=torch.float32, device=x.device)
    v[:, :d] = x
    v = v.view(r, nb, BLOCK)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    bits = torch.where(bad, torch.zeros_like(top), top).view(torch.int32)
    e = ((bits >> 23) - 127 - 6).clamp(min=-24 if dtype == torch.float16 else -126)
    inv = ((127 - e) << 23).to(torch.int32).view(torch.float32)  # 2^-e
    q = torch.round(v * inv[..., None]).clamp(-127, 127)
    q = torch.where(bad[..., None], torch.zeros_like(q), q)
    exps = torch.where(bad, torch.full_like(e, 255), e + 127)
    return q.view(r, nb * BLOCK)[:, :d].to(torch.int8).contiguous(), exps.to(torch.uint8).contiguous()


def _unpack(codes, exps):
    """The float32 values of a checkpoint."""
    r, d = codes.shape
    e = exps.to(torch.int32)
    scale = torch.where(e == 255, torch.full_like(e, 0x7FC00000), e << 23).view(torch.float32)
    return codes.float() * scale.repeat_interleave(BLOCK, 1)[:, :d]


def _act(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _act_grad(v, act):
    if act == "relu":
        return (v > 0).float()
    if act == "gelu":
        return (0.5 * (1.0 + torch.erf(v * math.sqrt(0.5)))
                + v * torch.exp(-0.5 * v * v) * (1.0 / math.sqrt(2.0 * math.pi)))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v))
        return 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * v * v)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-v))
        return s * (1.0 + v * (1.0 - s))
    return torch.ones_like(v)


def _plain(s):
    c = s["case"]
    t = DTYPES[c["dtype"]]
    if c["op"] == "norm":
        x = s["x"].float()
        mean = x.mean(-1)
        u = x - mean[:, None]
        rstd = 1.0 / torch.sqrt(u.square().mean(-1) + EPS)
        y = u * rstd[:, None] * s["weight"].float() + s["bias"].float()
        return {"y": y.to(t), "mean": mean, "rstd": rstd}
    if c["op"] == "norm_grad":
        x = s["x"].float() if "x" in s else _unpack(*s["x8"])
        dy = s["dy"].float()
        xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * s["weight"].float()
        dx = s["rstd"][:, None] * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        return {"dx": dx.to(t), "dweight": (dy * xh).sum(0).to(t), "dbias": dy.sum(0).to(t)}
    if c["op"] == "linear":
        pre = s["x"].float() @ s["weight"].float().t()
        if s["bias"] is not None:
            pre = pre + s["bias"].float()
        y = _act(pre, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        out = {"y": y.to(t)}
        if c["save"] == "exact":
            out["pre"] = pre.to(t)
        elif c["save"] == "8bit":
            out["pre"] = _unpack(*_pack(pre, t)).to(t)
        return out
    if c["op"] == "linear_grad":
        x = s["x"].float() if "x" in s else _unpack(*s["x8"])
        dpre = s["dy"].float()
        if c["act"] != "none":
            pre = s["pre"].float() if "pre" in s else _unpack(*s["pre8"])
            dpre = dpre * _act_grad(pre, c["act"])
        return {"dx": (dpre @ s["weight"].float()).to(t), "dweight": (dpre.t() @ x).to(t), "dbias": dpre.sum(0).to(t)}
    return {"values": _unpack(*_pack(s["x"], t)).to(t)}


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------
def _own(s):
    import scmp_kernels_b200 as S
    c = s["case"]
    if c["op"] == "norm":
        y, mean, rstd = S.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if c["op"] == "norm_grad":
        x = s["x"] if "x" in s else S.Act8(*s["x8"], DTYPES[c["dtype"]])
        dx, dw, db = S.layer_norm_backward(s["dy"], x, s["mean"], s["rstd"], s["weight"])
        return {"dx": dx, "dweight": dw, "dbias": db}
    act = None if c.get("act") == "none" else c.get("act")
    if c["op"] == "linear":
        if c["save"] == "none":
            return {"y": S.linear_forward(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"])}
        y, pre = S.linear_forward(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"],
                                  save=c["save"])
        return {"y": y, "pre": pre if c["save"] == "exact" else S.unpack_act8(pre)}
    if c["op"] == "linear_grad":
        t = DTYPES[c["dtype"]]
        x = s["x"] if "x" in s else S.Act8(*s["x8"], t)
        pre = s["pre"] if "pre" in s else S.Act8(*s["pre8"], t) if "pre8" in s else None
        dx, dw, db = S.linear_backward(s["dy"], x, s["weight"], activation=act, pre=pre)
        return {"dx": dx, "dweight": dw, "dbias": db}
    return {"values": S.unpack_act8(S.pack_act8(s["x"]))}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c, z = case, SIZE[case["dtype"]]
    r, d = c["rows"], c["d"]
    packed = 1.0 + 1.0 / BLOCK
    kept = packed if c.get("ckpt") == "8bit" else z
    if c["op"] == "norm":
        return {"bytes": 2 * z * r * d + 2 * z * d + 8 * r, "flops": 8 * r * d}
    if c["op"] == "norm_grad":
        return {"bytes": (2 * z + kept) * r * d + 8 * r + 3 * z * d, "flops": 14 * r * d}
    if c["op"] == "act8":
        return {"bytes": (2 * z + packed) * r * d, "flops": 4 * r * d}
    m = c["m"]
    if c["op"] == "linear":
        saved = {"none": 0, "exact": z, "8bit": packed}[c["save"]]
        return {"bytes": z * (r * d + m * d + r * m * (2 if c["residual"] else 1) + (m if c["bias"] else 0)) + saved * r * m,
                "flops": 2 * r * d * m}
    return {"bytes": z * (r * m + 2 * m * d + r * d + m) + kept * (r * d + (r * m if c["act"] != "none" else 0)),
            "flops": 4 * r * d * m}


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _two_to(e):
    """2^e in float64, by its bits (pow and exp2 are an ulp off on the device, which moves ties)."""
    return (e.to(torch.int64) + 1023 << 52).view(torch.float64)


def _exact_codes(values, half):
    """Values an 8-bit checkpoint of `values` (float64, (r, d)) stands for."""
    r, d = values.shape
    out = torch.empty_like(values)
    for j in range(0, d, BLOCK):
        b = values[:, j:j + BLOCK]
        top = b.abs().amax(1, keepdim=True)
        _, ex = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))
        e = ex.to(torch.float64) - 1 - 6
        e = torch.where(top > 0, e, torch.full_like(e, -200.0)).clamp(min=-24 if half else -126)
        step = _two_to(e)
        out[:, j:j + BLOCK] = torch.clamp(torch.round(b / step), -127, 127) * step
    return out


def _exact_act(v, act):
    """(value, derivative)"""
    one = torch.ones_like(v)
    if act == "relu":
        return torch.where(v > 0, v, 0 * v), torch.where(v > 0, one, 0 * one)
    if act == "gelu":
        phi = 0.5 * torch.erfc(-v / np.sqrt(2.0))
        return v * phi, phi + v * torch.exp(-v * v / 2) / np.sqrt(2 * np.pi)
    if act == "gelu_tanh":
        k = np.sqrt(2 / np.pi)
        th = torch.tanh(k * (v + 0.044715 * v ** 3))
        return v * (1 + th) / 2, (1 + th) / 2 + v / 2 * (1 - th ** 2) * k * (1 + 0.134145 * v ** 2)
    if act == "silu":
        sg = torch.sigmoid(v)
        return v * sg, sg + v * sg * (1 - sg)
    return v, one


def exact(case, seed):
    s = prepare(case, seed)
    c, t = s["case"], torch.float64
    if c["op"] == "act8":
        return {"values": _exact_codes(s["x"].to(t), c["dtype"] == "fp16")}
    if "x" in s:
        x = s["x"].to(t)
    else:
        codes, exps = s["x8"]
        x = codes.to(t) * _two_to(exps.to(t) - 127).repeat_interleave(BLOCK, 1)[:, :c["d"]]
    w = s["weight"].to(t)
    if c["op"] == "norm":
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + EPS) ** -0.5
        return {"y": torch.addcmul(s["bias"].to(t), (x - mean[:, None]) * rstd[:, None], w), "mean": mean, "rstd": rstd}
    if c["op"] == "norm_grad":
        dy, n = s["dy"].to(t), c["d"]
        h = (x - s["mean"].to(t)[:, None]) * s["rstd"].to(t)[:, None]
        s1, s2 = dy @ w, (dy * h) @ w
        dx = (dy * w - (s1[:, None] + h * s2[:, None]) / n) * s["rstd"].to(t)[:, None]
        return {"dx": dx, "dweight": torch.einsum("rd,rd->d", dy, h), "dbias": dy.sum(0)}
    if c["op"] == "linear":
        pre = torch.einsum("rd,md->rm", x, w)
        if c["bias"]:
            pre += s["bias"].to(t)
        y, _ = _exact_act(pre, c["act"])
        out = {"y": y + s["residual"].to(t) if c["residual"] else y}
        if c["save"] == "exact":
            out["pre"] = pre
        elif c["save"] == "8bit":
            out["pre"] = _exact_codes(pre, c["dtype"] == "fp16")
        return out
    dpre = s["dy"].to(t)
    if c["act"] != "none":
        if "pre" in s:
            pre = s["pre"].to(t)
        else:
            codes, exps = s["pre8"]
            pre = codes.to(t) * _two_to(exps.to(t) - 127).repeat_interleave(BLOCK, 1)[:, :c["m"]]
        dpre = dpre * _exact_act(pre, c["act"])[1]
    return {"dx": torch.einsum("rm,md->rd", dpre, w), "dweight": torch.einsum("rm,rd->md", dpre, x),
            "dbias": dpre.sum(0)}
