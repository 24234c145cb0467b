"""The exact layers (layer norm, linear, 8-bit checkpoints) against 64-bit formulas.

Bounds. ``U`` is a type's unit roundoff. A float32 sum of n terms t_i is off by
at most (n + 8) * 2^-23 * sum |t_i| whatever its order and rounding mode
(elementwise checks), and by about sqrt(n) * 2^-24 of its value's typical size
when the roundings are independent; the Frobenius checks allow four times that
plus one rounding of the output. Float32 products from the library's own
formulas (erf, exp, tanh) are allowed 2^-20 relative.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import scmp_kernels_b200 as S  # noqa: E402
from scmp_kernels_b200 import _lib  # noqa: E402

DEV = torch.device("cuda", 0)
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
E = 2.0 ** -23
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def act64(v, act):
    """(value, derivative) in 64 bits"""
    if act == "relu":
        return v.clamp(min=0), (v > 0).double()
    if act == "gelu":
        c = 0.5 * torch.erfc(-v / math.sqrt(2))
        return v * c, c + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (v + 0.044715 * v ** 3))
        return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * k * (1 + 3 * 0.044715 * v * v)
    if act == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    return v, torch.ones_like(v)


def close(got, want, bound):
    """|got - want| <= bound elementwise, `want` and `bound` in 64 bits."""
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} out of bound; worst {float((err - bound).max()):.3g} "
                           f"over at error {float(err.max()):.3g}")


def rel(got, want):
    n = float(want.norm())
    return float((got.double() - want).norm()) / n if n else float(got.double().norm())


# ---------------------------------------------------------------------------
# 8-bit checkpoints
# ---------------------------------------------------------------------------
def pack64(x):
    """(codes, exponent bytes) from the definition, in float64 on the CPU."""
    half = x.dtype == torch.float16
    v = x.double().cpu()
    r, d = v.shape
    nb = -(-d // 32)
    codes, exps = torch.zeros(r, d, dtype=torch.int8), torch.zeros(r, nb, dtype=torch.uint8)
    for b in range(nb):
        s = v[:, 32 * b:32 * b + 32]
        for i in range(r):
            if not torch.isfinite(s[i]).all():
                exps[i, b] = 255
                continue
            top = float(s[i].abs().max())
            e = max(math.frexp(top)[1] - 1 - 6 if top > 0 else -10 ** 6, -24 if half else -126)
            exps[i, b] = e + 127
            codes[i, 32 * b:32 * b + 32] = torch.round(s[i] * 2.0 ** -e).clamp(-127, 127).to(torch.int8)
    return codes, exps


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (4, 200), (7, 1000), (2, 8)])
def test_act8_codes_are_the_definition(dtype, shape):
    t = DT[dtype]
    x = randn(gen(1), *shape)
    x *= torch.pow(2.0, torch.randint(-20, 15, (shape[0], 1), device=DEV).float())
    if shape[1] > 8:
        x[0, 3], x[-1, 5] = 127.6 / 128 * 2.0, -0.0  # saturation near a power of two
        x[:, 7] = 0.5 * x[:, 7].round()              # ties
    x = x.to(t)
    a = S.pack_act8(x)
    codes, exps = pack64(x)
    assert torch.equal(a.codes.cpu(), codes) and torch.equal(a.exponents.cpu(), exps)
    v = S.unpack_act8(a)
    assert v.dtype == t
    want = codes.double() * torch.repeat_interleave(2.0 ** (exps.double() - 127), 32, 1)[:, :shape[1]]
    assert torch.equal(v.double().cpu(), want)  # exact in every type
    assert torch.equal(S.unpack_act8(a, torch.float32).double().cpu(), want)


@pytest.mark.parametrize("dtype", list(DT))
def test_act8_extremes(dtype):
    t = DT[dtype]
    fi = torch.finfo(t)
    x = torch.zeros(6, 70, device=DEV, dtype=t)
    x[1, 0], x[1, 40] = fi.max, -fi.max
    x[2, 3], x[2, 35] = float("inf"), float("nan")
    x[3, 1], x[3, 33], x[3, 69] = fi.tiny, fi.smallest_normal / 2, -fi.tiny
    x[4] = fi.max
    x[5, 64] = float("-inf")
    a = S.pack_act8(x)
    codes, exps = pack64(x)
    assert torch.equal(a.codes.cpu(), codes) and torch.equal(a.exponents.cpu(), exps)
    v = S.unpack_act8(a)
    assert torch.equal(v[0], x[0])
    assert v[2, :64].isnan().all() and (v[2, 64:] == 0).all() and v[5, 64:].isnan().all() and (v[5, :64] == 0).all()
    assert v[1].isfinite().all() and v[4].isfinite().all()
    assert (v[4].double() >= fi.max * 0.99).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_act8_strides_and_shapes(dtype):
    t = DT[dtype]
    big = randn(gen(2), 9, 130, dtype=t)
    views = [big[:, :96], big[:, 1:97], big[::2, 8:40], big.t(), randn(gen(3), 2, 3, 65, dtype=t),
             randn(gen(4), 4, 6, 64, dtype=t)[:, :3], big[:0]]
    for x in views:
        a = S.pack_act8(x)
        b = S.pack_act8(x.clone(memory_format=torch.contiguous_format))
        assert a.shape == x.shape and torch.equal(a.codes, b.codes) and torch.equal(a.exponents, b.exponents)
        assert torch.equal(S.unpack_act8(a), S.unpack_act8(b))
    assert S.pack_act8(big).nbytes == 9 * 130 + 9 * 5


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (3, 7), (5, 32), (17, 129), (9, 256), (33, 768), (2, 1000), (4, 1024), (7, 1031), (3, 2048),
               (5, 3000), (3, 4096), (2, 8192), (3, 5001), (1, 16384), (2, 16385), (2, 20000), (600, 64), (300, 2056)]


def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    y = h if w is None else h * w.double()
    y = y if b is None else y + b.double()
    return y, mean[..., 0], rstd[..., 0], h


def norm_inputs(shape, t, seed=5):
    g = gen(seed)
    x = randn(g, *shape) * 1.5 + 0.7
    x[:, :: max(1, shape[1] // 7)] *= 10
    w = randn(g, shape[1], scale=0.2) + 1.0
    b = randn(g, shape[1], scale=0.3)
    dy = randn(g, *shape)
    return x.to(t), w, b, dy.to(t)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_forward(dtype, shape):
    t, (r, d) = DT[dtype], shape
    x, w, b, _ = norm_inputs(shape, t)
    w, b = (w.to(t), b.to(t)) if d % 2 else (w, b)  # parameters of x's type, or float32
    y, mean, rstd, x8 = S.layer_norm_forward(x, w, b, eps=1e-5, checkpoint8=True)
    y64, m64, r64, h = norm64(x, w, b, 1e-5)
    n = d + 8
    amax = x.double().abs().mean(-1)
    close(mean, m64, n * E * amax)
    # x - mean loses up to (n E) of |x|'s mean; the variance is a sum of n squares of it
    slack = n * E * (1 + amax * r64)
    close(rstd, r64, 4 * slack * r64)
    close(y, y64, U[t] * y64.abs() + TINY[t] + 8 * slack[:, None] * ((h.abs() + 1) * w.double().abs() + b.double().abs()))
    assert rel(y, y64) <= U[t] + 4 * E * (1 + math.sqrt(d)) * float((1 + amax * r64).max())
    ref = S.pack_act8(x)
    assert torch.equal(x8.codes, ref.codes) and torch.equal(x8.exponents, ref.exponents)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_backward(dtype, shape, packed):
    t, (r, d) = DT[dtype], shape
    x, w, _, dy = norm_inputs(shape, t, 6)
    w = w.to(t) if d % 2 else w
    _, mean, rstd, x8 = S.layer_norm_forward(x, w, None, checkpoint8=True)
    src = x8 if packed else x
    xv = S.unpack_act8(x8).double() if packed else x.double()
    dx, dw, db = S.layer_norm_backward(dy, src, mean, rstd, w)
    # the formula on the statistics that were given
    h = (xv - mean.double()[:, None]) * rstd.double()[:, None]
    g = dy.double() * w.double()
    m1, m2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    rs = rstd.double()[:, None]
    dx64 = rs * (g - m1 - h * m2)
    n = d + 8
    # h is a difference of x and the mean: 2^-23 of (|x| + |mean|) rstd
    hb = 4 * E * (xv.abs() + mean.double().abs()[:, None]) * rs + 2 * E * h.abs()
    m2b = (g.abs() * (hb + n * E * h.abs())).mean(-1, keepdim=True)
    m1b = n * E * g.abs().mean(-1, keepdim=True)
    close(dx, dx64, U[t] * dx64.abs() + TINY[t] + rs * (4 * E * (g.abs() + m1.abs() + (h * m2).abs()) + m1b + hb * m2.abs()
                                                        + (h.abs() + hb) * m2b))
    wt = w.dtype
    dw64, db64 = (dy.double() * h).sum(0), dy.double().sum(0)
    assert dw.dtype == db.dtype == wt
    close(dw, dw64, U[wt] * dw64.abs() + TINY[wt] + ((r + 8) * E * h.abs() * dy.double().abs() + hb * dy.double().abs()).sum(0))
    close(db, db64, U[wt] * db64.abs() + TINY[wt] + (r + 8) * E * dy.double().abs().sum(0))


@pytest.mark.parametrize("dtype", list(DT))
def test_norm_optional_parts(dtype):
    t = DT[dtype]
    x, w, b, dy = norm_inputs((11, 264), t, 7)
    y, mean, rstd = S.layer_norm_forward(x)
    close(y, norm64(x, None, None, 1e-5)[0], 2 * U[t] * norm64(x, None, None, 1e-5)[0].abs() + 1e-4)
    y0 = S.layer_norm_forward(x, w)[0]
    y1 = S.layer_norm_forward(x, w, torch.zeros_like(w))[0]
    assert torch.equal(y0, y1)
    assert torch.equal(S.layer_norm_forward(x, None, b)[0], S.layer_norm_forward(x, torch.ones_like(b), b)[0])
    full = S.layer_norm_backward(dy, x, mean, rstd, w)
    part = S.layer_norm_backward(dy, x, mean, rstd, w, with_bias=False)
    assert torch.equal(full[0], part[0]) and torch.equal(full[1], part[1]) and part[2] is None
    dx, dw, db = S.layer_norm_backward(dy, x, mean, rstd)
    ones = S.layer_norm_backward(dy, x, mean, rstd, torch.ones_like(w))
    assert dw is None and torch.equal(dx, ones[0]) and db.dtype == t and torch.equal(db, ones[2].to(t))
    dx2 = S.layer_norm_backward(dy, x, mean, rstd, None, with_bias=False)
    assert torch.equal(dx2[0], dx) and dx2[1] is None and dx2[2] is None


def test_norm_special_rows():
    x = torch.randn(6, 300, device=DEV)
    x[1] = 3.25            # no variance: rstd = 1 / sqrt(eps), y = bias
    x[2, 17] = float("nan")
    x[3, 5] = float("inf")
    x[4] = 0
    w, b = torch.rand(300, device=DEV) + 0.5, torch.randn(300, device=DEV)
    y, mean, rstd = S.layer_norm_forward(x, w, b)
    assert torch.equal(y[1], b) and torch.equal(y[4], b)
    assert mean[1] == 3.25 and abs(float(rstd[1]) * math.sqrt(1e-5) - 1) < 1e-6
    assert y[2].isnan().all() and y[3].isnan().all()
    alone = S.layer_norm_forward(x[[0, 5]], w, b)[0]
    assert torch.equal(y[[0, 5]], alone)  # a bad row stays by itself
    dx, dw, db = S.layer_norm_backward(torch.ones_like(x), x, mean, rstd, w)
    assert dx[2].isnan().all() and dx[[0, 1, 4, 5]].isfinite().all() and dw.isnan().any() and db.isfinite().all()


@pytest.mark.parametrize("dtype", list(DT))
def test_norm_strides_and_empty(dtype):
    t = DT[dtype]
    big = randn(gen(8), 12, 400, dtype=t)
    w, b = randn(gen(9), 320, dtype=t), randn(gen(10), 320, dtype=t)
    wide = torch.randn(641, device=DEV).to(t)
    for x, ww, bb in [(big[:, :320], w, b), (big[:, 3:323], w, b), (big[::3, 40:360], wide[1:321], wide[320:640]),
                      (big.view(3, 4, 400)[..., 8:328], w, b), (big.view(3, 4, 400)[:, ::2, 8:328], wide[1:640:2], b)]:
        c = x.clone(memory_format=torch.contiguous_format)
        got, want = S.layer_norm_forward(x, ww, bb), S.layer_norm_forward(c, ww.clone(), bb.clone())
        for u, v in zip(got, want):
            assert u.shape == v.shape
            close(u, v.double(), 2 * U[t] * v.double().abs() + 1e-5)
        dy = randn(gen(11), *x.shape, dtype=t)
        for u, v in zip(S.layer_norm_backward(dy, x, *want[1:], ww), S.layer_norm_backward(dy, c, *want[1:], ww.clone())):
            close(u, v.double(), 2 * U[t] * v.double().abs() + 1e-4)
    e = big[:0, :320]
    y, mean, rstd = S.layer_norm_forward(e, w, b)
    assert y.shape == (0, 320) and mean.shape == (0,)
    dx, dw, db = S.layer_norm_backward(e, e, mean, rstd, w)
    assert dx.shape == (0, 320) and (dw == 0).all() and (db == 0).all()


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------
LIN_SHAPES = [(1, 1, 1), (1, 64, 33), (3, 5, 7), (1, 4096, 250), (2, 1000, 513), (8, 520, 96), (16, 256, 1000),
              (17, 300, 129), (32, 768, 264), (33, 63, 65), (64, 2048, 128), (100, 72, 300), (128, 128, 128),
              (197, 256, 777), (255, 513, 257), (300, 1024, 512), (512, 64, 40), (1025, 200, 304), (700, 1536, 520)]


def lin_inputs(shape, t, seed=20):
    r, d, m = shape
    g = gen(seed)
    x = randn(g, r, d, dtype=t)
    w = randn(g, m, d, dtype=t, scale=1 / math.sqrt(d))
    b = randn(g, m, scale=0.5)
    res = randn(g, r, m, dtype=t)
    return x, w, b, res


def product_bounds(x64, w64t, n):
    """(sum |x||w|, elementwise bound on a float32 sum of n products)"""
    s = x64.abs() @ w64t.abs()
    return s, (n + 8) * E * s


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", LIN_SHAPES)
def test_linear_forward(dtype, shape):
    t, (r, d, m) = DT[dtype], shape
    x, w, b, res = lin_inputs(shape, t)
    pre64 = x.double() @ w.double().t()
    s, pb = product_bounds(x.double(), w.double().t(), d)
    plain = S.linear_forward(x, w)
    close(plain, pre64, U[t] * pre64.abs() + TINY[t] + pb)
    assert rel(plain, pre64) <= U[t] + 4 * (math.sqrt(d) + 2) * 2.0 ** -24
    for act in ACTS:
        bias = b.to(t) if act in (None, "gelu") else b
        p64 = pre64 + bias.double()
        v64, g64 = act64(p64, act)
        y, pre = S.linear_forward(x, w, bias, activation=act, residual=res, save="exact")
        want = v64 + res.double()
        # activations have slopes of at most 1.13
        slack = 1.2 * (pb + 2 * E * p64.abs()) + 2.0 ** -20 * v64.abs() + 2.0 ** -22
        close(pre, p64, U[t] * p64.abs() + TINY[t] + pb + 2 * E * p64.abs())
        close(y, want, U[t] * want.abs() + TINY[t] + slack + 2 * E * want.abs())
        assert torch.equal(S.linear_forward(x, w, bias, activation=act, residual=res), y)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", LIN_SHAPES)
def test_linear_saves_the_checkpoint_of_its_pre_activation(dtype, shape):
    t, (r, d, m) = DT[dtype], shape
    x, w, b, _ = lin_inputs(shape, t, 21)
    y, p8 = S.linear_forward(x, w, b, activation="gelu", save="8bit")
    assert torch.equal(y, S.linear_forward(x, w, b, activation="gelu"))
    p64 = x.double() @ w.double().t() + b.double()
    _, pb = product_bounds(x.double(), w.double().t(), d)
    # a code is within half a step of the value; the step is at most max / 64 of its block, and a
    # block's largest values saturate by at most another half step
    nb = -(-m // 32)
    pad = torch.zeros(r, nb * 32, dtype=torch.float64, device=DEV)
    pad[:, :m] = p64.abs()
    step = (pad.view(r, nb, 32).amax(-1) * (1 + 2.0 ** -18) / 64).repeat_interleave(32, 1)[:, :m]
    close(S.unpack_act8(p8), p64, step + pb + 2 * E * p64.abs() + TINY[t])


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", LIN_SHAPES)
def test_linear_backward(dtype, shape, packed):
    t, (r, d, m) = DT[dtype], shape
    x, w, b, _ = lin_inputs(shape, t, 22)
    g = gen(23)
    dy, pre = randn(g, r, m, dtype=t), randn(g, r, m, dtype=t, scale=1.5)
    x8, p8 = S.pack_act8(x), S.pack_act8(pre)
    xv, pv = (S.unpack_act8(x8), S.unpack_act8(p8)) if packed else (x, pre)
    for act in ([None, "gelu"] if packed else ACTS):
        dx, dw, db = S.linear_backward(dy, x8 if packed else x, w, activation=act,
                                       pre=None if act is None else p8 if packed else pre, bias_dtype=torch.float32)
        dp64 = dy.double() * act64(pv.double(), act)[1]
        # dpre is rounded to the type once, but for a plain layer, whose dpre is dy
        db_ = 2.0 ** -20 * dy.double().abs() + (0 if act is None else U[t] * dp64.abs() + TINY[t])
        dx64, dw64 = dp64 @ w.double(), dp64.t() @ xv.double()
        _, xb = product_bounds(dp64, w.double(), m)
        _, wb = product_bounds(dp64.t(), xv.double(), r)
        if act is None:
            close(dx, dx64, U[t] * dx64.abs() + TINY[t] + xb)
            close(dw, dw64, U[t] * dw64.abs() + TINY[t] + wb)
        else:
            close(dx, dx64, U[t] * dx64.abs() + TINY[t] + 1.01 * (xb + db_ @ w.double().abs()))
            close(dw, dw64, U[t] * dw64.abs() + TINY[t] + 1.01 * (wb + db_.t() @ xv.double().abs()))
        assert rel(dx, dx64) <= U[t] * (1 if act is None else 2) + 4 * (math.sqrt(m) + 8) * 2.0 ** -24
        assert rel(dw, dw64) <= U[t] * (1 if act is None else 2) + 4 * (math.sqrt(r) + 8) * 2.0 ** -24
        close(db, dp64.sum(0), (r + 8) * E * dp64.abs().sum(0) + 2.0 ** -20 * dy.double().abs().sum(0))


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_backward_parts(dtype):
    t = DT[dtype]
    x, w, b, _ = lin_inputs((70, 96, 200), t, 24)
    dy, pre = randn(gen(25), 70, 200, dtype=t), randn(gen(26), 70, 200, dtype=t)
    kw = dict(activation="silu", pre=pre)
    dx, dw, db = S.linear_backward(dy, x, w, **kw)
    assert dx.dtype == dw.dtype == db.dtype == t
    got = S.linear_backward(dy, None, w, need_dweight=False, with_bias=False, **kw)
    assert torch.equal(got[0], dx) and got[1] is None and got[2] is None
    got = S.linear_backward(dy, x, None, need_dx=False, **kw)
    assert got[0] is None and torch.equal(got[1], dw) and torch.equal(got[2], db)
    got = S.linear_backward(dy, None, None, need_dx=False, need_dweight=False, **kw)
    assert got[0] is None and got[1] is None and torch.equal(got[2], db)
    assert S.linear_backward(dy, None, None, need_dx=False, need_dweight=False, with_bias=False, **kw) == (None, None, None)


@pytest.mark.parametrize("rows", [3, 90])
@pytest.mark.parametrize("dtype", list(DT))
def test_linear_strides_offsets_and_empty(dtype, rows):
    t = DT[dtype]
    g = gen(27)
    bigx, bigw, bigr = randn(g, rows, 400, dtype=t), randn(g, 150, 400, dtype=t, scale=0.1), randn(g, rows, 160, dtype=t)
    wt = randn(g, 136, 150, dtype=t, scale=0.1)
    for x, w, res in [(bigx[:, :136], bigw[:, :136], bigr[:, :150]), (bigx[:, 1:137], bigw[:, 3:139], bigr[:, 5:155]),
                      (bigx[:, 8:144], wt.t(), bigr[:, 8:158]), (bigx[:, :136], bigw[::2, :136], bigr[:, :75]),
                      (bigx[:, ::2][:, :136], bigw[:, 16:152], bigr[:, :150])]:
        a = S.linear_forward(x, w, None, activation="relu", residual=res)
        c = S.linear_forward(x.clone(memory_format=torch.contiguous_format), w.clone(memory_format=torch.contiguous_format),
                             None, activation="relu", residual=res.clone(memory_format=torch.contiguous_format))
        close(a, c.double(), 2 * U[t] * c.double().abs() + 1e-4)
        dy = randn(g, rows, 2 * w.shape[0], dtype=t)[:, 1:1 + w.shape[0]]
        got = S.linear_backward(dy, x, w)
        want = S.linear_backward(dy.contiguous(), x.contiguous(), w.contiguous())
        for u, v in zip(got, want):
            close(u, v.double(), 2 * U[t] * v.double().abs() + 1e-3)
    y3 = S.linear_forward(bigx[:, :390].reshape(rows, 3, 130), bigw[:, :130])
    assert y3.shape == (rows, 3, 150)
    assert torch.equal(y3.reshape(-1, 150), S.linear_forward(bigx[:, :390].reshape(-1, 130), bigw[:, :130]))
    e = bigx[:0]
    y, p8 = S.linear_forward(e, bigw, save="8bit")
    assert y.shape == (0, 150) and p8.shape == (0, 150)
    dx, dw, db = S.linear_backward(y, e, bigw)
    assert dx.shape == (0, 400) and dw.shape == (150, 400) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("dtype", list(DT))
def test_linear_non_finite_values_stay_in_their_row(dtype, rows):
    t = DT[dtype]
    x, w, b, res = lin_inputs((rows, 200, 96), t, 28)
    clean = S.linear_forward(x, w, b, residual=res)
    x = x.clone()
    x[1, 50] = float("nan")
    y, p8 = S.linear_forward(x, w, b, residual=res, save="8bit")
    keep = torch.arange(rows, device=DEV) != 1
    assert y[1].isnan().all() and torch.equal(y[keep], clean[keep])
    assert (p8.exponents[1] == 255).all() and S.unpack_act8(p8)[1].isnan().all()
    x[1, 50] = float("inf")
    y = S.linear_forward(x, w, b, residual=res)
    assert not y[1].isfinite().any() and torch.equal(y[keep], clean[keep])


# ---------------------------------------------------------------------------
# gradients against differences, autograd, streams, determinism, refusals
# ---------------------------------------------------------------------------
def block64(p, x):
    h = norm64(x, p["g"], p["c"], 1e-5)[0]
    u = act64(h @ p["w1"].t() + p["b1"], "gelu")[0]
    return u @ p["w2"].t() + p["b2"] + x


def test_gradients_against_differences():
    """Autograd through norm -> linear(gelu) -> linear(+residual) against central
    differences of the 64-bit block along random directions.

    The differences' own error at h = 1e-5 is about h^2 + 2^-53 / h, 1e-10 of the
    value's scale; the float32 gradient's is below sqrt(n) 2^-24 of its own, with
    n the longest sum (1e-4 allows for the three layers and the direction's
    cancellation)."""
    g = gen(30)
    d, m, r = 48, 80, 37
    p = dict(g=randn(g, d, scale=0.2) + 1, c=randn(g, d), w1=randn(g, m, d, scale=0.15), b1=randn(g, m),
             w2=randn(g, d, m, scale=0.15), b2=randn(g, d))
    x, out = randn(g, r, d), randn(g, r, d)
    q = {k: v.clone().requires_grad_() for k, v in p.items()}
    xg = x.clone().requires_grad_()
    h = S.layer_norm(xg, q["g"], q["c"])
    u = S.linear(h, q["w1"], q["b1"], activation="gelu")
    y = S.linear(u, q["w2"], q["b2"], residual=xg)
    y.backward(out)
    p64 = {k: v.double() for k, v in p.items()}
    names = list(p) + ["x"]
    for name in names:
        base = x.double() if name == "x" else p64[name]
        grad = xg.grad if name == "x" else q[name].grad
        v = torch.randn(base.shape, generator=g, device=DEV, dtype=torch.float64)
        eps = 1e-5

        def at(e):
            if name == "x":
                return (block64(p64, base + e * v) * out.double()).sum()
            return (block64({**p64, name: base + e * v}, x.double()) * out.double()).sum()
        diff = float((at(eps) - at(-eps)) / (2 * eps))
        dot = float((grad.double() * v).sum())
        assert abs(dot - diff) <= 1e-4 * float(grad.double().norm() * v.norm()), (name, dot, diff)


@pytest.mark.parametrize("act", ACTS)
def test_activation_gradient_against_differences(act):
    pre = torch.linspace(-9, 9, 1201, device=DEV)[None]  # zero is not on the grid's neighbours: relu's kink
    pre = pre[pre.abs() > 1e-3][None]
    dy = torch.ones_like(pre)
    db = S.linear_backward(dy, None, None, activation=act, pre=pre, need_dx=False, need_dweight=False)[2]
    h = 1e-6
    diff = (act64(pre.double() + h, act)[0] - act64(pre.double() - h, act)[0]) / (2 * h)
    close(db, diff[0], 2.0 ** -20 * (1 + diff[0].abs()) + 1e-8)


@pytest.mark.parametrize("dtype", list(DT))
def test_autograd_with_8bit_checkpoints(dtype):
    """The 8-bit block's gradients are those of the same calls made by hand, and
    near the exact block's (a code is within 1/64 of its block's largest value)."""
    t = DT[dtype]
    g = gen(31)
    x, w, b = randn(g, 60, 128, dtype=t), randn(g, 96, 128, dtype=t, scale=0.1), randn(g, 96)
    nw, nb, dy = randn(g, 128), randn(g, 128), randn(g, 60, 96, dtype=t)

    def go(checkpoint):
        leaves = [v.clone().requires_grad_() for v in (x, nw, nb, w, b)]
        h = S.layer_norm(leaves[0], leaves[1], leaves[2], checkpoint=checkpoint)
        y = S.linear(h, leaves[3], leaves[4], activation="gelu_tanh", checkpoint=checkpoint)
        y.backward(dy)
        return y.detach(), [v.grad for v in leaves]
    y, exact = go("exact")
    y8, eight = go("8bit")
    assert torch.equal(y, y8)
    h, mean, rstd, x8 = S.layer_norm_forward(x, nw, nb, checkpoint8=True)
    _, p8 = S.linear_forward(h, w, b, activation="gelu_tanh", save="8bit")
    dh, dw, db = S.linear_backward(dy, S.pack_act8(h), w, activation="gelu_tanh", pre=p8, bias_dtype=torch.float32)
    dx, dnw, dnb = S.layer_norm_backward(dh, x8, mean, rstd, nw)
    for u, v in zip(eight, (dx, dnw, dnb, dw, db)):
        assert torch.equal(u, v)
    for u, v in zip(eight, exact):
        assert rel(u, v.double()) < 0.05
    assert [u.dtype for u in eight] == [t, torch.float32, torch.float32, t, torch.float32]


def test_only_what_needs_a_gradient():
    x, w = torch.randn(5, 64, device=DEV), torch.randn(32, 64, device=DEV, requires_grad=True)
    y = S.linear(x, w, activation="relu")
    y.sum().backward()
    assert w.grad is not None and not x.requires_grad
    r = torch.randn(5, 32, device=DEV, requires_grad=True)
    S.linear(x, w.detach(), residual=r).sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))


def test_same_bits_every_time_and_on_another_stream():
    x, w, b, res = lin_inputs((513, 384, 640), torch.bfloat16, 40)
    dy = randn(gen(41), 513, 640, dtype=torch.bfloat16)

    def go():
        h, mean, rstd, x8 = S.layer_norm_forward(x, None, None, checkpoint8=True)
        y, p8 = S.linear_forward(h, w, b, activation="gelu", residual=res, save="8bit")
        dh, dw, db = S.linear_backward(dy, h, w, activation="gelu", pre=p8)
        dx, _, dnb = S.layer_norm_backward(dh, x8, mean, rstd)
        return [h, y, p8.codes, dh, dw, db, dx, dnb]
    want = go()
    for _ in range(3):
        for u, v in zip(go(), want):
            assert torch.equal(u, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = go()
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    assert _lib.device_error() == 0


def test_calls_can_be_captured_in_a_graph():
    x, w, b, res = lin_inputs((300, 256, 520), torch.bfloat16, 42)
    dy = randn(gen(43), 300, 520, dtype=torch.bfloat16)

    def go():
        h, mean, rstd = S.layer_norm_forward(x)
        y, pre = S.linear_forward(h, w, b, activation="silu", residual=res, save="exact")
        dh, dw, db = S.linear_backward(dy, h, w, activation="silu", pre=pre)
        return [y, dw, db, S.layer_norm_backward(dh, x, mean, rstd)[0]]
    go()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = go()
    x.copy_(randn(gen(44), 300, 256, dtype=torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    for u, v in zip(outs, go()):
        assert torch.equal(u, v)


def test_offsets_past_32_bits():
    """Row offsets of a tensor of more than 2^31 elements."""
    rows, d = (1 << 31) // 4096 + 40, 4096
    x = torch.empty(rows, d, dtype=torch.bfloat16, device=DEV)
    x[:8].normal_(generator=gen(50))
    x[-8:].normal_(generator=gen(51))
    x[8:-8] = 1.0
    a = S.pack_act8(x)
    tail = S.pack_act8(x[-8:])
    assert torch.equal(a.codes[-8:], tail.codes) and torch.equal(a.exponents[-8:], tail.exponents)
    assert torch.equal(S.unpack_act8(a)[-8:], S.unpack_act8(tail))
    y, mean, rstd = S.layer_norm_forward(x)
    yt, mt, rt = S.layer_norm_forward(x[-8:])
    assert torch.equal(y[-8:], yt) and torch.equal(rstd[-8:], rt)
    del y
    dx = S.layer_norm_backward(x, a, mean, rstd, with_bias=False)[0]
    assert torch.equal(dx[-8:], S.layer_norm_backward(x[-8:], tail, mt, rt, with_bias=False)[0])
    del dx
    w = torch.randn(32, d, device=DEV, generator=gen(52)).to(torch.bfloat16)
    y = S.linear_forward(x, w)
    close(y[-8:], S.linear_forward(x[-8:].clone(), w).double(), 0.02)
    dxl = S.linear_backward(y, None, w, need_dweight=False, with_bias=False)[0]
    close(dxl[-8:], S.linear_backward(y[-8:].clone(), None, w, need_dweight=False, with_bias=False)[0].double(), 2.0)


def test_refusals():
    x = torch.randn(4, 64, device=DEV)
    w = torch.randn(32, 64, device=DEV)
    v = torch.randn(64, device=DEV)
    y, mean, rstd = S.layer_norm_forward(x)
    p8 = S.pack_act8(x)
    bad = [
        (lambda: S.pack_act8(x.double()), "float32, bfloat16 or float16"),
        (lambda: S.pack_act8(x.cpu()), "CUDA tensor"),
        (lambda: S.pack_act8(x[:, :0]), "last axis"),
        (lambda: S.unpack_act8(p8, torch.float64), "dtype"),
        (lambda: S.Act8(p8.codes.float(), p8.exponents), "int8"),
        (lambda: S.Act8(p8.codes, p8.exponents[:, :1]), "exponents must be"),
        (lambda: S.Act8(p8.codes.t(), p8.exponents), "exponents must be"),
        (lambda: S.layer_norm_forward(x, v[:5]), "weight must be"),
        (lambda: S.layer_norm_forward(x, v.half()), "weight must be"),
        (lambda: S.layer_norm_forward(x, v, v.cpu()), "bias is on"),
        (lambda: S.layer_norm_forward(x, eps=-1.0), "eps"),
        (lambda: S.layer_norm_forward(x.long()), "float32"),
        (lambda: S.layer_norm_backward(x, x[:2], mean, rstd), "shape"),
        (lambda: S.layer_norm_backward(x, x.half(), mean, rstd), "dy is"),
        (lambda: S.layer_norm_backward(x, x, mean.double(), rstd), "mean must be"),
        (lambda: S.layer_norm_backward(x, x, mean, rstd[:2]), "rstd must be"),
        (lambda: S.layer_norm(x, checkpoint="4bit"), "checkpoint"),
        (lambda: S.linear_forward(x, w[:, :5]), "inner dimension"),
        (lambda: S.linear_forward(x, w.half()), "weight is"),
        (lambda: S.linear_forward(x, v), "2D"),
        (lambda: S.linear_forward(x, w, v), "bias must be"),
        (lambda: S.linear_forward(x, w, activation="tanh"), "activation"),
        (lambda: S.linear_forward(x, w, residual=x), "residual must be"),
        (lambda: S.linear_forward(x, w, save="4bit"), "save"),
        (lambda: S.linear_forward(x.cpu(), w), "CUDA tensor"),
        (lambda: S.linear_backward(x[:, :32], x, w, activation="relu"), "needs pre"),
        (lambda: S.linear_backward(x[:, :32], None, w), "needs x"),
        (lambda: S.linear_backward(x[:, :32], x, None), "needs the weight"),
        (lambda: S.linear_backward(x[:, :32], x[:3], w), "shape"),
        (lambda: S.linear_backward(x[:, :32], x, w, activation="relu", pre=x), "pre must be"),
        (lambda: S.linear_backward(x[:, :32], x, w, bias_dtype=torch.float16), "bias_dtype"),
        (lambda: S.linear(x, w, checkpoint="none"), "checkpoint"),
    ]
    for f, word in bad:
        with pytest.raises(ValueError, match=word):
            f()


def test_small_workspaces_are_refused():
    lib = _lib.lib()
    x = torch.randn(4, 64, device=DEV)
    st = lib.scmp_layer_norm_backward(x.data_ptr(), 64, x.data_ptr(), 64, None, None, _lib.F32, 4, 64, x.data_ptr(),
                                      x.data_ptr(), None, _lib.F32, x.data_ptr(), x.data_ptr(), None, x.data_ptr(), 8, None)
    assert st == _lib.SCMP_ERR_WORKSPACE and b"workspace" in lib.scmp_last_error()
    st = lib.scmp_linear_backward(x.data_ptr(), 64, x.data_ptr(), 64, None, None, x.data_ptr(), 64, x.data_ptr(), 64,
                                  None, None, _lib.F32, 4, 64, 64, 1, x.data_ptr(), None, None, _lib.F32, None, 0, None)
    assert st == _lib.SCMP_ERR_WORKSPACE and b"workspace" in lib.scmp_last_error()


# ---------------------------------------------------------------------------
# linear: many tiles, split tiles, odd pitches
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(5000, 130, 2600), (4500, 64, 2601), (2600, 1100, 1999), (300, 2500, 40)])
def test_linear_forward_of_many_tiles(dtype, shape):
    # several tiles of different columns in turn on every SM pair, with one accumulator
    # chain and with more; the last of few tiles in parts
    t, (r, d, m) = DT[dtype], shape
    x, w, b, res = lin_inputs(shape, t, 60)
    pre64 = x.double() @ w.double().t()
    _, pb = product_bounds(x.double(), w.double().t(), d)
    for bias in (b.to(t), b, None):
        p64 = pre64 if bias is None else pre64 + bias.double()
        for residual in (res, None):
            want = p64 if residual is None else p64 + residual.double()
            y = S.linear_forward(x, w, bias, residual=residual)
            close(y, want, U[t] * want.abs() + TINY[t] + pb + 2 * E * p64.abs() + 2 * E * want.abs())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(700, 1024, 1030), (394, 520, 1000), (300, 600, 5000), (12340, 320, 256),
                                   (40, 4000, 4100), (3000, 44, 300), (3000, 46, 300), (3000, 45, 301)])
def test_linear_gradients_together_and_alone(dtype, shape):
    t, (r, d, m) = DT[dtype], shape
    x, w, _, _ = lin_inputs(shape, t, 61)
    dy = randn(gen(62), r, m, dtype=t)
    dy64 = dy.double()
    dx64, dw64 = dy64 @ w.double(), dy64.t() @ x.double()
    _, xb = product_bounds(dy64, w.double(), m)
    _, wb = product_bounds(dy64.t(), x.double(), r)
    both = S.linear_backward(dy, x, w, with_bias=False)
    alone = (S.linear_backward(dy, None, w, need_dweight=False, with_bias=False)[0],
             S.linear_backward(dy, x, None, need_dx=False, with_bias=False)[1])
    for dx, dw in (both[:2], alone):
        close(dx, dx64, U[t] * dx64.abs() + TINY[t] + xb)
        close(dw, dw64, U[t] * dw64.abs() + TINY[t] + wb)
    again = S.linear_backward(dy, x, w, with_bias=False)
    assert torch.equal(again[0], both[0]) and torch.equal(again[1], both[1])
