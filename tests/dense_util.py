"""The dense operators in float64 with bounds on what a float32 / bfloat16 kernel may be off, element by element.

Bounds count roundings. A float32 sum of n products in any order is off by at most ``(n + 16) 2^-24`` of the sum of the
products' magnitudes (16: the rounded operands' missing part, the epilogue). A value rounded to bfloat16 is off by at
most 2^-8 of itself, the half-precision tape by 2^-11. CUDA's float32 exp, erf and tanh and the few operations around
them are within 16 float32 steps; exp(z) of the special-function unit, which bfloat16 results are made of, is within
2^-21 + 1.5 |z| 2^-24 of itself, 64 steps with what surrounds it for |z| < 32.
"""
import math

import torch

U32, U16, UTAPE = 2.0 ** -24, 2.0 ** -8, 2.0 ** -11
ACTS = ("none", "silu", "gelu", "gelu_tanh", "relu", "tanh", "sigmoid")
# no activation bends more than this (second derivatives), or is steeper than that
BEND, STEEP = 1.0, 1.2


def act64(z, act):
    """act(z), act'(z) in float64."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if act == "gelu":
        h = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * h, h + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    if act == "sigmoid":
        return s, s * (1 - s)
    return z * s, s * (1 + z * (1 - s))


def linear64(x, w, b=None, r=None, act="none"):
    """(y, bound, z, bound of z) for inputs of the kernel's own type."""
    half = x.dtype == torch.bfloat16
    x, w = x.double(), w.double()
    K = x.shape[-1]
    z = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    zb = (K + 16) * U32 * mag
    y, _ = act64(z, act)
    yb = zb * STEEP + (64 if half else 16) * U32 * (y.abs() + z.abs() + 1e-30)
    if r is not None:
        y = y + r.double()
        yb = yb + U32 * y.abs()
    if half:
        yb = yb + U16 * (y.abs() + yb)
    return y, yb, z, zb


def linear64_grads(x, w, b, gy, act="none"):
    """{name: (gradient, bound)}."""
    half = x.dtype == torch.bfloat16
    _, _, z, zb = linear64(x, w, b, None, act)
    x, w, gy = x.double(), w.double(), gy.double()
    M, N = gy.shape
    _, slope = act64(z, act)
    gz = gy * slope
    gzb = torch.zeros_like(gz)
    if act != "none":
        gzb = gy.abs() * (BEND * (zb + (UTAPE * z.abs() + 2.0 ** -24 if half else 0)) + (64 if half else 16) * U32 * (slope.abs() + 1))
    sumb = gzb  # what the bias gradient adds: not rounded to bfloat16 on the way
    if half and act != "none":
        gzb = gzb + U16 * (gz.abs() + gzb)
    out = {"x": (gz @ w, gzb @ w.abs() + (N + 16) * U32 * (gz.abs() @ w.abs())),
           "weight": (gz.t() @ x, gzb.t() @ x.abs() + (M + 16) * U32 * (gz.abs().t() @ x.abs())),
           "bias": (gz.sum(0), sumb.sum(0) + (M + 16) * U32 * gz.abs().sum(0))}
    if half:
        out = {k: (v, e + U16 * (v.abs() + e)) for k, (v, e) in out.items()}
    return out


def norm64(x, w=None, b=None, eps=1e-5):
    """(y, bound, xhat, rstd). The mean is off by (D + 2) steps of mean|x|; xhat by that, its own rounding and rstd's."""
    half = x.dtype == torch.bfloat16
    x = x.double()
    D = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * rstd
    off = ((D + 2) * x.abs().mean(-1, keepdim=True) + x.abs()) * U32 * rstd
    xhb = off * (1 + xh.abs()) + (D + 16) * U32 * xh.abs()
    y, yb = xh, xhb
    if w is not None:
        y, yb = y * w.double(), yb * w.double().abs()
    if b is not None:
        y = y + b.double()
    yb = yb + 4 * U32 * (y.abs() + (xh.abs() * w.double().abs() if w is not None else xh.abs()))
    if half:
        yb = yb + U16 * (y.abs() + yb)
    return y, yb, xh, rstd, xhb


def norm64_grads(x, w, gy, eps=1e-5, half_params=False):
    """{name: (gradient, bound)}; ``half_params``: the parameters' gradients are rounded to bfloat16."""
    half = x.dtype == torch.bfloat16
    _, _, xh, rstd, xhb = norm64(x, w, None, eps)
    gy = gy.double()
    M, D = gy.shape
    gw = gy if w is None else gy * w.double()
    m1, m2 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    gx = rstd * (gw - m1 - xh * m2)
    e1 = (D + 4) * U32 * gw.abs().mean(-1, keepdim=True)
    e2 = (gw.abs() * xhb).mean(-1, keepdim=True) + (D + 4) * U32 * (gw * xh).abs().mean(-1, keepdim=True)
    size = gw.abs() + m1.abs() + (xh * m2).abs()
    rel = 8 * U32 + (xhb / (1 + xh.abs())).amax(-1, keepdim=True)  # rstd's own error
    gxb = rstd * (e1 + xh.abs() * e2 + xhb * m2.abs() + rel * size)
    out = {"x": (gx, gxb + U16 * (gx.abs() + gxb) if half else gxb)}
    for name, v, e in (("weight", (gy * xh).sum(0), (gy.abs() * xhb).sum(0) + (M + 16) * U32 * (gy * xh).abs().sum(0)),
                       ("bias", gy.sum(0), (M + 16) * U32 * gy.abs().sum(0))):
        out[name] = (v, e + U16 * (v.abs() + e) if half_params else e)
    return out


def within(got, want, bound, what=""):
    """Assert |got - want| <= bound everywhere, and equal NaN and infinity."""
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: finite in other places"
    d = ((got - want).abs() - bound)[fine]
    if d.numel():
        k = int(d.argmax())
        assert float(d[k]) <= 0, (f"{what}: off by {float((got - want).abs()[fine][k]):.3e} where "
                                  f"{float(bound[fine][k]):.3e} is allowed (value {float(want[fine][k]):.3e})")
