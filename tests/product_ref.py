"""The matrix products in 64 bits on the CPU or GPU, with a bound on how far the kernels' outputs may be off.

Bounds, per output, with u = finfo.eps / 2 of the type (a rounding is off by at most half a step):
  z      fp32 sum of K exact or once-rounded products and a bias: (K + 4) 2^-24 (|x| |W|^T + |b|)
  y      z's error times the activation's largest slope (1.13 for gelu; the largest of all of them), the
         fp32 evaluation of the activation (2^-20 of |z| and 2^-22), the residual's addition, one rounding (u |y|)
  dz     dy times act' of the erring z (second derivatives below 1.2), the fp32 evaluation (2^-20); as an
         operand rounded once more (u |dz|). relu': any value between 0 and 1 where z's error spans 0
  dx, dW dz's error times the other operand, the fp32 sum, one rounding
  db     dz's error before its rounding, the fp32 sum, one rounding
and half of the type's smallest number wherever something is rounded to the type.
"""
import math

import torch

F64 = torch.float64
SLOPE, CURVE = 1.13, 1.2
ACTS = (None, "relu", "gelu", "gelu_tanh", "silu", "swiglu")


def _cdf(z):
    return torch.special.ndtr(z)


def act(name, z):
    return {None: lambda t: t, "relu": torch.relu, "gelu": lambda t: t * _cdf(t),
            "gelu_tanh": lambda t: t * torch.sigmoid(math.sqrt(8 / math.pi) * (t + 0.044715 * t ** 3)),
            "silu": lambda t: t * torch.sigmoid(t)}[name](z)


def act_grad(name, z):
    if name is None:
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return _cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(8 / math.pi)
        s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return s + z * s * (1 - s)


def _steps(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def product(x, w, b, name, r, dtype, dy=None):
    """{"y": (value, bound), and with dy "dx", "dw", "db"} of one group, in 64 bits."""
    u, tiny = _steps(dtype)
    e32 = 2.0 ** -24
    x, w = x.to(F64), w.to(F64)
    b = None if b is None else b.to(F64)
    r = None if r is None else r.to(F64)
    rows, k = x.shape
    z = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b, mag + b.abs()
    ez = (k + 4) * e32 * mag
    n = w.shape[0] // 2 if name == "swiglu" else w.shape[0]
    if name == "swiglu":
        g, up, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
        y = act("silu", g) * up
        ey = (SLOPE * eg + 2.0 ** -20 * (g.abs() + 0.25)) * (up.abs() + eu) + act("silu", g).abs() * eu
    else:
        y = act(name, z)
        ey = SLOPE * ez + (0 if name is None else 2.0 ** -20 * (z.abs() + 0.25))
    if r is not None:
        y = y + r
        ey = ey + 2 * e32 * (r.abs() + y.abs())
    out = {"y": (y, ey + u * (y.abs() + ey) + tiny)}
    if dy is None:
        return out
    dy = dy.to(F64)
    if name == "swiglu":
        s, ds = act("silu", g), act_grad("silu", g)
        es = SLOPE * eg + 2.0 ** -20 * (g.abs() + 0.25)
        eds = CURVE * eg + 2.0 ** -20 * (1 + g.abs())
        dz = torch.cat([dy * up * ds, dy * s], 1)
        edz = torch.cat([dy.abs() * (up.abs() * eds + eu * (ds.abs() + eds)), dy.abs() * es], 1)
    else:
        d = act_grad(name, z)
        dz = dy * d
        if name is None:
            edz = torch.zeros_like(dz)
        elif name == "relu":
            edz = torch.where(z.abs() <= ez, dy.abs(), torch.zeros_like(dy))
        else:
            edz = dy.abs() * (CURVE * ez + 2.0 ** -20 * (1 + z.abs()))
    erz = edz + (0 if name is None else u * (dz.abs() + edz) + tiny)

    def rounded(v, e):
        return v, e + u * (v.abs() + e) + tiny

    top = dz.abs() + erz
    out["dx"] = rounded(dz @ w, erz @ w.abs() + (w.shape[0] + 4) * e32 * (top @ w.abs()))
    out["dw"] = rounded(dz.t() @ x, erz.t() @ x.abs() + (rows + 4) * e32 * (top.t() @ x.abs()))
    out["db"] = rounded(dz.sum(0), (edz + (rows + 4) * e32 * top).sum(0))
    return out


def check(got, want, bound, what=""):
    """got is within `bound` of want, everywhere; the worst place is named."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    far = (got.to(F64) - want).abs() / bound.clamp_min(1e-300)
    far = torch.where(torch.isfinite(far), far, torch.full_like(far, math.inf))
    worst = int(far.argmax())
    assert float(far.max()) <= 1.0, (f"{what}: {float(got.flatten()[worst])} at {worst} of {tuple(got.shape)}, "
                                     f"want {float(want.flatten()[worst])} within {float(bound.flatten()[worst])}")
