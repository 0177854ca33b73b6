"""Plain 64-bit forms of the dense head's operators, with bounds on what a
correctly rounded 32-bit evaluation may be off by (shared by the GPU tests).

Unit roundoffs: u = 2^-24 of binary32, U of the tensors' own type.  A sum of n
products in binary32, in any order, is within (n + 2) u of the sum of their
magnitudes; a result rounded to the type adds U of its size (and half the
smallest subnormal, for float16)."""

import math

import torch

U32 = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
# The functions themselves (expf, erff and a few operations on their results).
FUNC = 16 * U32
# Largest |act'| and |act''| between the kinks.
SLOPE = {"none": 1.0, "relu": 1.0, "crelu": 1.0, "screlu": 2.0, "silu": 1.1, "gelu": 1.13}
CURVE = {"none": 0.0, "relu": 0.0, "crelu": 0.0, "screlu": 2.0, "silu": 0.5, "gelu": 0.8}


def act(z, name):
    """(act(z), act'(z)) in the type of z."""
    one = torch.ones_like(z)
    if name == "none":
        return z, one
    if name == "relu":
        return z.clamp(min=0), one * (z > 0)
    if name in ("crelu", "screlu"):
        c, inside = z.clamp(0, 1), one * ((z >= 0) & (z <= 1))
        return (c, inside) if name == "crelu" else (c * c, 2 * c * inside)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def rounded(err, value, dtype):
    return err + ROUND[dtype] * (value.abs() + err) + TINY[dtype]


def linear(x, w, b, r, name, dy=None):
    """{name: (value, bound)} of y and, where dy is given, dx, dw and db; inputs on the CPU in their own type."""
    dtype = x.dtype
    xd, wd = x.double(), w.double()
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    z, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    zerr = (K + 3) * U32 * mag
    a, d = act(z, name)
    y = a if r is None else a + r.double()
    yerr = SLOPE[name] * zerr + FUNC * (z.abs() + 1) + U32 * y.abs()
    out = {"y": (y, rounded(yerr, y, dtype))}
    if dy is not None:
        g = dy.double()
        derr = CURVE[name] * zerr
        if name in ("silu", "gelu", "screlu"):
            derr = derr + FUNC * (z.abs() + 1) + (0 if dtype == torch.float32 else 2.0 ** -14)
        dz = g * d
        plain = g.abs() * derr + U32 * dz.abs()  # the bias grad's terms are not rounded
        held = plain if name == "none" else rounded(plain, dz, dtype)  # the products' are
        dx, dw, db = dz @ wd, dz.t() @ xd, dz.sum(0)
        out["dx"] = (dx, rounded(held @ wd.abs() + (N + 3) * U32 * (dz.abs() + held) @ wd.abs(), dx, dtype))
        out["dw"] = (dw, rounded(held.t() @ xd.abs() + (M + 3) * U32 * (dz.abs() + held).t() @ xd.abs(), dw, dtype))
        out["db"] = (db, rounded(plain.sum(0) + (M + 3) * U32 * (dz.abs() + plain).sum(0), db, dtype))
    return out


def worst(got, ref):
    """The largest |got - value| over its bound (at most 1 where the evaluation is sound)."""
    value, bound = ref
    got = got.detach().cpu().double()
    assert got.shape == value.shape
    if got.numel() == 0:
        return 0.0
    off = (got - value).abs()
    assert torch.isfinite(off).all()
    return (off / bound.clamp(min=1e-300)).max().item()
