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


def balance(logits, mask, top_k, grad=1.0):
    """(loss, counts, dlogits), the floats with bounds; logits [T, E] on the CPU in their own type."""
    dtype, (T, E) = logits.dtype, logits.shape
    x = logits.double()
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.clone()
    keep &= (x > -math.inf).any(1)
    rows = x[keep]
    n = len(rows)
    counts = torch.zeros(E, dtype=torch.int64)
    for row in rows:  # the top_k largest, equal ones from the front, none at -inf
        order = sorted(range(E), key=lambda e: (-row[e].item(), e))[:top_k]
        for e in order:
            counts[e] += row[e].item() > -math.inf
    p = torch.softmax(rows, 1)
    spread = torch.where(rows > -math.inf, rows.max(1, keepdim=True).values - rows, torch.zeros_like(rows)).amax(
        1, keepdim=True) if n else torch.zeros(0, 1, dtype=torch.float64)
    relp = (2 * spread + E + 16) * U32
    f = counts.double() / (max(n, 1) * top_k)
    mean = p.sum(0) / max(n, 1)
    merr = (relp * p).sum(0) / max(n, 1) + (T / 2048 + 16) * U32 * mean
    loss = E * (f * mean).sum()
    lerr = E * (f * merr).sum() + 8 * U32 * loss
    d = torch.zeros(T, E, dtype=torch.float64)
    derr = torch.zeros(T, E, dtype=torch.float64)
    scale = abs(grad) * E / max(n, 1)
    dot = (f * p).sum(1, keepdim=True)
    d[keep] = grad * E / max(n, 1) * p * (f - dot)
    derr[keep] = scale * p * (2 * relp * (f - dot).abs() + (relp + (E + 8) * U32) * dot + 8 * U32 * f)
    return (loss, lerr + TINY[torch.float32]), counts, (d, torch.where(keep[:, None], rounded(derr, d, dtype), 0.0))


def distill(s, t, i, tau, weight=None):
    """loss [R] and ds [R, V] with bounds; inputs on the CPU."""
    dtype, (R, V), k = s.dtype, s.shape, t.shape[1]
    x, loss, lerr = s.double() / tau, torch.zeros(R, dtype=torch.float64), torch.zeros(R, dtype=torch.float64)
    ds, derr = torch.zeros(R, V, dtype=torch.float64), torch.zeros(R, V, dtype=torch.float64)
    w = torch.ones(R, dtype=torch.float64) if weight is None else weight.double()
    for r in range(R):
        full = (i[r] >= 0) & (i[r] < V) & (t[r].double() > -math.inf)
        if not full.any() or not (x[r] > -math.inf).any():
            continue
        tt, at = t[r][full].double() / tau, i[r][full].long()
        q, p = torch.softmax(tt, 0), torch.softmax(x[r], 0)
        logq, logp = torch.log_softmax(tt, 0), torch.log_softmax(x[r], 0)
        alive = x[r][x[r] > -math.inf]
        span = (alive.max() - alive.min()).item()
        relp = (4 * span + V / 64 + 24) * U32
        relq = (2 * (tt.max() - tt.min()).item() + k + 16) * U32
        used = q > 0
        terms = q[used] * (logq[used] - logp[at][used])
        loss[r] = tau * tau * terms.sum()
        size = (q[used] * (tt[used].abs() + tt.abs().max() + logq[used].abs() + x[r][at][used].abs())).sum()
        lerr[r] = tau * tau * (relq * size + (k + 16) * U32 * size + relp + 8 * U32 * (alive.abs().max() + math.log(V) + 1))
        each = torch.zeros(V, dtype=torch.float64).index_add_(0, at, q)
        ds[r] = w[r] * tau * (p - each)
        derr[r] = w[r].abs() * tau * (relp * p + relq * each + (k + 8) * U32 * (p + each))
    some = (derr != 0).any(1, keepdim=True)
    return (loss, lerr), (ds, torch.where(some, rounded(derr, ds, dtype), torch.zeros_like(derr)))
