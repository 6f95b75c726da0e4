"""Linear layers in 64 bits, from their definitions (include/splatx_hip.h), and the bounds within which a 32-bit evaluation of
them lies.

u is 2^-24, half a unit in the last place of 32 bits. Products of two 16-bit elements are exact in 32 bits, those of floats are
off by u. A sum of n terms in any order is within n u sum|terms|; twice that is allowed, as the matrix cores add a step's
products without saying how. An activation's own error is ACT relative to the largest of it and its argument: for floats what
the library's exponential, error function and quotient add up to (16 u), for 16-bit outputs that of Phi(-|z|), 2.5e-5 relative
with at most half of |z| before it, and of the hardware's exponential and reciprocal, 2^-22 each and the argument's rounding.
A slope has the same. dz may be rounded to the type before the products: UNIT |dz|."""
import math

import torch

from learned_ref import TINY, U32, UNIT

ACTS = ("none", "relu", "gelu", "silu", "sigmoid")
DZ_UNIT = {}  # of dz before the products, where it is not UNIT
ACT = {torch.float32: 16 * U32, torch.bfloat16: 4e-5, torch.float16: 4e-5}


def below(z):
    """Phi. (As 1 + erf it would lose the tail, 64 bits or not.)"""
    return 0.5 * torch.special.erfc(-z * math.sqrt(0.5))


def act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "gelu":
        return z * below(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    return torch.sigmoid(z) if name == "sigmoid" else z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return below(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    p = torch.sigmoid(z)
    if name == "silu":
        return p + z * p * torch.sigmoid(-z)
    return p * torch.sigmoid(-z) if name == "sigmoid" else torch.ones_like(z)


def parts(rows, ends):
    """(weight's index, rows) of each group."""
    if ends is None:
        return [((), slice(0, rows))]
    ends = [int(e) for e in ends]
    return [((i,), slice(a, e)) for i, (a, e) in enumerate(zip([0] + ends[:-1], ends))]


def fwd(x, w, b, name="none", residual=None, ends=None):
    """(y, pre) and the bounds of their errors."""
    rows, t, depth = x.shape[0], x.dtype, x.shape[1]
    out = torch.zeros(4, rows, w.shape[-2], dtype=torch.float64, device=x.device)
    for i, r in parts(rows, ends):
        xd, wd = x[r].double(), w[i].double()
        bias = b[i].double() if b is not None else torch.zeros(w.shape[-2], dtype=torch.float64, device=x.device)
        z = xd @ wd.t().contiguous() + bias
        off = 2 * (depth + 2) * U32 * (xd.abs() @ wd.abs().t().contiguous() + bias.abs())
        y = act(z, name)
        # no slope is steeper than 1.13
        off_y = 1.13 * off + (ACT[t] * torch.maximum(y.abs(), z.abs().clamp_max(8)) if name not in ("none", "relu") else 0)
        if residual is not None:
            rd = residual[r].double()
            off_y = off_y + 2 * U32 * (y.abs() + rd.abs())
            y = y + rd
        out[0, r], out[1, r] = y, off_y + UNIT[t] * (y.abs() + off_y) + TINY[t]
        out[2, r], out[3, r] = z, off + UNIT[t] * (z.abs() + off) + TINY[t]
    return (out[0], out[2]), (out[1], out[3])


def bwd(dy, x, w, pre=None, name="none", ends=None):
    """(dx, dweight, dbias) and the bounds of their errors."""
    rows, t, n = x.shape[0], x.dtype, w.shape[-2]
    new = lambda s: torch.zeros(2, *s, dtype=torch.float64, device=x.device)  # noqa: E731
    dx, dw, db = new(x.shape), new(w.shape), new(w.shape[:-1])
    for i, r in parts(rows, ends):
        d, xd, wd = dy[r].double(), x[r].double(), w[i].double()
        off = torch.zeros_like(d)
        if name != "none":
            z = pre[r].double()
            if name != "relu":
                off = d.abs() * ACT[t] * (1 + z.abs().clamp_max(8))
            d = d * slope(z, name)
        size, m = d.abs() + off, d.shape[0]
        rounded = off + DZ_UNIT.get(t, UNIT[t]) * size + TINY[t]
        final = lambda v, e: torch.stack([v, e + UNIT[t] * (v.abs() + e) + TINY[t]])  # noqa: E731
        dx[:, r] = final(d @ wd, rounded @ wd.abs() + 2 * (n + 2) * U32 * (size @ wd.abs()))
        dw[(slice(None), *i)] = final(d.t().contiguous() @ xd, rounded.t().contiguous() @ xd.abs() + 2 * (m + 2) * U32 * (size.t().contiguous() @ xd.abs()))
        db[(slice(None), *i)] = final(d.sum(0), off.sum(0) + 2 * (m + 2) * U32 * size.sum(0))
    return (dx[0], dw[0], db[0]), (dx[1], dw[1], db[1])
