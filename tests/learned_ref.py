"""The learned heads' operators in 64 bits on the CPU, from their definitions (include/splatx_hip.h), and the bounds
within which a 32-bit evaluation lies.

u is half a unit in the last place of 32 bits, 2^-24; UNIT has the types' (24, 8 and 11 significant bits). A sum of n values in any order that
chains at most k additions is within k u sum|values| of its own; the operators chain at most W / 32 + 16 of a row's W
(32 lanes or more share a row of over 32 values) and rows / 64 + 128 of a column's."""
import math

import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def norm_fwd(x, weight, bias, eps, residual=None):
    """(y, h, mean, rstd) and the bound of y's error, per element."""
    h = x.double()
    if residual is not None:
        h = (h + residual.double()).to(x.dtype).double()
    W = h.shape[-1]
    mean = h.sum(-1, keepdim=True) / W
    d = h - mean
    rstd = (d.square().sum(-1, keepdim=True) / W + eps).rsqrt()
    w = weight.double() if weight is not None else torch.ones(W, dtype=torch.float64)
    b = bias.double() if bias is not None else torch.zeros(W, dtype=torch.float64)
    y = d * rstd * w + b
    k = W / 32 + 16
    top = h.abs().amax(-1, keepdim=True)
    xhat = d * rstd
    # the mean is off by k u max|h|, a deviation by that and its own rounding, rstd by what the squares' sum chains
    bound = w.abs() * (k * U32 * top * rstd * (1 + xhat.abs()) + (k + 8) * U32 * xhat.abs()) + 2 * U32 * (y.abs() + b.abs())
    return y, h, mean.squeeze(-1), rstd.squeeze(-1), bound + UNIT[x.dtype] * y.abs() + TINY[x.dtype]


def norm_bwd(dy, h, mean, rstd, weight, dh=None):
    """(dx, dweight, dbias) and the bounds of their errors, for the mean and rstd given (floats, taken as they are). The
    bounds are those of the values in 32 bits: a rounding to a narrower type adds its own."""
    W, rows = h.shape[-1], h.numel() // h.shape[-1]
    dyd, hd, m, s = dy.double(), h.double(), mean.double()[..., None], rstd.double()[..., None]
    w = weight.double() if weight is not None else torch.ones(W, dtype=torch.float64)
    xhat = (hd - m) * s
    g = dyd * w
    mg, mgx = g.sum(-1, keepdim=True) / W, (g * xhat).sum(-1, keepdim=True) / W
    dx = s * (g - mg - xhat * mgx)
    # xhat is off by u of h - m and of itself
    off = 3 * U32 * xhat.abs()
    k = W / 32 + 16
    top_g, top_gx = g.abs().amax(-1, keepdim=True), (g * xhat).abs().amax(-1, keepdim=True)
    e = s * (4 * U32 * (g.abs() + mg.abs() + (xhat * mgx).abs()) + k * U32 * top_g + xhat.abs() * k * 2 * U32 * top_gx + off * mgx.abs() +
             xhat.abs() * 3 * U32 * top_gx)
    if dh is not None:
        dx = dx + dh.double()
    e = e + UNIT[h.dtype] * dx.abs() + TINY[h.dtype]
    chain = rows / 64 + 128
    flat = lambda t: t.reshape(rows, W).sum(0)  # noqa: E731
    return (dx, flat(dyd * xhat), flat(dyd)), (e, (chain + 4) * U32 * flat((dyd * xhat).abs()) + 1e-40,
                                               chain * U32 * flat(dyd.abs()) + 1e-40)


def _mix(h):
    h = h ^ (h >> 15)
    h = h * 0x6A09E667 & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = h * 0xBB67AE85 & 0xFFFFFFFF
    return h ^ (h >> 16)


def random_bits(seed, step, tensor, n):
    k = 0
    for word in (seed & 0xFFFFFFFF, seed >> 32, step & 0xFFFFFFFF, tensor):
        k = _mix((k + word * 0x9E3779B9) & 0xFFFFFFFF)
    return _mix((torch.arange(n, dtype=torch.int64) * 0x9E3779B9 + k) & 0xFFFFFFFF)


def code_values():
    """What each E4M3 byte stands for."""
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = math.nan if c & 127 == 127 else math.ldexp(1 + m / 8, e - 7) if e else math.ldexp(m / 8, -6)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def encode(x, bits, least):
    """(codes, scales) of x [n] in 64 bits."""
    n = x.numel()
    pad = -n % 256
    x = torch.nn.functional.pad(x, (0, pad)).view(-1, 256)
    bits = torch.nn.functional.pad(bits, (0, pad)).view(-1, 256)
    size = x.abs()
    finite = torch.isfinite(x)
    top = torch.where(finite, size, torch.zeros_like(size)).amax(1, keepdim=True)
    some = top >= 2.0 ** -100
    u = torch.where(some & finite, size * 448 / top.clamp_min(2.0 ** -120), torch.zeros_like(size))
    values = code_values()[:127]
    below = (torch.searchsorted(values, u.clamp_max(448), right=True) - 1).clamp(0, 125)
    frac = (u - values[below]) / (values[below + 1] - values[below])
    code = below + (frac + bits.double() / 65536 >= 1).long()
    if least:
        code = torch.where((size > 0) & some, code.clamp_min(1), code)
    code = torch.where(x < 0, code + 128, code)
    code = torch.where(finite, code, torch.full_like(code, 0x7F))
    return code.view(-1)[:n].to(torch.uint8), torch.where(some, top / 448, torch.zeros_like(top)).view(-1)


def decode(codes, scale):
    return code_values()[codes.long()] * scale.double().repeat_interleave(256)[:codes.numel()]


def adamw(p, g, m, v, *, step, lr, weight_decay, b1, b2, eps, scale=1.0):
    """(p, m, v) after a step, in 64 bits."""
    g = g.double() * scale
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    p = p.double() * (1 - lr * weight_decay) - lr / (1 - b1 ** step) * m / ((v / (1 - b2 ** step)).sqrt() + eps)
    return p, m, v
