"""The operators that train a learned head beside the splats, and the cases their speed is measured by.

- `ln_fwd`, `ln_bwd`: layer norm over [rows, width] features, one row per splat (or per ray, or per token of an image
  encoder), with the residual stream's addition before it and the gradient that reaches the sum past it.
- `grad_norm`: the 2-norm of every gradient of a model together.
- `adamw32`, `adamw8`: one AdamW step over many tensors, the moments held in 32 bits or in 8 with a scale per 256 elements.

Three layouts of tensors: `groups`, a cloud's six parameter groups; `head`, a small network's weights, biases and norms;
`flat`, tensors of odd sizes one after another in one buffer, as a program has them that keeps a model's parameters together.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "splatx-metal_amd", "python"))

own = False  # False: elementary torch operations in 32 bits; True: the framework's entry points

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
LN_EPS = 1e-5
BETAS = (0.9, 0.999)
ADAM_EPS = 1e-8
STEP = 1000        # steps taken so far, this one included
MAX_NORM = 1.0
BLOCK = 256        # elements that share a scale
GROUP_DIMS = (3, 4, 3, 1, 3, 45)                             # means, quats, scales, opacities, sh0, shN at degree 3
GROUP_LR = (1.6e-4, 1e-3, 5e-3, 5e-2, 2.5e-3, 1.25e-4)      # the trainer's rates


def listed():
    return [
        # a few thousand points of a first look at a capture, their 45 higher SH coefficients: a call's latency
        dict(name="ln_fwd_2k_45", kind="ln_fwd", rows=2000, width=45, type="f32", wtype="f32", add=False, pad=0),
        # a head's first norm over every splat of a full scene, on the 48 SH coefficients
        dict(name="ln_fwd_1m_48", kind="ln_fwd", rows=1_000_000, width=48, type="bf16", wtype="f32", add=False, pad=0),
        # an image encoder's tokens in a residual stream of rows longer than a wave's registers
        dict(name="ln_fwd_16k_2048_add", kind="ln_fwd", rows=16_383, width=2048, type="f16", wtype="same", add=True, pad=0),
        # the same three backward: the small head, every splat's 64 hidden features with a skip path, the encoder
        dict(name="ln_bwd_2k_45", kind="ln_bwd", rows=2000, width=45, type="f32", wtype="f32", add=False, pad=0),
        dict(name="ln_bwd_1m_64_add", kind="ln_bwd", rows=1_000_000, width=64, type="bf16", wtype="f32", add=True, pad=0),
        dict(name="ln_bwd_16k_2048", kind="ln_bwd", rows=16_383, width=2048, type="f16", wtype="same", add=False, pad=0),
        # a small head's ten gradients, and those of a full scene's cloud
        dict(name="norm_head_64", kind="grad_norm", layout="head", n=64, ptype="f32", gtype="bf16", clip=False),
        dict(name="norm_groups_1m", kind="grad_norm", layout="groups", n=1_000_000, ptype="f32", gtype="f32", clip=False),
        # the step of a small head in bf16 with its f32 master weights, clipped; of a full scene's cloud
        dict(name="adamw32_head_64", kind="adamw32", layout="head", n=64, ptype="bf16", gtype="bf16", clip=True),
        dict(name="adamw32_groups_1m", kind="adamw32", layout="groups", n=1_000_000, ptype="f32", gtype="f32", clip=False),
        # moments in 8 bits: odd tensors in one buffer, and the largest cloud of the benchmark's configurations
        dict(name="adamw8_flat_300k", kind="adamw8", layout="flat", n=300_007, ptype="f32", gtype="f32", clip=True),
        dict(name="adamw8_groups_2m", kind="adamw8", layout="groups", n=2_000_000, ptype="f32", gtype="f32", clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("ln_fwd", "ln_bwd", "ln_fwd", "ln_bwd", "grad_norm", "adamw32", "adamw8"))
    if kind.startswith("ln"):
        width = _log(rng, 4, 6000)
        rows = _log(rng, 1, min(1_200_000, 64_000_000 // width))
        return dict(kind=kind, rows=rows, width=width, type=rng.choice(("f32", "bf16", "f16")),
                    wtype=rng.choice(("f32", "same")), add=rng.random() < 0.4, pad=rng.choice((0, 0, 0, 1, 8)))
    layout = rng.choice(("groups", "head", "flat"))
    n = {"groups": (300, 1_500_000), "head": (8, 900), "flat": (50, 40_000_000)}[layout]
    ptype = "f32" if layout == "groups" else rng.choice(("f32", "bf16", "f16"))
    gtype = ptype if rng.random() < 0.7 else rng.choice(("f32", "bf16"))
    return dict(kind=kind, layout=layout, n=_log(rng, *n), ptype=ptype, gtype=gtype, clip=rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------------------------------

def _sizes(case):
    n = case["n"]
    if case["layout"] == "groups":
        return [n * d for d in GROUP_DIMS]
    if case["layout"] == "head":  # norm, linear, norm, linear, linear to a colour; 48 features in, n hidden
        return [48, 48, 48 * n, n, n, n, n * n, n, 3 * n, 3]
    return [max(1, int(n * w)) | 1 for w in (0.31, 0.002, 0.17, 0.0003, 0.25, 0.0, 0.2, 0.06)]


def _rates(case):
    """(learning rate, weight decay) of each tensor."""
    if case["layout"] == "groups":
        return [(lr, 0.0) for lr in GROUP_LR]
    return [(1e-3, 0.01 if n > 1000 else 0.0) for n in _sizes(case)]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _prepare_ln(case, seed):
    g = _generator(seed)
    rows, width, t = case["rows"], case["width"], TYPES[case["type"]]
    wt = torch.float32 if case["wtype"] == "f32" else t

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def held(v):  # rows of a wider buffer where the case has padding between them
        buf = torch.zeros(rows, width + case["pad"], device="cuda", dtype=t)
        buf[:, :width] = v
        return buf[:, :width]

    # features of rows of differing spread about the columns' means; every 97th row all zero: a splat out of view
    size = torch.exp(0.5 * normal(rows, 1))
    x = size * (normal(rows, width) + 0.5 * normal(width))
    x[96::97] = 0
    s = dict(case=case, weight=(1 + 0.1 * normal(width)).to(wt), bias=(0.1 * normal(width)).to(wt))
    if case["kind"] == "ln_fwd":
        s["x"] = held(x)
        if case["add"]:
            s["residual"] = held(0.5 * size * normal(rows, width))
        return s
    s["h"] = held(x)
    h = s["h"].double()
    mean = h.mean(1)
    s["mean"] = mean.float()
    s["rstd"] = (1 / torch.sqrt(((h - mean[:, None]) ** 2).mean(1) + LN_EPS)).float()
    dy = 1e-2 * normal(rows, width)
    dy[95::96] = 0
    s["dy"] = held(dy)
    if case["add"]:
        s["dh"] = held(1e-2 * normal(rows, width))
    return s


def _prepare_tensors(case, seed):
    g = _generator(seed)
    sizes, pt, gt = _sizes(case), TYPES[case["ptype"]], TYPES[case["gtype"]]
    total = sum(sizes)

    def split(buf):
        if case["layout"] == "flat":
            return list(buf.split(sizes))
        return [x.clone() for x in buf.split(sizes)]

    def normal():
        return torch.randn(total, device="cuda", generator=g)

    # a gradient of norm 1.5 that is zero for one row in twenty, in half precision 1024 times itself (the loss is scaled)
    scaled = 1024.0 if gt == torch.float16 else 1.0
    seen = torch.rand(total, device="cuda", generator=g) > 0.05
    typical = 1.5 / math.sqrt(total)
    grad = typical * scaled * torch.where(seen, normal(), torch.zeros((), device="cuda"))
    s = dict(case=case, grad=split(grad.to(gt)), grad_scale=1.0 / scaled)
    if case["kind"] == "grad_norm":
        return s
    param = 0.5 * normal()
    s["param"] = split(param.to(pt))
    if pt != torch.float32:
        s["master"] = split(param)
    if case["clip"]:
        s["norm"] = torch.stack([x.double().square().sum() for x in s["grad"]]).sum().sqrt().float()
    m = 0.3 * typical * torch.where(seen, normal(), torch.zeros((), device="cuda"))
    v = torch.where(seen, (typical * torch.exp(0.7 * normal())) ** 2, torch.zeros((), device="cuda"))
    if case["kind"] == "adamw32":
        s["exp_avg"], s["exp_avg_sq"] = split(m), split(v)
        return s
    s["seed"] = 12345 + seed
    for name, x in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
        codes, scales = [], []
        for p in split(x):
            blocks = _blocks(p)
            scale = blocks.abs().amax(1) / 448
            codes.append((blocks / scale.clamp_min(1e-30)[:, None]).reshape(-1)[:p.numel()].to(torch.float8_e4m3fn))
            scales.append(scale)
        s[name], s[name + "_scale"] = codes, scales
    return s


def prepare(case, seed):
    return (_prepare_ln if case["kind"].startswith("ln") else _prepare_tensors)(case, seed)


# ---- plain forms ------------------------------------------------------------------------------------------

def _ln_fwd(s):
    x = s["x"]
    h = (x.float() + s["residual"].float()).to(x.dtype) if "residual" in s else x
    hf = h.float()
    mean = hf.mean(1)
    d = hf - mean[:, None]
    rstd = torch.rsqrt((d * d).mean(1) + LN_EPS)
    y = (d * rstd[:, None] * s["weight"].float() + s["bias"].float()).to(x.dtype)
    return dict(y=y, mean=mean, rstd=rstd, **({"h": h} if "residual" in s else {}))


def _ln_bwd(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["h"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if "dh" in s:
        dx = dx + s["dh"].float()
    return dict(dx=dx.to(s["h"].dtype), dweight=(dy * xhat).sum(0).to(s["weight"].dtype), dbias=dy.sum(0).to(s["weight"].dtype))


def _grad_norm(s):
    return torch.stack([(x * x).sum() for x in (g.float() for g in s["grad"])]).sum().sqrt()


def _clip(s):
    """What a gradient is multiplied by. (The norms of the cases are finite: every step is taken.)"""
    if "norm" not in s:
        return s["grad_scale"]
    n = s["norm"] * s["grad_scale"]
    return s["grad_scale"] * torch.where(n > MAX_NORM, MAX_NORM / n, torch.ones_like(n))


def _update(s, param, m, v):
    """p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps) in place, lists of tensors."""
    c1, c2 = 1 - BETAS[0] ** STEP, 1 - BETAS[1] ** STEP
    denom = torch._foreach_sqrt(v)
    torch._foreach_div_(denom, math.sqrt(c2))
    torch._foreach_add_(denom, ADAM_EPS)
    step = torch._foreach_div(m, denom)
    rates = _rates(s["case"])
    torch._foreach_mul_(step, [-lr / c1 for lr, _ in rates])
    torch._foreach_mul_(param, [1 - lr * wd for lr, wd in rates])
    torch._foreach_add_(param, step)


def _moments(s, m, v):
    g = torch._foreach_mul([x.float() for x in s["grad"]], _clip(s))
    torch._foreach_mul_(m, BETAS[0])
    torch._foreach_add_(m, g, alpha=1 - BETAS[0])
    torch._foreach_mul_(v, BETAS[1])
    torch._foreach_add_(v, torch._foreach_mul(g, g), alpha=1 - BETAS[1])
    _update(s, s.get("master", s["param"]), m, v)
    if "master" in s:
        torch._foreach_copy_(s["param"], s["master"])


def _adamw32(s):
    _moments(s, s["exp_avg"], s["exp_avg_sq"])
    return _outputs(s)


def _outputs(s):
    return {k: s[k] for k in ("param", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale") if k in s}


def _blocks(x):
    """[blocks, 256] of a tensor's elements in order, zeros after its end."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _mix(h):
    """32 bits to 32 bits, each depending on all; whole numbers or tensors of them."""
    h = h ^ (h >> 15)
    h = h * 0x6A09E667 & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = h * 0xBB67AE85 & 0xFFFFFFFF
    return h ^ (h >> 16)


def _key(seed, tensor):
    k = 0
    for word in (seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF, STEP & 0xFFFFFFFF, tensor):
        k = _mix((k + word * 0x9E3779B9) & 0xFFFFFFFF)
    return k


def _random(seed, tensor, n):
    """32 random bits for each element of the step's tensor."""
    return _mix((torch.arange(n, device="cuda") * 0x9E3779B9 + _key(seed, tensor)) & 0xFFFFFFFF)


def _encode(x, bits, least):
    """E4M3 codes and scales of x: |x| in units of its block's maximum / 448, rounded up to the next code with the
    probability of what lies above the code below (16 random bits); `least`: what is not zero gets code 1 at least."""
    n = x.numel()
    blocks, bits = _blocks(x), _blocks(bits)
    size = blocks.abs()
    top = size.amax(1, keepdim=True)
    some = top >= 2.0 ** -100  # smaller ones count as zero
    u = torch.where(some, size * (448.0 / top), torch.zeros_like(size)).clamp_max(448.0)
    low = u < 2.0 ** -6  # below the least normal code the codes are 2^-9 apart
    t = torch.where(low, u + 2.0 ** -6, u).view(torch.int32)
    code = ((t + (bits << 4).int()) >> 20) - torch.where(low, 968, 960)
    if least:
        code = torch.where((size > 0) & some, code.clamp_min(1), code)
    code = torch.where(blocks < 0, code + 128, code)
    scale = torch.where(some, top / 448.0, torch.zeros_like(top))
    return code.to(torch.uint8).view(-1)[:n].view(torch.float8_e4m3fn), scale.view(-1)


def _decode(code, scale):
    return (_blocks(code.float()) * scale[:, None]).view(-1)[:code.numel()]


def _adamw8(s):
    m = [_decode(c, k) for c, k in zip(s["exp_avg"], s["exp_avg_scale"])]
    root = [_decode(c, k) for c, k in zip(s["exp_avg_sq"], s["exp_avg_sq_scale"])]
    v = torch._foreach_mul(root, root)
    _moments(s, m, v)
    bits = [_random(s["seed"], i, x.numel()) for i, x in enumerate(m)]
    new = [_encode(x, b & 0xFFFF, False) for x, b in zip(m, bits)]
    root = [_encode(x.sqrt(), b >> 16, True) for x, b in zip(v, bits)]
    s["exp_avg"], s["exp_avg_scale"] = [c for c, _ in new], [k for _, k in new]
    s["exp_avg_sq"], s["exp_avg_sq_scale"] = [c for c, _ in root], [k for _, k in root]
    return _outputs(s)


PLAIN = {"ln_fwd": _ln_fwd, "ln_bwd": _ln_bwd, "grad_norm": _grad_norm, "adamw32": _adamw32, "adamw8": _adamw8}


# ---- the framework's ----------------------------------------------------------------------------------------

_backend = None


def _get_backend():
    global _backend
    if _backend is None:
        import splatx_torch

        _backend = splatx_torch.TorchBackend(0)
    return _backend


def _own_ln_fwd(s):
    y, h, mean, rstd = _get_backend().layer_norm_fwd(s["x"], s["weight"], s["bias"], eps=LN_EPS, residual=s.get("residual"))
    return dict(y=y, mean=mean, rstd=rstd, **({"h": h} if "residual" in s else {}))


def _own_ln_bwd(s):
    dx, dweight, dbias = _get_backend().layer_norm_bwd(s["dy"], s["h"], s["mean"], s["rstd"], s["weight"], dh=s.get("dh"))
    return dict(dx=dx, dweight=dweight, dbias=dbias)


def _own_grad_norm(s):
    return _get_backend().grad_norm(s["grad"])


def _own_adamw(s):
    rates = _rates(s["case"])
    more = dict(exp_avg_scale=s["exp_avg_scale"], exp_avg_sq_scale=s["exp_avg_sq_scale"], seed=s["seed"]) if "seed" in s else {}
    _get_backend().adamw_step(s["param"], s["grad"], s["exp_avg"], s["exp_avg_sq"], step=STEP, lr=[lr for lr, _ in rates],
                              weight_decay=[wd for _, wd in rates], b1=BETAS[0], b2=BETAS[1], eps=ADAM_EPS,
                              master=s.get("master"), grad_scale=s["grad_scale"], grad_norm=s.get("norm"),
                              max_norm=MAX_NORM if "norm" in s else 0.0, **more)
    return _outputs(s)


OWN = {"ln_fwd": _own_ln_fwd, "ln_bwd": _own_ln_bwd, "grad_norm": _own_grad_norm, "adamw32": _own_adamw, "adamw8": _own_adamw}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------

def work(case):
    if case["kind"].startswith("ln"):
        n, b = case["rows"] * case["width"], SIZE[case["type"]]
        wb = 4 if case["wtype"] == "f32" else b
        if case["kind"] == "ln_fwd":  # x (residual) in, y (h) and the statistics out
            return dict(bytes=n * b * (4 if case["add"] else 2) + 8 * case["rows"] + 2 * wb * case["width"], flops=8 * n)
        return dict(bytes=n * b * (4 if case["add"] else 3) + 8 * case["rows"] + 3 * wb * case["width"], flops=14 * n)
    n, g = sum(_sizes(case)), SIZE[case["gtype"]]
    if case["kind"] == "grad_norm":
        return dict(bytes=n * g, flops=2 * n)
    each = g + 8 + (SIZE[case["ptype"]] if case["ptype"] != "f32" else 0)
    if case["kind"] == "adamw32":
        return dict(bytes=n * (each + 16), flops=14 * n)
    return dict(bytes=n * (each + 4) + 16 * sum(-(-k // BLOCK) for k in _sizes(case)), flops=30 * n)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def _exact_ln(case, s):
    w = s["weight"].double()
    if case["kind"] == "ln_fwd":
        h = s["x"].double()
        if case["add"]:  # the sum is an output of the input's type, and what is normalised
            h = (h + s["residual"].double()).to(s["x"].dtype).double()
        mu = h.sum(1, keepdim=True) / case["width"]
        inv = ((h - mu).square().sum(1, keepdim=True) / case["width"] + LN_EPS).pow(-0.5)
        out = dict(y=(h - mu) * inv * w + s["bias"].double(), mean=mu[:, 0], rstd=inv[:, 0])
        return dict(out, h=h) if case["add"] else out
    dy, inv = s["dy"].double(), s["rstd"].double()[:, None]
    xhat = (s["h"].double() - s["mean"].double()[:, None]) * inv
    dxhat = dy * w
    # dx = s (I - 1 1^T / W - xhat xhat^T / W) dxhat
    dx = inv * (dxhat - (dxhat.sum(1, keepdim=True) + xhat * (dxhat * xhat).sum(1, keepdim=True)) / case["width"])
    return dict(dx=dx + s["dh"].double() if case["add"] else dx, dweight=(dy * xhat).sum(0), dbias=dy.sum(0))


def _exact_codes(x, bits, least):
    n = x.numel()
    x, bits = _blocks(x), _blocks(bits)
    top = x.abs().amax(1, keepdim=True)
    scale = top / 448
    u = x.abs() / torch.where(top > 0, scale, torch.ones_like(scale))
    apart = torch.exp2(torch.floor(torch.log2(u.clamp_min(2.0 ** -6))) - 3)  # between the codes about u
    q = (torch.floor(u / apart + bits.double() / 65536) * apart).clamp_max(448)
    if least:
        q = torch.where(x > 0, q.clamp_min(2.0 ** -9), q)
    return (q * x.sign()).reshape(-1)[:n], scale.reshape(-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("ln"):
        return _exact_ln(case, s)
    if case["kind"] == "grad_norm":
        return sum(g.double().square().sum() for g in s["grad"]).sqrt()
    out = dict(param=[], exp_avg=[], exp_avg_sq=[])
    if "master" in s:
        out["master"] = []
    eight = case["kind"] == "adamw8"
    if eight:
        out.update(exp_avg_scale=[], exp_avg_sq_scale=[])
    scale = s["grad_scale"]
    if case["clip"]:
        scale *= min(1.0, MAX_NORM / (scale * s["norm"].double().item()))
    for i, (lr, wd) in enumerate(_rates(case)):
        g = s["grad"][i].double() * scale
        m, v = s["exp_avg"][i].double(), s["exp_avg_sq"][i].double()
        if eight:
            m = (_blocks(m) * s["exp_avg_scale"][i].double()[:, None]).reshape(-1)[:g.numel()]
            v = (_blocks(v) * s["exp_avg_sq_scale"][i].double()[:, None]).reshape(-1)[:g.numel()].square()
        m = BETAS[0] * m + (1 - BETAS[0]) * g
        v = BETAS[1] * v + (1 - BETAS[1]) * g * g
        p = (s["master"] if "master" in s else s["param"])[i].double()
        p = p - lr * wd * p - lr * (m / (1 - BETAS[0] ** STEP)) / ((v / (1 - BETAS[1] ** STEP)).sqrt() + ADAM_EPS)
        out["param"].append(p)
        if "master" in s:
            out["master"].append(p)
        if eight:
            bits = _random(s["seed"], i, g.numel())
            m, sm = _exact_codes(m, bits & 0xFFFF, False)
            v, sv = _exact_codes(v.sqrt(), bits >> 16, True)
            out["exp_avg_scale"].append(sm)
            out["exp_avg_sq_scale"].append(sv)
        out["exp_avg"].append(m)
        out["exp_avg_sq"].append(v)
    return out
