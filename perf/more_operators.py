"""The layers of a learned head beside the splats, and the cases their speed is measured by.

- `fwd`: y = act(x W^T + bias) + residual over [rows, features], one row per splat (or per token of an image encoder); for
  training also `pre`, x W^T + bias as the backward reads it.
- `bwd`: its gradients dx, dweight, dbias from dy, x, the weight and `pre`.
- `grouped_fwd`, `grouped_bwd`: the same where the rows come in groups of any sizes with weights of their own, as a scene cut
  into cells has a head for each, or a batch of several photographs an own layer for each.
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
ACTS = ("none", "relu", "gelu", "silu", "sigmoid")
MOST_FLOPS = 5e11   # of a drawn case (in 32 bits a tenth)
MOST_BYTES = 1.2e9


def listed():
    base = dict(type="bf16", act="none", bias=True, add=False, pad=0, train=False, groups=0, behind=0)
    return [dict(base, **c) for c in (
        # an image's embedding into a head's hidden features: one row, a call's latency
        dict(name="fwd_1_16_64", kind="fwd", rows=1, n_in=16, n_out=64, bias=False),
        # a head's first layer over every splat of a full scene
        dict(name="fwd_1m_48_64", kind="fwd", rows=1_000_000, n_in=48, n_out=64),
        # a hidden layer of it in training
        dict(name="fwd_1m_64_64_gelu", kind="fwd", rows=1_000_000, n_in=64, n_out=64, act="gelu", train=True),
        # an image encoder asked for a few tokens: its weights' bytes
        dict(name="fwd_9_2048_8192", kind="fwd", rows=9, n_in=2048, n_out=8192, type="f16", act="silu"),
        # its layer back into the residual stream over all tokens
        dict(name="fwd_16k_8192_2048_add", kind="fwd", rows=16_383, n_in=8192, n_out=2048, type="f16", add=True),
        # a first look at a capture: a few thousand points' 45 higher SH coefficients
        dict(name="bwd_2k_45_64", kind="bwd", rows=2000, n_in=45, n_out=64, type="f32", act="relu"),
        # the full scene's hidden layer, the encoder's
        dict(name="bwd_1m_64_64_gelu", kind="bwd", rows=1_000_000, n_in=64, n_out=64, act="gelu"),
        dict(name="bwd_16k_2048_4096_gelu", kind="bwd", rows=16_383, n_in=2048, n_out=4096, type="f16", act="gelu"),
        # a layer for each of a scene's cells; a wider one of a few large groups
        dict(name="grouped_fwd_1m_64_64", kind="grouped_fwd", rows=1_000_000, n_in=64, n_out=64, act="relu", train=True, groups=200,
             behind=1000),
        dict(name="grouped_fwd_20k_1024_1408", kind="grouped_fwd", rows=20_001, n_in=1024, n_out=1408, act="silu", groups=16),
        # the same backward, the cells' in 32 bits
        dict(name="grouped_bwd_300k_48_64", kind="grouped_bwd", rows=300_000, n_in=48, n_out=64, type="f32", act="relu", groups=200,
             behind=1000),
        dict(name="grouped_bwd_20k_1024_1408", kind="grouped_bwd", rows=20_001, n_in=1024, n_out=1408, act="silu", groups=16),
    )]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("fwd", "bwd", "grouped_fwd", "grouped_bwd"))
    t = rng.choice(("f32", "bf16", "bf16", "f16"))
    form = rng.choice(("head", "head", "encoder", "few"))  # narrow layers of many rows, wide ones, wide ones of few rows
    if form == "head":
        n_in, n_out, most = _log(rng, 3, 300), _log(rng, 1, 300), 1_200_000
    else:
        n_in, n_out, most = _log(rng, 200, 8192), _log(rng, 200, 8192), 40 if form == "few" else 30_000
    if rng.random() < 0.5:  # most layers have widths of whole vectors
        n_in, n_out = -(-n_in // 16) * 16, -(-n_out // 16) * 16
    products = (2 if kind.endswith("bwd") else 1)
    most = min(most, MOST_FLOPS * (0.1 if t == "f32" else 1) / (2 * n_in * n_out * products), MOST_BYTES / (SIZE[t] * (n_in + 2 * n_out)))
    rows = _log(rng, 1, max(most, 2))
    groups = behind = 0
    if kind.startswith("grouped"):
        groups = _log(rng, 1, max(2, min(256, MOST_BYTES / 4 / (SIZE[t] * n_in * n_out))))
        behind = rng.choice((0, 0, rows // 10))
    act = rng.choice(ACTS)
    fwd = kind.endswith("fwd")
    return dict(kind=kind, rows=rows, n_in=n_in, n_out=n_out, type=t, act=act, bias=rng.random() < 0.8, add=fwd and rng.random() < 0.3,
                pad=rng.choice((0, 0, 0, 1, 8)), train=fwd and act != "none" and rng.random() < 0.5, groups=groups, behind=behind)


# ---- inputs --------------------------------------------------------------------------------------------

def _sizes(case, seed):
    """Rows of each group: a few large ones, many small ones, one in ten of none."""
    g = torch.Generator().manual_seed(seed)
    n, rows = case["groups"], case["rows"] - case["behind"]
    share = torch.exp(1.2 * torch.randn(n, generator=g)) * (torch.rand(n, generator=g) > 0.1)
    share[int(torch.randint(n, (1,), generator=g))] += 0.5
    ends = torch.round(torch.cumsum(share.double(), 0) / share.double().sum() * rows).long()
    return torch.diff(ends, prepend=torch.zeros(1, dtype=torch.long)).tolist()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, n_in, n_out, t, pad = case["rows"], case["n_in"], case["n_out"], TYPES[case["type"]], case["pad"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def held(v):  # rows of a wider buffer where the case has padding between them
        if not pad:
            return v.to(t)
        buf = torch.zeros(v.shape[0], v.shape[1] + pad, device="cuda", dtype=t)
        buf[:, :v.shape[1]] = v
        return buf[:, :v.shape[1]]

    # normalised features, a layer's weights as they are initialised and learned; every 97th row is a splat out of view
    x = normal(rows, n_in)
    x[96::97] = 0
    lead = (case["groups"],) if case["groups"] else ()
    s = dict(case=case, x=held(x), weight=(normal(*lead, n_out, n_in) / math.sqrt(n_in)).to(t))
    if case["bias"]:
        s["bias"] = (0.1 * normal(*lead, n_out)).to(t)
    if case["groups"]:
        s["sizes"] = _sizes(case, seed)
        s["ends"] = torch.cumsum(torch.tensor(s["sizes"], device="cuda"), 0)
    if case["kind"].endswith("fwd"):
        if case["add"]:
            s["residual"] = held(normal(rows, n_out))
        return s
    dy = 1e-2 * normal(rows, n_out)
    dy[95::96] = 0
    s["dy"] = held(dy)
    if case["act"] != "none":
        s["pre"] = held(normal(rows, n_out))
    return s


# ---- plain forms ------------------------------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return torch.sigmoid(z) if act == "sigmoid" else z


def _slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    p = torch.sigmoid(z)
    return p * (1 + z * (1 - p)) if act == "silu" else p * (1 - p)


def _plain_fwd(s):
    case, t = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    bias = s["bias"].float() if "bias" in s else None
    if case["groups"]:
        z = torch.zeros(case["rows"], case["n_out"], device="cuda")
        at = 0
        for i, n in enumerate(s["sizes"]):
            if n:
                z[at:at + n] = x[at:at + n] @ w[i].t()
                if bias is not None:
                    z[at:at + n] += bias[i]
            at += n
    else:
        at = case["rows"]
        z = x @ w.t()
        if bias is not None:
            z += bias
    y = _act(z, case["act"])
    if "residual" in s:
        y = y + s["residual"].float()
    y[at:] = 0  # the rows of no group
    return dict(y=y.to(t), **({"pre": z.to(t)} if case["train"] else {}))


def _plain_bwd(s):
    case, t = s["case"], s["x"].dtype
    x, w, dz = s["x"].float(), s["weight"].float(), s["dy"].float()
    if case["act"] != "none":
        dz = dz * _slope(s["pre"].float(), case["act"])
    if not case["groups"]:
        out = dict(dx=dz @ w, dweight=dz.t() @ x, dbias=dz.sum(0))
    else:
        out = dict(dx=torch.zeros(case["rows"], case["n_in"], device="cuda"), dweight=torch.zeros_like(w), dbias=torch.zeros_like(w[:, :, 0]))
        at = 0
        for i, n in enumerate(s["sizes"]):
            if n:
                d = dz[at:at + n]
                out["dx"][at:at + n] = d @ w[i]
                out["dweight"][i] = d.t() @ x[at:at + n]
                out["dbias"][i] = d.sum(0)
            at += n
    if not case["bias"]:
        del out["dbias"]
    return {k: v.to(t) for k, v in out.items()}


# ---- the framework's ----------------------------------------------------------------------------------------

_backend = None


def _get_backend():
    global _backend
    if _backend is None:
        import splatx_torch

        _backend = splatx_torch.TorchBackend(0)
    return _backend


def _own_fwd(s):
    b, case = _get_backend(), s["case"]
    more = dict(activation=case["act"], residual=s.get("residual"), want_pre=case["train"])
    if case["groups"]:
        y, pre = b.grouped_linear_fwd(s["x"], s["weight"], s["ends"], s.get("bias"), **more)
    else:
        y, pre = b.linear_fwd(s["x"], s["weight"], s.get("bias"), **more)
    return dict(y=y, **({"pre": pre} if case["train"] else {}))


def _own_bwd(s):
    b, case = _get_backend(), s["case"]
    more = dict(pre=s.get("pre"), activation=case["act"], want_dbias=case["bias"])
    if case["groups"]:
        dx, dweight, dbias = b.grouped_linear_bwd(s["dy"], s["x"], s["weight"], s["ends"], **more)
    else:
        dx, dweight, dbias = b.linear_bwd(s["dy"], s["x"], s["weight"], **more)
    return dict(dx=dx, dweight=dweight, **({"dbias": dbias} if case["bias"] else {}))


def run(state):
    if state["case"]["kind"].endswith("fwd"):
        return (_own_fwd if own else _plain_fwd)(state)
    return (_own_bwd if own else _plain_bwd)(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------

def work(case):
    rows, n_in, n_out, b = case["rows"] - case["behind"], case["n_in"], case["n_out"], SIZE[case["type"]]
    each, groups = n_out * n_in + (n_out if case["bias"] else 0), max(1, case["groups"])
    read = min(groups, rows) * each + 8 * case["groups"] // b  # of groups without rows nothing is read
    if case["kind"].endswith("fwd"):  # x (residual) in, y (pre) out
        written = case["rows"] * n_out * (1 + case["train"])
        return dict(bytes=b * (rows * (n_in + n_out * case["add"]) + read + written), flops=2 * rows * n_in * n_out)
    acts = case["act"] != "none"
    return dict(bytes=b * (rows * (n_in + n_out * (1 + acts)) + read + case["rows"] * n_in + groups * each), flops=4 * rows * n_in * n_out)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------

def _parts(case, s):
    """(weight's index, rows) of each group that has some."""
    if not case["groups"]:
        return [((), slice(0, case["rows"]))]
    ends = s["ends"].tolist()
    return [((i,), slice(a, e)) for i, (a, e) in enumerate(zip([0] + ends[:-1], ends)) if e > a]


def exact(case, seed):
    s = prepare(case, seed)
    act, x = case["act"], s["x"]
    normal_below = lambda z: torch.special.ndtr(z)  # noqa: E731
    if case["kind"].endswith("fwd"):
        y = torch.zeros(case["rows"], case["n_out"], device="cuda", dtype=torch.float64)
        pre = torch.zeros_like(y) if case["train"] else None
        for i, r in _parts(case, s):
            z = torch.mm(x[r].double(), s["weight"][i].double().t())
            if case["bias"]:
                z = z + s["bias"][i].double()
            if pre is not None:
                pre[r] = z
            if act == "relu":
                z = torch.where(z > 0, z, torch.zeros_like(z))
            elif act == "gelu":
                z = z * normal_below(z)
            elif act in ("silu", "sigmoid"):
                z = (z if act == "silu" else 1) / (1 + torch.exp(-z))
            y[r] = z + s["residual"][r].double() if case["add"] else z
        return dict(y=y) if pre is None else dict(y=y, pre=pre)
    dx = torch.zeros(case["rows"], case["n_in"], device="cuda", dtype=torch.float64)
    dweight = torch.zeros(s["weight"].shape, device="cuda", dtype=torch.float64)
    dbias = torch.zeros(s["weight"].shape[:-1], device="cuda", dtype=torch.float64)
    for i, r in _parts(case, s):
        d = s["dy"][r].double()
        if act != "none":
            z = s["pre"][r].double()
            if act == "relu":
                d = torch.where(z > 0, d, torch.zeros_like(d))
            elif act == "gelu":  # of z Phi(z)
                d = d * (normal_below(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
            else:
                below, above = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
                d = d * (below + z * below * above if act == "silu" else below * above)
        dx[r] = torch.mm(d, s["weight"][i].double())
        dweight[i] = torch.mm(d.t(), x[r].double())
        dbias[i] = d.sum(0)
    return dict(dx=dx, dweight=dweight, **({"dbias": dbias} if case["bias"] else {}))
