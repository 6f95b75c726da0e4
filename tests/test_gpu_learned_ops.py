"""Layer norm, gradient norm and AdamW on device tensors against their definitions in 64 bits (learned_ref)."""
import math

import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

import learned_ref as ref
import splatx_hip as sh

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def tb():
    import splatx_torch
    b = splatx_torch.TorchBackend(0)
    yield b
    b.close()


def randn(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float32).to(dtype)


def held(t, pad):
    """t on the device, its rows `pad` elements further apart than they are long."""
    if not pad:
        return t.cuda()
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, :t.shape[1]] = t.cuda()
    return wide[:, :t.shape[1]]


def within(got, want, bound, what):
    got = got.cpu().double()
    d = (got - want).abs()
    bad = ~((d <= bound) | (got == want))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}, worst {(d / bound)[bad].max():.3g} of the bound"


WIDTHS = [1, 2, 3, 4, 7, 8, 16, 31, 32, 33, 45, 48, 63, 64, 65, 96, 100, 128, 129, 250, 256, 257, 384, 511, 512, 513, 768, 1000, 1024,
          1025, 1536, 2047, 2048, 2050, 4096, 4100, 5000, 8191, 8192, 8200, 12001, 16384, 16392, 20000, 40000, 65537]
NORM_CASES = [(w, t, 0, True, F32 if i % 2 else t) for i, w in enumerate(WIDTHS) for t in (F32, BF16, F16)]
NORM_CASES += [(w, t, pad, add, F32) for w in (1, 5, 45, 64, 200, 1024, 3000, 9000, 30000) for t in (F32, BF16)
               for pad, add in ((1, False), (8, True), (3, True))]


@pytest.mark.parametrize("width,dtype,pad,add,wtype", NORM_CASES)
def test_layer_norm(tb, width, dtype, pad, add, wtype):
    """Forward and backward at every width where a kernel's split of the row changes, rows padded or not, odd counts of rows;
    zero rows, rows far from zero and rows of one value among them."""
    rows = max(3, min(301, 200_000 // width)) | 1
    print(f"width {width} rows {rows} {dtype} pad {pad} add {add}", flush=True)
    x = randn(rows, width, seed=width) * torch.exp(randn(rows, 1, seed=1))
    x[::5] += 40.0
    x[1] = 0
    x[2] = 3.0
    x = x.to(dtype)
    r = randn(rows, width, seed=3, dtype=dtype)
    if add:
        r[1:3] = 0
    w, b = (1 + 0.2 * randn(width, seed=4)).to(wtype), (0.3 * randn(width, seed=5)).to(wtype)
    y, h, mean, rstd, bound = ref.norm_fwd(x, w, b, 1e-5, r if add else None)
    gy, gh, gm, gs = tb.layer_norm_fwd(held(x, pad), w.cuda(), b.cuda(), 1e-5, held(r, pad) if add else None)
    assert gy.shape == x.shape and gy.dtype == dtype
    assert torch.equal(gh.cpu().double(), h)
    within(gy, y, bound, "y")
    k = (width / 32 + 16) * ref.U32
    within(gm, mean, k * h.abs().amax(-1) + 1e-40, "mean")
    within(gs, rstd, rstd * (k * (2 + h.abs().amax(-1) * rstd * 2) + 8 * ref.U32), "rstd")

    dy, dh = randn(rows, width, seed=6, dtype=dtype), randn(rows, width, seed=7, dtype=dtype)
    dy[3 % rows] = 0
    (dx, dw, db), (ex, ew, eb) = ref.norm_bwd(dy, gh.cpu(), gm.cpu(), gs.cpu(), w, dh if add else None)
    g = tb.layer_norm_bwd(held(dy, pad), held(gh.cpu(), pad), gm, gs, w.cuda(), held(dh, pad) if add else None)
    assert g[1].dtype == wtype and g[2].dtype == wtype and g[0].dtype == dtype
    within(g[0], dx, ex, "dx")
    within(g[1], dw, ew + ref.UNIT[wtype] * dw.abs() + ref.TINY[wtype], "dweight")
    within(g[2], db, eb + ref.UNIT[wtype] * db.abs() + ref.TINY[wtype], "dbias")


@pytest.mark.parametrize("width,dtype,rows", [(w, t, r) for w, t in ((45, F32), (48, BF16), (64, F16), (320, BF16), (1024, F32))
                                              for r in (1, 2, 63, 64, 65, 255, 257, 1023, 4097, 70_001) if r * w < 20_000_000])
def test_layer_norm_row_counts(tb, width, dtype, rows):
    print(f"rows {rows} width {width} {dtype}", flush=True)
    x = randn(rows, width, seed=rows, dtype=dtype)
    w, b = 1 + 0.2 * randn(width, seed=4), 0.3 * randn(width, seed=5)
    y, h, mean, rstd, bound = ref.norm_fwd(x, w, b, 1e-5)
    gy, gh, gm, gs = tb.layer_norm_fwd(x.cuda(), w.cuda(), b.cuda())
    within(gy, y, bound, "y")
    dy = randn(rows, width, seed=6, dtype=dtype)
    want, bounds = ref.norm_bwd(dy, x, gm.cpu(), gs.cpu(), w)
    got = tb.layer_norm_bwd(dy.cuda(), gh, gm, gs, w.cuda())
    for a, c, e, name in zip(got, want, bounds, ("dx", "dweight", "dbias")):
        within(a, c, e, name)
    again = tb.layer_norm_bwd(dy.cuda(), gh, gm, gs, w.cuda())
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("width", [8, 9, 15, 16, 23, 45, 64, 127, 200, 301, 505, 512, 1001])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("off", [(1, 1, 1), (1, 0, 2), (0, 3, 1), (2, 2, 1)])
def test_layer_norm_rows_off_words(tb, width, dtype, off):
    """16-bit rows that begin off a multiple of four bytes, each input in its own way, up to the last element of its tensor."""
    rows = 131

    def held_off(t, k):
        flat = torch.full((k + t.numel(),), float("nan"), dtype=t.dtype, device="cuda")
        flat[k:] = t.flatten().cuda()
        return flat[k:].view(t.shape)

    x, r = randn(rows, width, seed=1, dtype=dtype), randn(rows, width, seed=2, dtype=dtype)
    w, b = 1 + 0.2 * randn(width, seed=4), 0.3 * randn(width, seed=5)
    for add in (False, True):
        y, h, mean, rstd, bound = ref.norm_fwd(x, w, b, 1e-5, r if add else None)
        gy, gh, gm, gs = tb.layer_norm_fwd(held_off(x, off[0]), w.cuda(), b.cuda(), 1e-5, held_off(r, off[1]) if add else None)
        assert torch.equal(gh.cpu().double(), h)
        within(gy, y, bound, "y")
        dy, dh = randn(rows, width, seed=6, dtype=dtype), randn(rows, width, seed=7, dtype=dtype)
        want, bounds = ref.norm_bwd(dy, gh.cpu(), gm.cpu(), gs.cpu(), w, dh if add else None)
        got = tb.layer_norm_bwd(held_off(dy, off[0]), held_off(gh.cpu(), off[1]), gm, gs, w.cuda(), held_off(dh, off[2]) if add else None)
        for g, c, e, name in zip(got, want, bounds, ("dx", "dweight", "dbias")):
            within(g, c, e, name)


def test_layer_norm_parts(tb):
    """Without weight, bias, statistics; single gradients; shapes of one, two and four dimensions; no rows."""
    x = randn(70, 33, seed=1)
    y, h, mean, rstd, bound = ref.norm_fwd(x, None, None, 1e-3)
    gy, gh, gm, gs = tb.layer_norm_fwd(x.cuda(), eps=1e-3, stats=False)
    assert gm is None and gs is None and gh.data_ptr() != gy.data_ptr()
    within(gy, y, bound, "y")
    b = randn(33, seed=2)
    within(tb.layer_norm_fwd(x.cuda(), None, b.cuda(), 1e-3)[0], y + b.double(), bound + 2 * ref.U32 * (y.abs() + 2 * b.abs()), "y with bias only")
    _, _, gm, gs = tb.layer_norm_fwd(x.cuda(), eps=1e-3)
    dy = randn(70, 33, seed=3)
    full = tb.layer_norm_bwd(dy.cuda(), x.cuda(), gm, gs)
    for i in range(3):
        one = tb.layer_norm_bwd(dy.cuda(), x.cuda(), gm, gs, want_dx=i == 0, want_dweight=i == 1, want_dbias=i == 2)
        assert [t is not None for t in one] == [i == k for k in range(3)]
        assert torch.equal(one[i], full[i])
    four = x[:60].view(3, 4, 5, 33).cuda()
    gy4, _, gm4, _ = tb.layer_norm_fwd(four, eps=1e-3)
    assert gy4.shape == four.shape and gm4.shape == (3, 4, 5) and torch.equal(gy4.view(60, 33), gy[:60])
    gy1, _, gm1, _ = tb.layer_norm_fwd(x[0].cuda(), eps=1e-3)
    assert gy1.shape == (33,) and gm1.shape == () and torch.equal(gy1, gy[0])
    none = torch.empty(0, 33, device="cuda")
    assert tb.layer_norm_fwd(none)[0].shape == (0, 33)
    empty = torch.empty(0, device="cuda")
    dx, dw, db = tb.layer_norm_bwd(none, none, empty, empty)
    assert dx.shape == (0, 33) and not dw.any() and not db.any()


def test_layer_norm_broadcast_and_interleaved_rows(tb):
    """One row read for all (stride 0), rows between another tensor's, a transposed view refused."""
    row = randn(1, 48, seed=1)
    wide = row.cuda().expand(130, 48)
    y, _, m, s = tb.layer_norm_fwd(wide)
    assert torch.equal(y, tb.layer_norm_fwd(row.cuda())[0].expand(130, 48))
    dx, dw, db = tb.layer_norm_bwd(torch.ones(130, 48, device="cuda"), wide, m, s)
    within(db, torch.full((48,), 130.0, dtype=torch.float64), 0, "dbias")
    both = randn(90, 100, seed=2).cuda()
    a, b = both[:, :50], both[:, 50:]
    y, h, _, _ = tb.layer_norm_fwd(a, residual=b)
    want = ref.norm_fwd(a.cpu(), None, None, 1e-5, b.cpu())
    within(y, want[0], want[4], "y")
    with pytest.raises(sh.SxInvalidArgument):
        tb.layer_norm_fwd(both.t())


@pytest.mark.parametrize("width", [3, 45, 64, 300, 1024, 3000, 20000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_layer_norm_values_not_finite_stay_in_their_row(tb, width, dtype):
    x = randn(9, width, seed=1, dtype=dtype)
    clean = tb.layer_norm_fwd(x.cuda())
    for v, row in ((math.nan, 2), (math.inf, 4), (-math.inf, 8)):
        x[row, width // 2] = v
    y = tb.layer_norm_fwd(x.cuda())[0].cpu()
    bad = [2, 4, 8]
    good = [i for i in range(9) if i not in bad]
    assert torch.isnan(y[bad]).all() and torch.equal(y[good], clean[0].cpu()[good])
    dy = randn(9, width, seed=2, dtype=dtype)
    ok = tb.layer_norm_bwd(dy.cuda(), clean[1], clean[2], clean[3])
    dy[5, 0] = math.nan
    got = tb.layer_norm_bwd(dy.cuda(), clean[1], clean[2], clean[3])
    rest = [i for i in range(9) if i != 5]
    assert torch.isnan(got[0][5]).all() and torch.equal(got[0][rest], ok[0][rest])
    assert torch.isnan(got[1][0]) and torch.equal(got[1][1:], ok[1][1:]) and torch.equal(got[2][1:], ok[2][1:])


def test_layer_norm_far_from_zero_and_large(tb):
    """A mean 10^4 times the spread keeps its deviations; values whose sum of squares is near the type's end."""
    x = 1e4 + randn(50, 640, seed=1)
    y, h, mean, rstd, bound = ref.norm_fwd(x, None, None, 1e-5)
    within(tb.layer_norm_fwd(x.cuda())[0], y, bound, "y far from zero")
    x = randn(50, 640, seed=2) * 1e17
    y, h, mean, rstd, bound = ref.norm_fwd(x, None, None, 1e-5)
    within(tb.layer_norm_fwd(x.cuda())[0], y, bound, "large y")
    x = (randn(50, 640, seed=3) * 15000).clamp(-65000, 65000).half()
    y, h, mean, rstd, bound = ref.norm_fwd(x, None, None, 1e-5)
    within(tb.layer_norm_fwd(x.cuda())[0], y, bound, "y of large halves")


def test_layer_norm_offsets_past_32_bits(tb):
    """2.2 * 10^9 elements: the last rows' offsets need more than 31 bits, and more than 32 in bytes."""
    rows, width = 45_000_001, 48
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    tail = randn(1000, width, seed=1, dtype=BF16)
    x[-1000:] = tail.cuda()
    y, h, m, s = tb.layer_norm_fwd(x)
    want = ref.norm_fwd(tail, None, None, 1e-5)
    within(y[-1000:], want[0], want[4], "y")
    assert not y[:-1000].any()
    del y
    dy = torch.zeros_like(x)
    dyt = randn(1000, width, seed=2, dtype=BF16)
    dy[-1000:] = dyt.cuda()
    got = tb.layer_norm_bwd(dy, x, m, s)
    want, bounds = ref.norm_bwd(dyt, tail, m[-1000:].cpu(), s[-1000:].cpu(), None)
    within(got[0][-1000:], want[0], bounds[0], "dx")
    within(got[1], want[1], bounds[1], "dweight")
    within(got[2], want[2], bounds[2], "dbias")


@pytest.mark.parametrize("width", [5, 45, 130])
def test_layer_norm_gradient_against_differences(tb, width):
    """Along random directions of x, weight and bias: central differences of the definition in 64 bits."""
    import splatx_torch
    x, w, b = randn(7, width, seed=1), 1 + 0.2 * randn(width, seed=2), randn(width, seed=3)
    r, cy, ch = (randn(7, width, seed=k) for k in (4, 5, 6))
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, r)]
    y, h = splatx_torch.layer_norm(tb, leaves[0], leaves[1], leaves[2], 1e-5, leaves[3])
    ((y * cy.cuda()).sum() + (h * ch.cuda()).sum()).backward()

    def f(x, w, b, r):
        h = x + r
        d = h - h.mean(-1, keepdim=True)
        y = d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b
        return float((y * cy.double()).sum() + (h * ch.double()).sum())

    base = [t.double() for t in (x, w, b, r)]
    for i, leaf in enumerate(leaves):
        d = randn(*leaf.shape, seed=20 + i).double()
        e = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + e * d, base[i] - e * d
        slope = (f(*up) - f(*down)) / (2 * e)
        got = float((leaf.grad.cpu().double() * d).sum())
        # differences of 64-bit values: e^2 times a third derivative below 10^3 |d|^3, and 2^-52 / e of the sum's size
        assert abs(got - slope) <= 2e-5 * (float((leaf.grad.cpu().double() * d).abs().sum()) + 1), (i, got, slope)


def test_layer_norm_autograd_paths(tb):
    """Gradients that are one value broadcast, a transposed gradient, h alone used, frozen rows."""
    import splatx_torch
    x, w = randn(20, 64, seed=1).cuda().requires_grad_(), randn(64, seed=2).cuda().requires_grad_()
    splatx_torch.layer_norm(tb, x, w).sum().backward()
    want = ref.norm_bwd(torch.ones(20, 64), x.detach().cpu(), *(t.cpu() for t in tb.layer_norm_fwd(x.detach())[2:]), w.detach().cpu())
    within(x.grad, want[0][0], want[1][0], "dx")
    x.grad = None
    c = randn(64, 20, seed=3).cuda()
    (splatx_torch.layer_norm(tb, x, w).t() * c).sum().backward()
    want = ref.norm_bwd(c.cpu().t(), x.detach().cpu(), *(t.cpu() for t in tb.layer_norm_fwd(x.detach())[2:]), w.detach().cpu())
    within(x.grad, want[0][0], want[1][0], "dx of a transposed gradient")
    x.grad, r = None, randn(20, 64, seed=4).cuda().requires_grad_()
    splatx_torch.layer_norm(tb, x, w, residual=r)[1].sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x)) and torch.equal(r.grad, torch.ones_like(x))
    w.grad = None
    splatx_torch.layer_norm(tb, x.detach(), w).sum().backward()
    assert w.grad is not None


# ---- gradient norm -------------------------------------------------------------------------------------

@pytest.mark.parametrize("sizes", [[1], [3], [0, 5, 0], [255, 257, 1, 4096], [1_000_003], [17] * 400, [1, 300_000, 2, 70_001, 3], []])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_grad_norm(tb, sizes, dtype):
    print(sizes[:6], dtype, flush=True)
    ts = [randn(n, seed=i, dtype=dtype) for i, n in enumerate(sizes)]
    want = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    got = tb.grad_norm([t.cuda() for t in ts])
    assert got.shape == () and abs(float(got) - want) <= 2 * ref.U32 * want
    assert torch.equal(got, tb.grad_norm([t.cuda() for t in ts]))


def test_grad_norm_mixed_types_views_and_extremes(tb):
    flat = randn(10_000, seed=1).cuda()
    ts = [flat[1:1002], flat[1003:1004], flat[2001:9999], randn(77, seed=2, dtype=BF16).cuda()[1:], randn(33, seed=3, dtype=F16).cuda()]
    want = math.sqrt(sum(float(t.cpu().double().square().sum()) for t in ts))
    assert abs(float(tb.grad_norm(ts)) - want) <= 2 * ref.U32 * want
    for v in (1e30, 1e-30, 3e38, 1e-42):  # squares beyond 32 bits' range both ways
        t = torch.full((100,), v)
        want = math.sqrt(100 * float(t[0].double()) ** 2)
        got = float(tb.grad_norm([t.cuda()]))
        assert got == math.inf if want > 3.4028235e38 else abs(got - want) <= 2 * ref.U32 * want + 1.5e-45
    for v in (math.nan, math.inf, -math.inf):
        t = torch.ones(5000)
        t[4321] = v
        assert not math.isfinite(float(tb.grad_norm([torch.ones(10).cuda(), t.cuda()])))


# ---- AdamW ---------------------------------------------------------------------------------------------

HYPER = dict(b1=0.9, b2=0.999, eps=1e-8)


def tensors(sizes, ptype, gtype, seed=0, flat=False):
    """(params, masters, grads, m, v) on the CPU."""
    out = [[] for _ in range(5)]
    for i, n in enumerate(sizes):
        p = randn(n, seed=seed + 10 * i)
        g = (0.01 * randn(n, seed=seed + 10 * i + 1)).to(gtype)
        g[torch.rand(n, generator=torch.Generator().manual_seed(i)) < 0.1] = 0
        m = 0.003 * randn(n, seed=seed + 10 * i + 2)
        v = (0.01 * randn(n, seed=seed + 10 * i + 3)).square()
        for k, t in enumerate((p.to(ptype), p, g, m, v)):
            out[k].append(t)
    return out


def on_device(ts, offset=0):
    """Copies on the device, one after another in one buffer from element `offset` on; None: each its own."""
    if offset is None:
        return [t.cuda() for t in ts]
    if not ts:
        return []
    buf = torch.zeros(offset + sum(t.numel() for t in ts), dtype=ts[0].dtype, device="cuda")
    views, at = [], offset
    for t in ts:
        views.append(buf[at:at + t.numel()])
        views[-1].copy_(t)
        at += t.numel()
    return views


def adam_bound(p, g, m, v, new, lr, step):
    """Of a step in 32 bits: the new moments within 3 u of their terms' sizes, the quotient within that over the root (8 u
    of it and, where the two terms of m cancel, of them), the parameter rounded twice."""
    c1 = 1 - 0.9 ** step
    root = (new[2] / (1 - 0.999 ** step)).sqrt() + 1e-8
    terms = 0.9 * m.double().abs() + 0.1 * g.double().abs()
    em = 3 * ref.U32 * terms + 1e-45
    ev = 4 * ref.U32 * new[2] + 3e-45
    ep = 3 * ref.U32 * p.double().abs() + abs(lr) / c1 * (em + 10 * ref.U32 * terms + 1e-38) / root
    return ep, em, ev


SIZES = [[1], [2, 3], [255], [256], [257, 1], [1023, 1024, 1025], [70_001], [5] * 90, [4096, 0, 7, 100_000, 1, 64]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s[:4])))
@pytest.mark.parametrize("ptype,gtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("offset", [None, 0, 1, 3])
def test_adamw32(tb, sizes, ptype, gtype, offset):
    print(sizes[:6], ptype, gtype, offset, flush=True)
    p, master, g, m, v = tensors(sizes, ptype, gtype)
    step, wd = 7, 0.02
    lrs = [1e-3 * (i + 1) for i in range(len(sizes))]
    dev = [on_device(t, offset) for t in (p, master, g, m, v)]
    tb.adamw_step(dev[0], dev[2], dev[3], dev[4], step=step, lr=lrs, weight_decay=wd, master=None if ptype == F32 else dev[1], **HYPER)
    for i in range(len(sizes)):
        new = ref.adamw(master[i], g[i], m[i], v[i], step=step, lr=lrs[i], weight_decay=wd, **HYPER)
        ep, em, ev = adam_bound(master[i], g[i], m[i], v[i], new, lrs[i], step)
        within(dev[3][i], new[1], em, "m")
        within(dev[4][i], new[2], ev, "v")
        if ptype == F32:
            within(dev[0][i], new[0], ep, "param")
        else:
            within(dev[1][i], new[0], ep, "master")
            assert torch.equal(dev[0][i], dev[1][i].to(ptype))
        assert torch.equal(dev[2][i].cpu(), g[i])


def coded(ts):
    """Moments as 8-bit states: (values, codes, scales) for lists of tensors."""
    out = [[], [], []]
    for i, t in enumerate(ts):
        codes, scale = ref.encode(t.double(), ref.random_bits(99, 1, i, t.numel()) & 0xFFFF, False)
        scale = scale.float()
        for k, x in enumerate((ref.decode(codes, scale), codes, scale)):
            out[k].append(x)
    return out


def same_codes(got, want, what):
    """A value within 32-bit rounding of where it would round up may land either side: by one code, in one of 2^9 at most
    (the error of 8 u or so of a value against codes at least 2^-4 of it apart, drawn on a grid of 2^-16)."""
    a, b = got.cpu().view(torch.uint8).int(), want.int()
    off = a != b
    assert int(off.sum()) <= 2 + a.numel() // 512, f"{what}: {int(off.sum())} of {a.numel()} codes differ"
    assert (((a - b).abs() == 1) | ~off).all(), what


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s[:4])))
@pytest.mark.parametrize("ptype,gtype", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("offset", [None, 1])
def test_adamw8(tb, sizes, ptype, gtype, offset):
    print(sizes[:6], ptype, gtype, offset, flush=True)
    p, master, g, m, v = tensors(sizes, ptype, gtype, seed=5)
    step, wd, lr, seed = 3, 0.02, 2e-3, (7 << 40) + 12345
    mv, mc, ms = coded(m)
    rv, rc, rs = coded([x.sqrt() for x in v])
    dev = [on_device(t, offset) for t in (p, master, g, mc, rc, ms, rs)]
    tb.adamw_step(dev[0], dev[2], dev[3], dev[4], step=step, lr=lr, weight_decay=wd, master=None if ptype == F32 else dev[1],
                  exp_avg_scale=dev[5], exp_avg_sq_scale=dev[6], seed=seed, **HYPER)
    for i, n in enumerate(sizes):
        new = ref.adamw(master[i], g[i], mv[i], rv[i].square(), step=step, lr=lr, weight_decay=wd, **HYPER)
        ep, em, ev = adam_bound(master[i], g[i], mv[i], rv[i].square(), new, lr, step)
        # the moments' decoding adds 3 u of theirs
        within(dev[0][i] if ptype == F32 else dev[1][i], new[0], 2 * ep, "param")
        if ptype != F32:
            assert torch.equal(dev[0][i], dev[1][i].to(ptype))
        bits = ref.random_bits(seed, step, i, n)
        codes, scale = ref.encode(new[1], bits & 0xFFFF, False)
        within(dev[5][i], scale, 8 * ref.U32 * scale, "exp_avg_scale")
        same_codes(dev[3][i], codes, "exp_avg")
        codes, scale = ref.encode(new[2].sqrt(), bits >> 16, True)
        within(dev[6][i], scale, 8 * ref.U32 * scale, "exp_avg_sq_scale")
        same_codes(dev[4][i], codes, "exp_avg_sq")


def one_step8(tb, p, g, m, r, **kw):
    """One 8-bit step of a single tensor from (values of) m and the root r: (param, codes and scales on the CPU)."""
    _, mc, ms = coded([m])
    _, rc, rs = coded([r])
    dev = [t.cuda() for t in (p, g, mc[0], rc[0], ms[0], rs[0])]
    tb.adamw_step([dev[0]], [dev[1]], [dev[2]], [dev[3]], exp_avg_scale=[dev[4]], exp_avg_sq_scale=[dev[5]],
                  **{**HYPER, "step": 1, "lr": 1e-3, "seed": 1, **kw})
    return [t.cpu() for t in (dev[0], dev[2], dev[3], dev[4], dev[5])]


def test_adamw8_blocks_of_nothing_and_values_not_finite(tb):
    z = torch.zeros(700)
    p, mc, rc, ms, rs = one_step8(tb, torch.ones(700), z, z, z)
    assert torch.equal(p, torch.ones(700)) and not mc.any() and not rc.any() and not ms.any() and not rs.any()
    # a gradient that is no number: its own element alone, this step and after
    g = randn(700, seed=1)
    good = one_step8(tb, torch.ones(700), g, z, z)
    for bad in (math.nan, math.inf, -math.inf):
        g2 = g.clone()
        small = int(g[256:512].abs().argmin()) + 256  # not its block's largest
        g2[small] = bad
        p, mc, rc, ms, rs = one_step8(tb, torch.ones(700), g2, z, z)
        keep = torch.arange(700) != small
        assert mc[small] == 0x7F and rc[small] == 0x7F and not torch.isfinite(p[small])
        for a, b in ((p, good[0]), (mc, good[1]), (rc, good[2])):
            assert torch.equal(a[keep], b[keep])
        assert torch.equal(ms, good[3]) and torch.equal(rs, good[4])
    # magnitudes 10^7 apart in one block: the small roots keep a code, and no step is larger than the bound of the ratio
    g = torch.full((256,), 1e-7)
    g[3] = 1.0
    p, mc, rc, ms, rs = one_step8(tb, torch.ones(256), g, torch.zeros(256), torch.zeros(256))
    assert (rc > 0).all() and torch.isfinite(p).all()
    # below 2^-100 a block counts as zero
    tiny = torch.full((256,), 1e-33)
    _, mc, rc, ms, rs = one_step8(tb, torch.ones(256), tiny, torch.zeros(256), torch.zeros(256))
    assert not mc.any() and not rc.any() and not ms.any() and not rs.any()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_second_moments_down_to_the_least_float(tb, bits):
    """Elements without gradients for long: their second moments decay through the subnormal numbers to zero, and no root of
    one is anything but small."""
    v = torch.tensor([2.0 ** -e for e in range(60, 150)] + [0.0, 1e-38, 1.1754942e-38, 1.4e-45, 3e-42])
    n = v.numel()
    p, g, m = randn(n, seed=1), torch.zeros(n), torch.zeros(n)
    if bits == 32:
        d = [t.cuda() for t in (p, g, m, v)]
        tb.adamw_step([d[0]], [d[1]], [d[2]], [d[3]], step=9, lr=1e-3, **{**HYPER, "eps": 1e-20})
        new = ref.adamw(p, g, m, v, step=9, lr=1e-3, weight_decay=0.0, **{**HYPER, "eps": 1e-20})
        within(d[3], new[2], 4 * ref.U32 * new[2] + 3e-45, "v")
        got = d[0].cpu()
    else:  # the gradients that give these moments, in blocks of their own size
        g = (v.double() / 1e-3).sqrt().float()
        _, codes, scale = coded([m])
        d = [t.cuda() for t in (p, g, codes[0], codes[0], scale[0], scale[0])]
        tb.adamw_step([d[0]], [d[1]], [d[2]], [d[3]], step=9, lr=1e-30, exp_avg_scale=[d[4]], exp_avg_sq_scale=[d[5]], **HYPER)
        root = v.double().sqrt()
        codes, _ = ref.encode(root, ref.random_bits(0, 9, 0, n) >> 16, True)
        same_codes(d[3][v > 1e-37], codes[v > 1e-37], "exp_avg_sq")
        assert (d[3].cpu().view(torch.uint8) < 0x7F).all()
        got = d[0].cpu()
    assert torch.equal(got, p)


def test_adamw8_moments_follow_a_steady_gradient(tb):
    """200 steps of one gradient per element: the moments' averages over elements of one size go where the exact ones go,
    though a step of the second moment moves a root by a twentieth of the codes' distance: to nearest it would not move."""
    import splatx_torch
    n = 1 << 16
    size = torch.ones(n)
    size[::256] = 1.7  # each block's largest
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = splatx_torch.AdamW(tb, [p], lr=1e-4, weight_decay=0.0, state_bits=8, seed=3)
    for _ in range(200):
        p.grad = size.cuda()
        opt.step()
    m, v = opt.moments(0)
    rest = torch.arange(n) % 256 != 0
    # the mean over 65,000 elements of a spread of under half the value: within 5 sigma, 1 %, and the root's
    # square above its mean's square by the codes' spread of at most an eighth: 1.6 %
    assert abs(float(m.cpu()[rest].mean()) - (1 - 0.9 ** 200)) <= 0.01
    want = 1 - 0.999 ** 200
    assert abs(float(v.cpu()[rest].sqrt().mean()) / math.sqrt(want) - 1) <= 0.05


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_clipping_and_left_out_steps(tb, bits):
    n = 3000
    p, g = randn(n, seed=1), randn(n, seed=2)
    m, r = 0.1 * randn(n, seed=3), randn(n, seed=4).abs()

    def step(norm, **kw):
        if bits == 8:
            return one_step8(tb, p, g, m, r, grad_norm=norm, **kw)
        d = [t.cuda() for t in (p, g, m, r.square())]
        tb.adamw_step([d[0]], [d[1]], [d[2]], [d[3]], **{**HYPER, "step": 1, "lr": 1e-3, "grad_norm": norm, **kw})
        return [d[0].cpu(), d[2].cpu(), d[3].cpu()]

    before = [p] + ([x for t in (coded([m]), coded([r])) for x in (t[1][0],)] + [coded([m])[2][0], coded([r])[2][0]] if bits == 8 else [m, r.square()])
    for v in (math.nan, math.inf, -math.inf):
        for a, b in zip(step(torch.tensor(v).cuda(), max_norm=1.0), before):
            assert torch.equal(a, b)
        for a, b in zip(step(torch.tensor(v).cuda()), before):
            assert torch.equal(a, b)
    norm = tb.grad_norm([g.cuda()])
    plain = step(None)
    for a, b in zip(step(norm, max_norm=1e6), plain):  # not reached
        assert torch.equal(a, b)
    clipped = step(norm, max_norm=0.5)
    scale = 0.5 / float(norm)
    old = (m, r.square()) if bits == 32 else (coded([m])[0][0], coded([r])[0][0].square())
    new = ref.adamw(p, g, *old, step=1, lr=1e-3, weight_decay=0.0, scale=scale, **HYPER)
    ep, _, _ = adam_bound(p, g * scale, *old, new, 1e-3, 1)
    within(clipped[0], new[0], 2 * ep, "clipped param")
    # the loss scale: gradients 8 times theirs, the norm of those, and an eighth of both
    got = [x for x in step(norm * 8, max_norm=0.5, grad_scale=1 / 8)]
    want = ref.adamw(p, g / 8, *old, step=1, lr=1e-3, weight_decay=0.0, scale=0.5 / float(norm) , **HYPER)
    scaled = ref.adamw(p, g, *old, step=1, lr=1e-3, weight_decay=0.0, scale=0.5 / float(norm) / 8, **HYPER)
    assert torch.equal(want[0], scaled[0]) or (want[0] - scaled[0]).abs().max() < 1e-15
    ep, _, _ = adam_bound(p, g * scale / 8, *old, scaled, 1e-3, 1)
    within(got[0], scaled[0], 2 * ep, "param of scaled gradients")


def test_adamw_offsets_past_32_bits(tb):
    """2.2 * 10^9 elements in 8 bits, gradients in bfloat16: the last elements' places need more than 31 bits."""
    n = 2_200_000_123
    p = torch.zeros(n, device="cuda")
    g = torch.zeros(n, dtype=BF16, device="cuda")
    m, r = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    ms, rs = (torch.zeros(-(-n // 256), device="cuda") for _ in range(2))
    tail = randn(1000, seed=1, dtype=BF16)
    g[-1000:] = tail.cuda()
    tb.adamw_step([p], [g], [m], [r], step=1, lr=1e-2, exp_avg_scale=[ms], exp_avg_sq_scale=[rs], seed=1, **HYPER)
    new = ref.adamw(torch.zeros(1000), tail, torch.zeros(1000), torch.zeros(1000), step=1, lr=1e-2, weight_decay=0.0, **HYPER)
    within(p[-1000:], new[0], 1e-2 * 40 * ref.U32, "param")
    assert not p[:-1000].any() and bool(m[-900:].any())
    want = math.sqrt(float(tail.double().square().sum()))
    assert abs(float(tb.grad_norm([g])) - want) <= 2 * ref.U32 * want


# ---- streams, graphs, refusals --------------------------------------------------------------------------

def test_other_streams_and_a_graph(tb):
    """On a side stream, and captured: replays with new inputs in place equal the eager results, other work between them."""
    x, r, w = randn(300, 96, seed=1).cuda(), randn(300, 96, seed=2).cuda(), randn(96, seed=3).cuda()
    dy = randn(300, 96, seed=4).cuda()
    p, m, v = randn(96, seed=5).cuda(), torch.zeros(96).cuda(), torch.zeros(96).cuda()

    def work():
        y, h, mean, rstd = tb.layer_norm_fwd(x, w, None, residual=r)
        dx, dw, _ = tb.layer_norm_bwd(dy, h, mean, rstd, w, want_dbias=False)
        norm = tb.grad_norm([dw])
        tb.adamw_step([p], [dw], [m], [v], step=1, lr=1e-2, grad_norm=norm, max_norm=1.0)
        return y, dx, dw, norm

    def reset():
        p.copy_(randn(96, seed=5))
        m.zero_()
        v.zero_()

    side = torch.cuda.Stream()
    reset()
    torch.cuda.synchronize()
    eager = [t.clone() for t in work()] + [p.clone()]
    reset()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        out = work()
    side.synchronize()
    for a, b in zip([*out, p], eager):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(4):
        x.copy_(randn(300, 96, seed=30 + k))
        reset()
        want = [t.clone() for t in work()] + [p.clone()]
        reset()
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip([*out, p], want):
            assert torch.equal(a, b), k
        (torch.randn(1000, device="cuda") ** 2).sum().item()


def test_on_the_backends_own_stream(tb):
    """Without a queue the call runs on the backend's stream and returns when it is done."""
    import ctypes as C

    import splatx_torch as st
    x, y = randn(100, 48, seed=1).cuda(), torch.empty(100, 48).cuda()
    torch.cuda.synchronize()
    rc = tb.lib.sxh_layer_norm_fwd(tb.handle, C.byref(st.LayerNormInputs(x.data_ptr(), None, None, None, 100, 48, 48, 0, 1e-5, 0, 0)),
                                   C.byref(st.LayerNormOutputs(y.data_ptr(), None, None, None, 48, 0)), None)
    assert rc == sh.SXH_OK, tb.lib.sxh_last_error()
    assert torch.equal(y, tb.layer_norm_fwd(x)[0])


def test_refusals(tb):
    """What is wrong with a call is said before anything runs."""
    import ctypes as C

    import splatx_torch as st
    x = randn(40, 32, seed=1).cuda()
    bad = pytest.raises(sh.SxInvalidArgument)
    with bad:
        tb.layer_norm_fwd(x.cpu())
    with bad:
        tb.layer_norm_fwd(x.double())
    with bad:
        tb.layer_norm_fwd(x, weight=torch.ones(31).cuda())
    with bad:
        tb.layer_norm_fwd(x, weight=torch.ones(32, dtype=BF16).cuda())
    with bad:
        tb.layer_norm_fwd(x, eps=0.0)
    with bad:
        tb.layer_norm_fwd(x, residual=x[:20])
    with bad:
        tb.layer_norm_fwd(torch.empty(3, 0, device="cuda"))
    with bad:
        tb.layer_norm_bwd(x, x, torch.ones(39).cuda(), torch.ones(40).cuda())
    with bad:
        tb.layer_norm_bwd(x, x, torch.ones(40).cuda(), torch.ones(40).cuda(), want_dx=False, want_dweight=False, want_dbias=False)
    with bad:
        tb.layer_norm_bwd(x, x, torch.ones(40).cuda(), torch.ones(40).cuda(), dh=x, want_dx=False)
    f = lambda *a, **k: tb.adamw_step(*a, **{"step": 1, "lr": 1e-3, **k})  # noqa: E731
    p, g, m, v = (randn(100, seed=i).cuda() for i in range(4))
    with bad:
        f([p], [g], [m], [v], step=0)
    with bad:
        f([p], [g], [m], [v], b1=1.0)
    with bad:
        f([p], [g], [m], [v], eps=0.0)
    with bad:
        f([p], [g], [m], [v], max_norm=1.0)
    with bad:
        f([p], [g], [m], [v], lr=math.nan)
    with bad:
        f([p], [g], [m], [v], lr=[1e-3, 1e-3])
    with bad:
        f([p, p], [g, g], [m, m], [v, v])  # one tensor twice
    with bad:
        f([p], [p], [m], [v])
    with bad:
        f([p], [g], [m], [m])
    with bad:
        f([p[:99]], [g], [m], [v])
    with bad:
        f([p.bfloat16()], [g], [m], [v])  # no master
    with bad:
        f([p[::2]], [g[::2]], [m[:50]], [v[:50]])
    with bad:
        f([p], [g], [m.bfloat16()], [v])
    with bad:
        f([p], [g], [m], [v], exp_avg_scale=[v[:1]])
    with bad:
        f([p], [g], [m], [v], seed=-1)
    with bad:
        f([p], [g], [m], [v], lr=None)
    with bad:
        tb.grad_norm([p.double()])
    with bad:
        tb.grad_norm([p.cpu()])
    # at the C boundary: host memory, buffers that end early, overlaps, a short workspace
    call = lambda a, o: tb.lib.sxh_layer_norm_fwd(tb.handle, C.byref(a), C.byref(o), C.byref(st.Queue(None)))  # noqa: E731
    y, host = torch.empty_like(x), torch.empty(40, 32)
    i = lambda ptr, rows=40, stride=32, t=0: st.LayerNormInputs(ptr, None, None, None, rows, 32, stride, 0, 1e-5, t, 0)  # noqa: E731
    o = lambda ptr, stride=32: st.LayerNormOutputs(ptr, None, None, None, stride, 0)  # noqa: E731
    assert call(i(x.data_ptr()), o(y.data_ptr())) == sh.SXH_OK
    for a, b in ((i(host.data_ptr()), o(y.data_ptr())), (i(x.data_ptr()), o(host.data_ptr())), (i(None), o(y.data_ptr())),
                 (i(x.data_ptr()), o(None)), (i(x.data_ptr(), rows=1 << 40), o(y.data_ptr())), (i(x.data_ptr(), rows=-1), o(y.data_ptr())),
                 (i(x.data_ptr(), stride=31), o(y.data_ptr())), (i(x.data_ptr()), o(y.data_ptr(), stride=0)),
                 (i(x.data_ptr()), o(x.data_ptr() + 4)), (i(x.data_ptr()), o(x.data_ptr())), (i(x.data_ptr() + 2), o(y.data_ptr())),
                 (i(x.data_ptr(), t=7), o(y.data_ptr())), (i(x.data_ptr(), stride=1 << 62), o(y.data_ptr()))):
        assert call(a, b) == sh.SXH_ERR_INVALID_ARGUMENT
    norm = torch.empty(1).cuda()
    table = st._NORM_ROW.pack(x.data_ptr(), x.numel(), 0)
    work = torch.empty(tb.lib.sxh_grad_norm_workspace(1), dtype=torch.uint8).cuda()
    n = work.numel()
    assert tb.lib.sxh_grad_norm(tb.handle, table, 1, norm.data_ptr(), work.data_ptr(), n - 1, None) == sh.SXH_ERR_INVALID_ARGUMENT
    assert tb.lib.sxh_grad_norm(tb.handle, table, 1, x.data_ptr(), work.data_ptr(), n, None) == sh.SXH_ERR_INVALID_ARGUMENT
    assert tb.lib.sxh_grad_norm(tb.handle, table, 1, None, work.data_ptr(), n, None) == sh.SXH_ERR_INVALID_ARGUMENT
    assert tb.lib.sxh_grad_norm(None, table, 1, norm.data_ptr(), work.data_ptr(), n, None) == sh.SXH_ERR_INVALID_ARGUMENT
    torch.cuda.synchronize()


# ---- the optimizer ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_class(tb, bits):
    """Mixed types with and without gradients, a saved and restored state going on with the same bits."""
    import splatx_torch

    def model():
        return [torch.nn.Parameter(t.cuda()) for t in (randn(40, 20, seed=1), randn(64, seed=2, dtype=BF16), randn(5, seed=3), randn(300, seed=4, dtype=F16))]

    def grads(params, k):
        for i, p in enumerate(params):
            p.grad = None if i == 2 and k % 2 else randn(*p.shape, seed=50 + 10 * k + i, dtype=p.dtype).cuda()

    def make(params):
        return splatx_torch.AdamW(tb, [dict(params=params[:2], lr=1e-2), dict(params=params[2:], weight_decay=0.0)], state_bits=bits,
                                  max_norm=3.0, seed=11)

    a = model()
    oa = make(a)
    for k in range(3):
        grads(a, k)
        norm = oa.step()
        want = math.sqrt(sum(float(p.grad.double().square().sum()) for p in a if p.grad is not None))
        assert abs(float(norm) - want) <= 1e-6 * want
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ob = make(b)
    ob.load_state_dict(oa.state_dict())
    for k in range(3, 6):
        grads(a, k), grads(b, k)
        oa.step(), ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q) and torch.isfinite(p.float()).all()
    assert not torch.equal(a[0].detach().cpu(), randn(40, 20, seed=1))


def test_adamw_is_seen_by_autograd(tb):
    """A step between a forward and its backward is an in-place change of what was saved."""
    import splatx_torch
    w = torch.nn.Parameter(randn(300, seed=1).cuda())
    opt = splatx_torch.AdamW(tb, [w])
    (w * w).sum().backward()
    late = (w * w).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.backward()


def test_lists_that_shrink_during_the_call(tb):
    lrs, ts = [], [[randn(50, seed=4 * k + i).cuda() for i in range(2)] for k in range(4)]

    class Rate:
        def __init__(self, gone):
            self.gone = gone

        def __float__(self):
            self.gone.clear()
            return 1e-3

    before = [t.clone() for t in ts[0]]
    lrs += [Rate(lrs), 1e-3]
    with pytest.raises(sh.SxInvalidArgument, match="lr has changed"):
        tb.adamw_step(*ts, step=1, lr=lrs)
    grads = list(ts[1])
    with pytest.raises(sh.SxInvalidArgument, match="grads has changed"):
        tb.adamw_step(ts[0], grads, ts[2], ts[3], step=1, lr=[Rate(grads), 1e-3])
    assert all(torch.equal(a, b) for a, b in zip(ts[0], before))
