"""Linear layers as programs use them: gradients through autograd and against differences, other streams, graphs, strides, values
that are not finite, long buffers, refusals, and the appearance head on them."""
import ctypes as C
import math

import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

import linear_ref as ref
import splatx_hip as sh

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = (F32, BF16, F16)


@pytest.fixture(scope="module")
def st():
    import splatx_torch
    return splatx_torch


@pytest.fixture(scope="module")
def tb(st):
    b = st.TorchBackend(0)
    yield b
    b.close()


def randn(*shape, seed=0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def within(got, want, bound, what):
    d = (got.double() - want).abs()
    bad = ~((d <= bound) | (got == want))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}, worst {(d / bound)[bad].max():.3g} of the bound"


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("groups", [0, 3])
def test_gradient_against_differences(tb, st, act, groups):
    """Of c . y along a direction of all inputs at once, in float: the slope of central differences. The differences' own error is
    h^2 times a third derivative, and that of y's roundings 2^-24 sqrt(n) |y| / h: with h 2^-6 both stay under a hundredth of the slope
    of unit directions here (n = 1000 outputs)."""
    rows, n_in, n_out = 50, 24, 20
    lead, ends = ((groups,), torch.tensor([20, 20, 45], device="cuda")) if groups else ((), None)
    inputs = [randn(rows, n_in, seed=1), randn(*lead, n_out, n_in, seed=2) / 5, randn(*lead, n_out, seed=3), randn(rows, n_out, seed=4)]
    if act == "relu":  # away from the corner: a step moves z by less than 0.05
        z = ref.fwd(inputs[0], inputs[1], inputs[2], ends=ends)[0][1]
        inputs[2] = inputs[2] * 0 + 40.0 * torch.sign(inputs[2])
    leaves = [t.clone().requires_grad_() for t in inputs]
    c = randn(rows, n_out, seed=5)

    def f(x, w, b, r):
        y = st.grouped_linear(tb, x, w, ends, b, act, r) if groups else st.linear(tb, x, w, b, act, r)
        return (y.double() * c.double()).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    for k in range(4):
        d = [torch.zeros_like(t) for t in inputs]
        d[k] = randn(*inputs[k].shape, seed=10 + k)
        d[k] /= d[k].norm()
        h = 2.0 ** -6
        with torch.no_grad():
            diff = (f(*[t + h * e for t, e in zip(inputs, d)]) - f(*[t - h * e for t, e in zip(inputs, d)])).item() / (2 * h)
        slope = (grads[k].double() * d[k].double()).sum().item()
        assert abs(diff - slope) <= 0.01 * grads[k].double().norm().item() + 1e-4, (k, diff, slope)


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_paths(tb, st, dtype):
    """Three dimensions, a broadcast gradient, a transposed one, inputs without gradients, a bias of another shape."""
    x, w, b = randn(4, 7, 40, seed=1, dtype=dtype), randn(24, 40, seed=2, dtype=dtype) / 6, randn(1, 24, seed=3, dtype=dtype)
    r = randn(4, 7, 24, seed=4, dtype=dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    y = st.linear(tb, *leaves[:3], "silu", leaves[3])
    assert y.shape == (4, 7, 24)
    y.sum().backward()
    ones = torch.ones(28, 24, device="cuda", dtype=dtype)
    _, pre = tb.linear_fwd(x, w, b, "silu", None, True)
    dx, dw, db = tb.linear_bwd(ones.view(4, 7, 24), x, w, pre, "silu")
    assert torch.equal(leaves[0].grad, dx) and torch.equal(leaves[1].grad, dw) and torch.equal(leaves[2].grad, db.view(1, 24))
    assert torch.equal(leaves[3].grad, ones.view(4, 7, 24))
    # some inputs only
    w2 = w.clone().requires_grad_()
    st.linear(tb, x, w2, None, "silu").sum().backward()
    _, pre = tb.linear_fwd(x, w, None, "silu", None, True)
    assert torch.equal(w2.grad, tb.linear_bwd(ones.view(4, 7, 24), x, w, pre, "silu", want_dx=False, want_dbias=False)[1])
    x2 = x.view(28, 40).clone().requires_grad_()
    y = st.linear(tb, x2, w, b)
    (gx,) = torch.autograd.grad(y, x2, randn(24, 28, seed=9, dtype=dtype).t())
    assert torch.equal(gx, tb.linear_bwd(randn(24, 28, seed=9, dtype=dtype).t().contiguous(), x2.detach(), w)[0])
    with torch.no_grad():
        assert not st.linear(tb, x, w, b, "gelu").requires_grad
    # a weight shared by two layers
    w3 = torch.randn(16, 16, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype).requires_grad_()
    x3 = randn(33, 16, seed=5, dtype=dtype)
    h = st.linear(tb, x3, w3)
    st.linear(tb, h, w3).sum().backward()
    one = torch.ones(33, 16, device="cuda", dtype=dtype)
    dh, d1, _ = tb.linear_bwd(one, h.detach(), w3.detach())
    d2 = tb.linear_bwd(dh, x3, w3.detach())[1]
    assert torch.equal(w3.grad, d2 + d1)


def test_grouped_autograd_leaves_rows_of_no_group(tb, st):
    x, w, b, r = (t.requires_grad_() for t in (randn(20, 12, seed=1), randn(3, 8, 12, seed=2), randn(3, 8, seed=3), randn(20, 8, seed=4)))
    ends = torch.tensor([5, 5, 13], device="cuda")
    y = st.grouped_linear(tb, x, w, ends, b, "gelu", r)
    assert not y[13:].any() and y[:13].all()
    y.sum().backward()
    assert not x.grad[13:].any() and not r.grad[13:].any() and (r.grad[:13] == 1).all()
    assert not w.grad[1].any() and not b.grad[1].any() and w.grad[0].any() and w.grad[2].any()


CALLS = [(300, 48, 64, None), (9, 2048, 300, None), (5000, 64, 64, None), (700, 520, 520, None), (5000, 64, 64, [1000, 0, 3000]), (600, 520, 300, [100, 400, 1])]


@pytest.mark.parametrize("rows,n_in,n_out,sizes", CALLS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_other_streams_and_a_graph(tb, rows, n_in, n_out, sizes, dtype):
    """On a side stream, and captured: replays with new inputs in place equal the eager results, other work between them."""
    x, dy, r = randn(rows, n_in, seed=1, dtype=dtype), randn(rows, n_out, seed=2, dtype=dtype), randn(rows, n_out, seed=3, dtype=dtype)
    lead = () if sizes is None else (len(sizes),)
    w, b = randn(*lead, n_out, n_in, seed=4, dtype=dtype), randn(*lead, n_out, seed=5, dtype=dtype)
    ends = None if sizes is None else torch.cumsum(torch.tensor(sizes), 0).cuda()

    def work():
        if sizes is None:
            y, pre = tb.linear_fwd(x, w, b, "gelu", r, True)
            return (y, pre, *tb.linear_bwd(dy, x, w, pre, "gelu"))
        y, pre = tb.grouped_linear_fwd(x, w, ends, b, "gelu", r, True)
        return (y, pre, *tb.grouped_linear_bwd(dy, x, w, ends, pre, "gelu"))

    torch.cuda.synchronize()
    eager = [t.clone() for t in work()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = work()
    side.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(out, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(4):
        x.copy_(randn(rows, n_in, seed=30 + k, dtype=dtype))
        if sizes is not None:  # (other groups' sizes too: a graph holds none of them)
            ends.copy_(torch.cumsum(torch.tensor([s + (k if i == 0 else 0) for i, s in enumerate(sizes)]), 0))
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        graph.replay()
        for a, e in zip(out, want):
            assert torch.equal(a, e), k
        (torch.randn(1000, device="cuda") ** 2).sum().item()


def test_two_calls_at_once(tb):
    """On two streams over the same inputs: each has a workspace of its own."""
    x, dy, w = randn(6000, 64, seed=1, dtype=BF16), randn(6000, 64, seed=2, dtype=BF16), randn(64, 64, seed=3, dtype=BF16)
    want = tb.linear_bwd(dy, x, w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(tb.linear_bwd(dy, x, w))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, e) for a, e in zip(o, want))


def test_on_the_backends_own_stream(tb, st):
    x, w, y = randn(100, 48, seed=1), randn(32, 48, seed=2), torch.empty(100, 32, device="cuda")
    torch.cuda.synchronize()
    rc = tb.lib.sxh_linear_fwd(tb.handle, C.byref(st.LinearInputs(x.data_ptr(), w.data_ptr(), None, None, None, 100, 48, 32, 0, 48, 0, 0, 0, 0)),
                               C.byref(st.LinearOutputs(y.data_ptr(), None, 32, 0, None, 0)), None)
    assert rc == sh.SXH_OK, tb.lib.sxh_last_error()
    assert torch.equal(y, tb.linear_fwd(x, w)[0])


@pytest.mark.parametrize("n_in,n_out", [(48, 64), (300, 520), (2048, 40)])
@pytest.mark.parametrize("rows,sizes", [(9, None), (700, None), (700, [300, 0, 200])])
def test_strides(tb, n_in, n_out, rows, sizes):
    """One row read for all (stride 0), column ranges of one buffer, three dimensions; a transposed view refused."""
    lead = () if sizes is None else (len(sizes),)
    w = randn(*lead, n_out, n_in, seed=1, dtype=BF16)
    ends = None if sizes is None else torch.cumsum(torch.tensor(sizes), 0).cuda()
    f = (lambda x, **k: tb.linear_fwd(x, w, **k)[0]) if sizes is None else (lambda x, **k: tb.grouped_linear_fwd(x, w, ends, **k)[0])
    one, r = randn(1, n_in, seed=2, dtype=BF16), randn(1, n_out, seed=3, dtype=BF16)
    assert torch.equal(f(one.expand(rows, n_in), residual=r.expand(rows, n_out)),
                       f(one.expand(rows, n_in).contiguous(), residual=r.expand(rows, n_out).contiguous()))
    both = randn(rows, 2 * n_in + 6, seed=4, dtype=BF16)
    assert torch.equal(f(both[:, 3:3 + n_in]), f(both[:, 3:3 + n_in].contiguous()))
    assert torch.equal(f(both[:, :n_in].contiguous().view(1, rows, n_in))[0], f(both[:, :n_in]))
    with pytest.raises(sh.SxInvalidArgument):
        f(both[:, :n_in].contiguous().t().contiguous().t())
    dy = randn(1, n_out, seed=5, dtype=BF16).expand(rows, n_out)
    g = (lambda d, x: tb.linear_bwd(d, x, w)) if sizes is None else (lambda d, x: tb.grouped_linear_bwd(d, x, w, ends))
    for a, b in zip(g(dy, one.expand(rows, n_in)), g(dy.contiguous(), one.expand(rows, n_in).contiguous())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,n_in,n_out", [(40, 45, 33), (5, 2048, 64), (300, 520, 300), (5000, 64, 64), (33, 3, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_values_not_finite_stay_in_their_row(tb, rows, n_in, n_out, dtype):
    """Of a row that is not finite its own y and dx, and what sums over it; of the padding behind rows nothing."""
    x, w, dy = randn(rows, n_in, seed=1, dtype=dtype), randn(n_out, n_in, seed=2, dtype=dtype), randn(rows, n_out, seed=3, dtype=dtype)
    clean, ok = tb.linear_fwd(x, w)[0], tb.linear_bwd(dy, x, w)
    x2, dy2 = x.clone(), dy.clone()
    x2[3, n_in - 1] = math.nan
    x2[1, 0] = math.inf
    dy2[2, n_out - 1] = math.nan
    y = tb.linear_fwd(x2, w)[0]
    rest = [i for i in range(rows) if i not in (1, 3)]
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[1]).any() and torch.equal(y[rest], clean[rest])
    dx, dw, db = tb.linear_bwd(dy2, x, w)
    rest = [i for i in range(rows) if i != 2]
    assert torch.isnan(dx[2]).all() and torch.equal(dx[rest], ok[0][rest])
    assert torch.isnan(dw[-1]).all() and torch.isnan(db[-1]) and torch.equal(dw[:-1], ok[1][:-1]) and torch.equal(db[:-1], ok[2][:-1])
    # relu's slope is 0 wherever pre is not above 0, whatever dy
    dy2[2] = math.inf
    pre = randn(rows, n_out, seed=4, dtype=dtype)
    pre[2] = -1
    dx, dw, db = tb.linear_bwd(dy2, x, w, pre, "relu")
    assert not dx[2].any() and torch.isfinite(dx).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_activations_far_out(tb, dtype):
    """Down to where a tail vanishes, up to the type's end, by a weight that passes the value on."""
    v = torch.cat([torch.linspace(-40, 40, 4001), torch.tensor([0.0, -0.0, 1e-6, -1e-6, 300.0, -300.0, 6e4, -6e4])]).to(dtype).cuda().view(-1, 1)
    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    for act in ref.ACTS:
        (y, _), (ey, _) = ref.fwd(v, one, None, act)
        got = tb.linear_fwd(v, one, None, act)[0]
        within(got, y, ey, act)
        if act != "none":
            # the tail keeps its relative precision where the type holds it (the exponent's rounding: |z|^2 units of 2^-24)
            few = (y.abs() > 1e-4 if dtype == F16 else y.abs() > 1e-30) & (v.double() > -12)
            rel = ((got.double() - y).abs() / y.abs().clamp_min(1e-300))[few]
            assert rel.max() <= ref.UNIT[dtype] + (5e-5 if dtype != F32 else 400 * ref.U32), act
        dy = torch.ones_like(v)
        if act != "none":
            (dx, _, _), (ex, _, _) = ref.bwd(dy, v, one, v, act)
            within(tb.linear_bwd(dy, v, one, v, act)[0], dx, ex, act)


def test_offsets_past_32_bits(tb):
    """Rows whose bytes and elements lie past 2^32 of their buffers' beginnings."""
    rows, n = 34_000_000, 64
    x = torch.empty(rows, n, dtype=BF16, device="cuda").normal_()
    w = randn(64, 64, seed=1, dtype=BF16) / 8
    y = tb.linear_fwd(x, w, None, "relu")[0]
    for at in (0, rows // 2, rows - 777):
        part = slice(at, at + 777)
        assert torch.equal(y[part], tb.linear_fwd(x[part].contiguous(), w, None, "relu")[0])
    ends = torch.tensor([rows - 1000, rows - 500], device="cuda")
    w2 = torch.stack([w, -w])
    dx, dw, _ = tb.grouped_linear_bwd(y, x, w2, ends)
    last = slice(rows - 1000, rows - 500)
    want = tb.linear_bwd(y[last].contiguous(), x[last].contiguous(), -w)
    assert torch.equal(dx[last], want[0]) and not dx[rows - 500:].any()
    e = ref.bwd(y[last], x[last], -w)
    within(dw[1], e[0][1], e[1][1], "dweight")
    del y, dx
    # rows far apart
    wide = torch.empty(40, 120_000_000, dtype=BF16, device="cuda")[:, :520]
    wide.normal_()
    w = randn(300, 520, seed=2, dtype=BF16)
    assert torch.equal(tb.linear_fwd(wide, w)[0], tb.linear_fwd(wide.contiguous(), w)[0])
    dy = randn(40, 300, seed=3, dtype=BF16)
    assert all(torch.equal(a, b) for a, b in zip(tb.linear_bwd(dy, wide, w), tb.linear_bwd(dy, wide.contiguous(), w)))


@pytest.mark.parametrize("rows,n_in,n_out", [(70, 48, 64), (300, 300, 520), (5000, 64, 64), (12, 700, 40)])
def test_rows_of_no_group_are_left_as_they_were(tb, st, rows, n_in, n_out):
    """Without `clear`, of y, pre and dx; whatever lies in them; with it they are zero. Nothing past the rows is written."""
    x, w, dy = randn(rows, n_in, seed=1), randn(2, n_out, n_in, seed=2), randn(rows, n_out, seed=3)
    end = rows - 7
    ends = torch.tensor([rows // 3, end], device="cuda")
    x[end:] = math.nan
    dy[end:] = math.nan
    for clear in (0, 1):
        y, pre, dx = (torch.full((rows + 3, n), 7.5, device="cuda") for n in (n_out, n_out, n_in))
        a = st.LinearInputs(x.data_ptr(), w.data_ptr(), None, None, ends.data_ptr(), rows, n_in, n_out, 2, n_in, 0, 0, 2, clear)
        work = torch.empty(max(tb.lib.sxh_linear_fwd_workspace(C.byref(a)), 16), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        rc = tb.lib.sxh_linear_fwd(tb.handle, C.byref(a), C.byref(st.LinearOutputs(y.data_ptr(), pre.data_ptr(), n_out, n_out, work.data_ptr(), work.numel())), None)
        assert rc == 0, tb.lib.sxh_last_error()
        a = st.LinearGradsIn(dy.data_ptr(), None, x.data_ptr(), w.data_ptr(), ends.data_ptr(), rows, n_in, n_out, 2, n_out, 0, n_in, 0, 0, clear)
        work = torch.empty(tb.lib.sxh_linear_bwd_workspace(C.byref(a)), dtype=torch.uint8, device="cuda")
        rc = tb.lib.sxh_linear_bwd(tb.handle, C.byref(a), C.byref(st.LinearGrads(dx.data_ptr(), None, None, n_in, work.data_ptr(), work.numel())), None)
        assert rc == 0, tb.lib.sxh_last_error()
        left = 0.0 if clear else 7.5
        for t in (y, pre, dx):
            assert (t[end:rows] == left).all() and (t[rows:] == 7.5).all() and torch.isfinite(t[:end]).all() and (t[:end] != 7.5).all()
    assert torch.isfinite(torch.cat([t.flatten() for t in tb.grouped_linear_bwd(dy, x, w, ends)])).all()


@pytest.mark.parametrize("n_in,n_out", [(48, 64), (300, 260), (64, 64)])
def test_ends_that_do_not_ascend_touch_no_other_rows(tb, n_in, n_out):
    """Descending, negative and too large ends: which rows a group has is not specified, what is written lies in the outputs."""
    rows = 5000
    x, w, dy = randn(rows, n_in, seed=1), randn(4, n_out, n_in, seed=2), randn(rows, n_out, seed=3)
    for bad in ([9000, 100, 3000, 5000], [-5, 2 ** 62, 7, -2 ** 62], [4000, 3000, 2000, 1000], [2 ** 40] * 4):
        print(bad, flush=True)
        ends = torch.tensor(bad, device="cuda")
        y, pre = tb.grouped_linear_fwd(x, w, ends, None, "relu", None, True)
        out = tb.grouped_linear_bwd(dy, x, w, ends, pre, "relu")
        torch.cuda.synchronize()
        assert y.shape == (rows, n_out) and out[1].shape == w.shape
    ends = torch.tensor([rows, rows, rows, rows], device="cuda")
    assert torch.equal(tb.grouped_linear_fwd(x, w, ends)[0], tb.linear_fwd(x, w[0])[0])


def test_no_rows(tb):
    w, none = randn(24, 40, seed=1, dtype=BF16), torch.empty(0, 40, device="cuda", dtype=BF16)
    assert tb.linear_fwd(none, w, None, "relu", None, True)[0].shape == (0, 24)
    for n_out, n_in in ((24, 40), (300, 520)):
        for groups in (0, 3):
            w = randn(*((groups,) if groups else ()), n_out, n_in, seed=1, dtype=BF16)
            x, dy = torch.empty(0, n_in, device="cuda", dtype=BF16), torch.empty(0, n_out, device="cuda", dtype=BF16)
            ends = torch.zeros(3, dtype=torch.int64, device="cuda")
            dx, dw, db = tb.grouped_linear_bwd(dy, x, w, ends) if groups else tb.linear_bwd(dy, x, w)
            assert dx.shape == (0, n_in) and dw.shape == w.shape and not dw.any() and not db.any()


def test_single_gradients(tb):
    for rows, n_in, n_out, sizes in CALLS:
        lead = () if sizes is None else (len(sizes),)
        x, dy, w, z = randn(rows, n_in, seed=1), randn(rows, n_out, seed=2), randn(*lead, n_out, n_in, seed=3), randn(rows, n_out, seed=4)
        ends = None if sizes is None else torch.cumsum(torch.tensor(sizes), 0).cuda()
        for act in ("none", "gelu"):
            pre = z if act == "gelu" else None
            f = lambda **k: tb.linear_bwd(dy, x, w, pre, act, **k) if sizes is None else tb.grouped_linear_bwd(dy, x, w, ends, pre, act, **k)  # noqa: E731
            full = f()
            for i in range(3):
                one = f(want_dx=i == 0, want_dweight=i == 1, want_dbias=i == 2)
                assert [t is not None for t in one] == [i == k for k in range(3)]
                assert torch.equal(one[i], full[i]), (rows, act, i)


def test_refusals(tb, st):
    """What is wrong with a call is said before anything runs."""
    x, w, b, r = randn(40, 32, seed=1), randn(24, 32, seed=2), randn(24, seed=3), randn(40, 24, seed=4)
    wg, ends = randn(3, 24, 32, seed=5), torch.tensor([10, 20, 40], device="cuda")
    bad = pytest.raises(sh.SxInvalidArgument)
    for args, kw in (((x.cpu(), w), {}), ((x.double(), w), {}), ((x, w.bfloat16()), {}), ((x, w.t()), {}), ((x, w[:, :31].contiguous()), {}),
                     ((x, wg), {}), ((x, w[0]), {}), ((x, w, b[:23]), {}), ((x, w, b.bfloat16()), {}), ((x, w, b.cpu()), {}),
                     ((x, w, b), dict(activation="tanh")), ((x, w, b), dict(residual=r[:39])), ((x, w, b), dict(residual=x)),
                     ((x, w, b), dict(residual=r.half())), ((x, w, b), dict(residual=r.view(1, 40, 24))), ((x.t(), w), {}), ((None, w), {}), ((x, None), {}),
                     ((torch.empty(3, 0, device="cuda"), torch.empty(4, 0, device="cuda")), {}), ((x, torch.empty(0, 32, device="cuda")), {})):
        with bad:
            tb.linear_fwd(*args, **kw)
    for args in ((x, w, ends), (x, wg, ends.int()), (x, wg, ends[:2]), (x, wg, ends.cpu()), (x, wg, None), (x, wg, [10, 20, 40]), (x, wg[:0], ends[:0]),
                 (x, wg, ends.view(1, 3)), (x, wg, torch.arange(6, device="cuda")[::2])):
        with bad:
            tb.grouped_linear_fwd(*args)
    with bad:
        tb.linear_bwd(r, x, w, None, "gelu")
    with bad:
        tb.linear_bwd(r, x, w, r, "none")
    with bad:
        tb.linear_bwd(r, x, w, want_dx=False, want_dweight=False, want_dbias=False)
    with bad:
        tb.linear_bwd(x, x, w)
    with bad:
        tb.linear_bwd(r[:39], x, w)
    with bad:
        tb.linear_bwd(r, x, w, x, "gelu")
    # at the C boundary: host memory, buffers that end early, overlaps, a short workspace
    y, host = torch.empty(40, 24, device="cuda"), torch.empty(40, 32)
    p = lambda t: t if t is None or isinstance(t, int) else t.data_ptr()  # noqa: E731
    i = lambda x=x, w=w, rows=40, stride=32, bias=None, residual=None, ends=None, groups=0: st.LinearInputs(  # noqa: E731
        p(x), p(w), p(bias), p(residual), p(ends), rows, 32, 24, groups, stride, 24, 0, 0, 0)
    o = lambda y=y, pre=None, stride=24: st.LinearOutputs(p(y), p(pre), stride, 24, None, 0)  # noqa: E731
    call = lambda a, c: tb.lib.sxh_linear_fwd(tb.handle, C.byref(a), C.byref(c), C.byref(st.Queue(None)))  # noqa: E731
    assert call(i(), o()) == sh.SXH_OK
    for a, c in ((i(x=host), o()), (i(w=host), o()), (i(x=None), o()), (i(w=None), o()), (i(), o(y=None)), (i(), o(y=host)), (i(rows=1 << 36), o()),
                 (i(stride=31), o()), (i(), o(stride=23)), (i(), o(stride=0)), (i(x=y, stride=0), o()), (i(), o(y=x)), (i(), o(pre=y)), (i(residual=y), o()),
                 (i(bias=y), o()), (i(x=x.data_ptr() + 2), o()), (i(w=wg, ends=host, groups=3), o()), (i(w=wg, ends=ends.data_ptr() + 4, groups=3), o()),
                 (i(w=wg, ends=ends, groups=30_000), o()), (i(stride=1 << 61), o())):
        assert call(a, c) == sh.SXH_ERR_INVALID_ARGUMENT
    g = st.LinearGradsIn(p(r), None, p(x), p(w), None, 40, 32, 24, 0, 24, 0, 32, 0, 0, 0)
    n = tb.lib.sxh_linear_bwd_workspace(C.byref(g))
    work, dx, dw = torch.empty(n, dtype=torch.uint8, device="cuda"), torch.empty(40, 32, device="cuda"), torch.empty(24, 32, device="cuda")
    back = lambda *a: tb.lib.sxh_linear_bwd(tb.handle, C.byref(g), C.byref(st.LinearGrads(*[p(t) for t in a])), C.byref(st.Queue(None)))  # noqa: E731
    assert back(dx, dw, None, 32, work, n) == sh.SXH_OK
    for a in ((dx, dw, None, 32, work, n - 1), (dx, dw, None, 32, None, n), (dx, dw, None, 32, host, n), (dx, dw, None, 32, work.data_ptr() + 8, n), (dx, dx, None, 32, work, n),
              (x, dw, None, 32, work, n), (dx, w, None, 32, work, n), (dx, dw, r, 32, work, n), (dx, dw, None, 31, work, n), (work, dw, None, 32, work, n)):
        assert back(*a) == sh.SXH_ERR_INVALID_ARGUMENT
    torch.cuda.synchronize()


# ---- the head -----------------------------------------------------------------------------------------------

def plain(head, features, image, cells):
    """The head in 64 bits on the CPU, from copies of its parameters."""
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in head.named_parameters()}

    def norm(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    def layer(x, name):
        w, b = p[name + ".weight"], p[name + ".bias"]
        if cells is None:
            return x @ w.t() + b
        return torch.stack([w[c] @ v + b[c] for v, c in zip(x, cells.tolist())])

    x = norm(features.cpu().double(), p["norm_weight"], p["norm_bias"])
    stream = x @ p["enter.weight"].t() + p["enter.bias"] + p["embedding"][image] @ p["mix.weight"].t()
    for i in range(len(head.blocks)):
        b = f"blocks.{i}."
        u = layer(norm(stream, p[b + "norm_weight"], p[b + "norm_bias"]), b + "up")
        stream = stream + layer(torch.nn.functional.gelu(u), b + "down")
    return norm(stream, p["last_weight"], p["last_bias"]) @ p["leave.weight"].t() + p["leave.bias"], p


@pytest.mark.parametrize("cut", [False, True])
def test_fused_head_gradients_against_64_bits(tb, cut):
    import appearance_head
    torch.manual_seed(3)
    cells = torch.randint(5, (777,), generator=torch.Generator().manual_seed(2)) * 2 if cut else None  # (cells 1, 3, ... have no splats)
    head = appearance_head.AppearanceHead(tb, 12, 3, hidden=20, embedding=5, dtype=F32, fused=True, cells=cells)
    torch.nn.init.normal_(head.leave.weight)
    features, c = torch.randn(777, 12, device="cuda"), torch.randn(777, 3, device="cuda")
    out = head(features, 1)
    (out * c).sum().backward()
    want, p = plain(head, features, 1, cells)
    (want * c.cpu().double()).sum().backward()
    # a dozen operations of 32 bits with sums of at most 777 terms: some thousands of units of 2^-24 of the largest value
    assert (out.cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()
    for k, v in head.named_parameters():
        g = p[k].grad
        assert (v.grad.cpu().double() - g).norm() <= 1e-4 * g.norm() + 1e-12, k


@pytest.mark.parametrize("cells", [0, 7])
def test_fused_head_trains(cells):
    """A run of the operators together: norms, layers, the rasteriser's gradients, the step."""
    import appearance_head
    losses = appearance_head.demo(n=3000, images=3, steps=12, width=96, height=64, sh_degree=2, quiet=True, fused=True, cells=cells)
    assert all(math.isfinite(x) for x in losses)
