"""Layer norm, gradient norm and AdamW where sums are exact, rows and launches are many, or a program changes things between
calls (the operators over their ordinary range: test_gpu_learned_ops)."""
import math

import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

import learned_ref as ref
from test_gpu_learned_ops import BF16, F16, F32, randn, tb, within  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,dtype", [(20_000, F32), (40_000, BF16), (40_000, F16)])
def test_layer_norm_long_rows_about_their_exact_mean(tb, width, dtype):
    """Rows past a workgroup's registers whose sums are whole numbers below 2^24, exact in any order: rows of one value give
    the bias to the bit; rows of small steps about a large value keep the steps as a row about zero does."""
    w, b = 1 + 0.2 * randn(width, seed=4), 0.3 * randn(width, seed=5)
    x = torch.tensor([100.0, 1000.0, -1000.0, 117 * 512.0, 0.0])[:, None].expand(5, width).to(dtype).contiguous()
    y, _, mean, _ = tb.layer_norm_fwd(x.cuda(), w.cuda(), b.cuda())
    assert torch.equal(mean.cpu(), x[:, 0].float())
    assert torch.equal(y.cpu(), b.to(dtype).expand(5, width))
    step = torch.arange(width) % 5 - 2  # (sum 0)
    x = torch.stack([(256 if dtype == F32 else 126) + step[torch.randperm(width, generator=torch.Generator().manual_seed(i))] for i in range(3)])
    x = x.to(dtype)
    y, _, mean, _ = tb.layer_norm_fwd(x.cuda(), w.cuda(), b.cuda())
    assert torch.equal(mean.cpu(), x.double().mean(1).float())
    want, _, _, rstd, _ = ref.norm_fwd(x, w, b, 1e-5)
    xhat = (x.double() - x.double().mean(1, keepdim=True)) * rstd[:, None]
    # rstd: the squares' sum is exact too, a quotient, a root and a quotient of it half a unit each; then two products and a sum
    bound = 8 * ref.U32 * (w.double() * xhat).abs() + 2 * ref.U32 * (want.abs() + b.double().abs())
    within(y, want, bound + ref.UNIT[dtype] * want.abs() + ref.TINY[dtype], "y")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_layer_norm_rows_of_one_value_give_the_bias(tb, dtype):
    """At every width up to 6000: a row of one value whose sums are exact in any order (whole numbers of few bits) has that
    value as its mean, and the bias as its output, to the bit."""
    x = torch.tensor([100.0, 1000.0, -3000.0, 117 * 512.0, 0.0]).to(dtype).cuda()
    b = randn(6000, seed=1).cuda()
    wrong = torch.zeros(6001, dtype=torch.int64, device="cuda")
    for width in range(1, 6001):
        if width % 1000 == 1:
            print(dtype, "width", width, flush=True)
        y, _, mean, _ = tb.layer_norm_fwd(x[:, None].expand(5, width).contiguous(), None, b[:width])
        wrong[width] = (y != b[:width].to(dtype)).sum() + (mean != x.float()).sum()
    assert not wrong.any(), f"{int((wrong > 0).sum())} widths, first {wrong.nonzero()[:8].flatten().tolist()}"


def test_adamw_of_more_elements_than_a_launch(tb):
    """2^34 and some elements in 8 bits, gradients in bfloat16 (137 GB): a launch takes 2^34 - 1024 of them."""

    torch.cuda.empty_cache()
    border, n = 2 ** 34 - 1024, 2 ** 34 + 5003
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GiB of device memory")
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda")
    m, r = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    ms, rs = (torch.zeros(-(-n // 256), device="cuda") for _ in range(2))
    grads, places = randn(3000, seed=1, dtype=BF16), [(7, 507), (border - 500, border + 1000), (n - 1000, n)]
    for at, (i, j) in zip((0, 500, 2000), places):
        g[i:j] = grads[at:at + j - i].cuda()
    tb.adamw_step([p], [g], [m], [r], step=1, lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, exp_avg_scale=[ms], exp_avg_sq_scale=[rs], seed=1)
    new = ref.adamw(torch.zeros(3000), grads, torch.zeros(3000), torch.zeros(3000), step=1, lr=1e-2, weight_decay=0.0, b1=0.9, b2=0.999, eps=1e-8)
    got = torch.cat([p[i:j].cpu() for i, j in places])
    within(got, new[0], 1e-2 * 40 * ref.U32, "param")
    codes = torch.cat([m[i:j].cpu() for i, j in places])
    assert ((codes & 0x7F) > 0)[grads.abs() > 0.1].all()
    for i, j in places:
        p[i:j] = 0
    for i in range(0, n, 1 << 31):
        assert not p[i:i + (1 << 31)].any(), i
    want = math.sqrt(float(grads.double().square().sum()))
    assert abs(float(tb.grad_norm([g])) - want) <= 2 * ref.U32 * want
    del p, g, m, r, ms, rs
    torch.cuda.empty_cache()


def test_adamw_of_lists_whose_items_are_replaced(tb):
    """A number's conversion that puts other tensors into the lists: the step is of those that are there once the numbers are
    known, all of one kind from one list, and autograd hears of the parameter that was stepped."""
    kinds = [[randn(5000, seed=4 * k + i).cuda() for i in range(2)] for k in range(4)]
    kinds[3] = [t.square() for t in kinds[3]]
    others = [[randn(5000, seed=50 + 4 * k + i).cuda() for i in range(2)] for k in range(3)] + [[t.square() for t in kinds[2]]]
    want = [[t.clone() for t in ts] for ts in others]
    tb.adamw_step(*want, step=1, lr=1e-3)
    before = [[t.clone() for t in ts] for ts in kinds]

    class Rate:
        def __float__(self):
            for ts, other in zip(lists, others):
                ts[:] = other
            return 1e-3

    lists, versions = [list(ts) for ts in kinds], [t._version for t in kinds[0] + others[0]]
    tb.adamw_step(*lists, step=1, lr=[1e-3, Rate()])
    for ts, old in zip(kinds, before):
        assert all(torch.equal(a, b) for a, b in zip(ts, old))
    for ts, new in zip(others, want):
        assert all(torch.equal(a, b) for a, b in zip(ts, new))
    assert [t._version for t in kinds[0]] == versions[:2] and all(t._version > v for t, v in zip(others[0], versions[2:]))


def optimizer_params(dtype=F32):
    return [torch.nn.Parameter(randn(n, seed=n).to(dtype).cuda()) for n in (700, 3000)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_parameters_count_their_own_steps(tb, bits, dtype):
    """A parameter whose first gradient comes at the sixth step takes its first step then, as it would alone; the second one
    with no gradient between them as well."""
    import splatx_torch
    p = optimizer_params(dtype)
    opt = splatx_torch.AdamW(tb, p, lr=1e-2, state_bits=bits)
    for k in range(6):
        p[0].grad = randn(700, seed=20 + k, dtype=dtype).cuda()
        p[1].grad = randn(3000, seed=40, dtype=dtype).cuda() if k == 5 else None
        opt.step()
    q = optimizer_params(dtype)[1]
    alone = splatx_torch.AdamW(tb, [q], lr=1e-2, state_bits=bits)
    q.grad = randn(3000, seed=40, dtype=dtype).cuda()
    alone.step()
    assert torch.equal(p[1], q)  # (a first step's parameters do not depend on the moments' rounding)
    assert [int(s["taken"][0]) for s in opt.state] == [6, 1] and opt.steps == 6


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps_left_out_are_not_counted(tb, bits):
    """Overflowed steps before the first and between others: the parameters go where they would have gone without them."""
    import splatx_torch
    p, q = optimizer_params(), optimizer_params()
    a = splatx_torch.AdamW(tb, p, lr=1e-2, state_bits=bits, max_norm=1e3)
    b = splatx_torch.AdamW(tb, q, lr=1e-2, state_bits=bits, max_norm=1e3)
    for k, bad in enumerate((True, True, False, True, False) if bits == 32 else (True, True, False)):
        for i in (0, 1):
            g = randn(p[i].numel(), seed=60 + 2 * k + i).cuda()
            if bad:
                p[i].grad = g.clone()
                p[i].grad[5] = float("inf")
            else:
                p[i].grad, q[i].grad = g, g
        a.step()
        if not bad:
            b.step()
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    assert a.steps > b.steps and [int(s["taken"][0]) for s in a.state] == [b.steps] * 2


def test_adamw_loads_states_without_counts(tb):
    """A state saved before parameters counted their own steps: all of them took every step."""
    import splatx_torch
    p = optimizer_params()
    opt = splatx_torch.AdamW(tb, p)
    for k in range(3):
        for x in p:
            x.grad = randn(x.numel(), seed=70 + k).cuda()
        opt.step()
    d = opt.state_dict()
    for s in d["state"]:
        del s["taken"]
    q = [torch.nn.Parameter(x.detach().clone()) for x in p]
    other = splatx_torch.AdamW(tb, q)
    other.load_state_dict(d)
    for x, y in zip(p, q):
        x.grad = y.grad = randn(x.numel(), seed=80).cuda()
    opt.step(), other.step()
    assert all(torch.equal(x, y) for x, y in zip(p, q))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 36, 80])
def test_adamw_step_by_counts_on_the_device(tb, bits, count):
    """Some tensors of a call with counts of their own, more than one launch takes; and the counts refused where they are wrong."""
    import splatx_hip as sh
    from test_gpu_learned_ops import HYPER, adam_bound, coded
    taken = [torch.tensor([k % 7, 0]).cuda() for k in range(count)]
    p, g, m = ([randn(100 + k, seed=3 * k + j) for k in range(count)] for j in range(3))
    r = [randn(100 + k, seed=900 + k).abs() for k in range(count)]
    if bits == 8:
        (m, mc, ms), (r, rc, rs) = coded(m), coded(r)
        dev = [[t.cuda() for t in ts] for ts in (p, g, mc, rc)]
        more = dict(exp_avg_scale=[t.cuda() for t in ms], exp_avg_sq_scale=[t.cuda() for t in rs])
    else:
        dev, more = [[t.cuda() for t in ts] for ts in (p, g, m, [t.square() for t in r])], {}
    tb.adamw_step(*dev, step=50, lr=[1e-3 * (k + 1) for k in range(count)], taken=taken, **more, **HYPER)
    for k in range(count):
        v = r[k].square()
        new = ref.adamw(p[k], g[k], m[k], v, step=k % 7 + 1, lr=1e-3 * (k + 1), weight_decay=0.0, **HYPER)
        within(dev[0][k], new[0], 2 * adam_bound(p[k], g[k], m[k], v, new, 1e-3 * (k + 1), k % 7 + 1)[0], "param")
        assert int(taken[k][0]) == k % 7 + 1
    for bad in ([t.int() for t in taken], [t[:1] for t in taken], taken[:-1], [t.cpu() for t in taken], [dev[3][0]] * count):
        with pytest.raises(sh.SxInvalidArgument):
            tb.adamw_step(*dev, step=50, lr=1e-3, taken=bad, **more, **HYPER)


def test_adamw_in_a_graph_counts_its_replays(tb):
    """Captured with counts on the device, each replay is the next step."""
    p, m, v = (randn(2000, seed=1).cuda(), torch.zeros(2000).cuda(), torch.zeros(2000).cuda())
    g, taken = torch.zeros(2000).cuda(), torch.zeros(2, dtype=torch.int64).cuda()
    q = [t.clone() for t in (p, m, v, taken)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tb.adamw_step([p], [g], [m], [v], step=1, lr=1e-2, taken=[taken])
    for k in range(4):
        g.copy_(randn(2000, seed=90 + k))
        tb.adamw_step([q[0]], [g], [q[1]], [q[2]], step=1, lr=1e-2, taken=[q[3]])
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip((p, m, v), q):
            assert torch.equal(a, b), k
        assert int(taken[0]) == k + 1
        (torch.randn(1000, device="cuda") ** 2).sum().item()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_adamw_weights_set_after_the_optimizer_was_made(tb, bits, dtype):
    """16-bit parameters loaded, edited through .data or given other storage after their masters were taken: steps go on from
    what they are, the elements that nobody set from their masters."""
    import splatx_torch
    sizes, lr = (700, 3001, 64), 1e-3
    p = [torch.nn.Parameter(randn(n, seed=n).to(dtype).cuda()) for n in sizes]
    opt = splatx_torch.AdamW(tb, p, lr=lr, weight_decay=0.0, state_bits=bits, seed=5)
    loaded = [randn(n, seed=n + 1).to(dtype).cuda() for n in sizes]

    def load():
        with torch.no_grad():
            p[0].copy_(loaded[0])
        p[1].data.copy_(loaded[1])
        p[2].data = loaded[2].clone()

    load()
    q = [torch.nn.Parameter(t.clone()) for t in loaded]
    fresh = splatx_torch.AdamW(tb, q, lr=lr, weight_decay=0.0, state_bits=bits, seed=5)
    for k in range(5):
        if k == 3:  # the weights again, and some of a tensor's only
            with torch.no_grad():
                p[1][100:1001:3] = 0.25
                q[1][100:1001:3] = 0.25
            fresh.state[1]["master"][100:1001:3] = 0.25
        for i, n in enumerate(sizes):
            p[i].grad = q[i].grad = randn(n, seed=100 + 10 * k + i, dtype=dtype).cuda()
        opt.step(), fresh.step()
        for x, y, s, t in zip(p, q, opt.state, fresh.state):
            assert torch.equal(x, y) and torch.equal(s["master"], t["master"]) and torch.equal(x, s["master"].to(dtype))
    assert all(bool((s["master"] != x.float()).any()) for x, s in zip(p, opt.state))  # (the masters hold more than the parameters)
    # without `adopt` the operator's parameters are its masters' roundings, whatever they were
    s, x = opt.state[0], torch.zeros_like(p[0])
    want = s["master"].clone()
    kw = dict(exp_avg_scale=[s["exp_avg_scale"]], exp_avg_sq_scale=[s["exp_avg_sq_scale"]]) if bits == 8 else {}
    tb.adamw_step([x], [torch.zeros_like(x)], [s["exp_avg"]], [s["exp_avg_sq"]], step=1, lr=0.0, master=[s["master"]], **kw)
    assert torch.equal(s["master"], want) and torch.equal(x, want.to(dtype))


@pytest.mark.parametrize("wshape,bshape", [((1, 64), (64,)), ((64,), (1, 1, 64)), ((8, 8), (64, 1)), ((64,), (64,))])
def test_layer_norm_weights_of_any_shape_get_gradients_of_it(tb, wshape, bshape):
    import splatx_torch
    x, w, b, dy = (randn(30, 64, seed=1), 1 + 0.2 * randn(64, seed=2), randn(64, seed=3), randn(30, 64, seed=4).cuda())
    flat = [t.cuda().requires_grad_() for t in (x, w, b)]
    splatx_torch.layer_norm(tb, *flat).backward(dy)
    shaped = [t.cuda().requires_grad_() for t in (x, w.view(wshape), b.view(bshape))]
    splatx_torch.layer_norm(tb, *shaped).backward(dy)
    for a, c in zip(shaped, flat):
        assert a.grad.shape == a.shape and torch.equal(a.grad.flatten(), c.grad.flatten())
    only = shaped[1].detach().clone().requires_grad_()
    splatx_torch.layer_norm(tb, x.cuda(), only).backward(dy)
    assert torch.equal(only.grad.flatten(), flat[1].grad)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-30, 0.5, 1.0, 2.5, 1e30])
def test_adamw_eps(tb, bits, eps):
    """The whole range of eps: above 1, where it outweighs the roots, and down to 1e-30."""
    from test_gpu_learned_ops import coded
    hyper = dict(b1=0.9, b2=0.999, eps=eps)
    p, g, m, r = randn(3000, seed=1), randn(3000, seed=2), 0.1 * randn(3000, seed=3), randn(3000, seed=4).abs()
    if bits == 8:
        (m, mc, ms), (r, rc, rs) = ([t[0] for t in coded([x])] for x in (m, r))
        dev, more = [t.cuda() for t in (p, g, mc, rc)], dict(exp_avg_scale=[ms.cuda()], exp_avg_sq_scale=[rs.cuda()])
    else:
        dev, more = [t.cuda() for t in (p, g, m, r.square())], {}
    tb.adamw_step(*([t] for t in dev), step=3, lr=1e-2 * max(eps, 1.0), **more, **hyper)
    lr = 1e-2 * max(eps, 1.0)
    new = ref.adamw(p, g, m, r.square(), step=3, lr=lr, weight_decay=0.0, **hyper)
    # as in test_gpu_learned_ops.adam_bound, with this eps in the denominator
    terms = 0.9 * m.double().abs() + 0.1 * g.double().abs()
    below = (new[2] / (1 - 0.999 ** 3)).sqrt() + eps
    bound = 3 * ref.U32 * p.double().abs() + lr / (1 - 0.9 ** 3) * (13 * ref.U32 * terms + 1e-38) / below
    within(dev[0], new[0], 2 * bound, "param")


def inside(got, want, bound, what):
    """As `within`, on the device."""
    got = got.double()
    bad = ~(((got - want).abs() <= bound) | (got == want))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


def device_randn(*shape, seed, dtype):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def backward_against_64_bits(tb, rows, width, dtype, off=0):
    """Layer norm's gradients of random rows, without and with dh; `off`: rows that begin that many elements into their tensors.
    A column's sum chains the rows of a thread (here 44 at most), 6 additions over a wave, 4 over a workgroup's, then 16 of a
    thread's share of at most 1024 partial sums, 16 and 2: under 96, so that a row left out or counted twice shows."""
    print(f"rows {rows} width {width} {dtype} off {off}", flush=True)

    def held(seed):
        flat = torch.full((off + rows * width,), float("nan"), dtype=dtype, device="cuda")
        flat[off:] = device_randn(rows * width, seed=seed, dtype=dtype)
        return flat[off:].view(rows, width)

    h, dy, dh = (held(k) for k in (1, 2, 3))
    w = 1 + 0.2 * device_randn(width, seed=4, dtype=F32)
    _, _, mean, rstd = tb.layer_norm_fwd(h, w)
    for add in (None, dh):
        want, bounds = ref.norm_bwd(dy, h, mean, rstd, w, add)
        got = tb.layer_norm_bwd(dy, h, mean, rstd, w, add)
        xhat = (h.double() - mean.double()[:, None]) * rstd.double()[:, None]
        bounds = bounds[0], 100 * ref.U32 * (dy.double() * xhat).abs().sum(0) + 1e-40, 96 * ref.U32 * dy.double().abs().sum(0) + 1e-40
        for a, b, e, name in zip(got, want, bounds, ("dx", "dweight", "dbias")):
            inside(a, b, e, f"{name}, dh {add is not None}")


@pytest.mark.parametrize("rows,width,dtype", [
    (1_000_003, 1, F32), (500_001, 3, F16), (900_001, 4, F32), (500_001, 5, BF16), (600_001, 8, F16), (300_001, 9, BF16), (200_003, 16, F32),
    (250_001, 23, BF16), (30_001, 100, F32), (50_001, 200, BF16), (20_001, 250, F32), (20_001, 301, F16), (9_001, 301, F32), (7_001, 1000, BF16),
    (1_301, 1100, F32), (3_001, 2056, F16), (901, 2500, F32), (901, 5000, BF16), (601, 4100, F32), (601, 10_000, BF16), (601, 6200, F32),
    (601, 13_000, F16), (20_001, 9000, F32), (9_001, 20_001, BF16)])
def test_layer_norm_backward_of_more_rows_than_at_a_time(tb, rows, width, dtype):
    """Each split of a row (1 to 1024 threads, one, three and four vectors a thread, a loop over the row), with rows for two to
    fourteen turns of every workgroup: the columns' sums go on over the turns, the next rows are loaded ahead."""
    backward_against_64_bits(tb, rows, width, dtype)


@pytest.mark.parametrize("rows,width", [(600_001, 9), (250_001, 23), (110_001, 45), (110_001, 46), (70_001, 101), (50_001, 201), (20_001, 301), (20_001, 511)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_layer_norm_backward_of_many_rows_off_words(tb, rows, width, dtype):
    """The same of 16-bit rows that begin off a multiple of four bytes, up to a wave for a row."""
    backward_against_64_bits(tb, rows, width, dtype, off=1)


@pytest.mark.parametrize("rows,width,dtype", [(22_003, 1032, BF16), (11_003, 1024, F32), (5_603, 4096, F16), (5_603, 2048, F32), (2_803, 8192, BF16),
                                              (2_303, 5000, F32), (1_503, 8000, F32), (1_503, 15_000, F16)])
def test_layer_norm_backward_past_the_caches(tb, rows, width, dtype):
    """Over 128 MiB of 16-byte aligned rows, 256 threads or more a row."""
    backward_against_64_bits(tb, rows, width, dtype)


@pytest.mark.parametrize("rows,width,add", [(3_200_001, 520, False), (2_200_003, 520, True), (8_500_001, 260, False)])
def test_layer_norm_forward_of_more_rows_than_a_grid(tb, rows, width, add):
    """More rows than 2^20 workgroups take at a time: the same rows again after some millions give the same bits."""
    head = device_randn(5_001, width, seed=1, dtype=BF16)
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    x[:5_001], x[-5_001:] = head, head
    r = x * 0.5 if add else None
    w, b = 1 + 0.2 * device_randn(width, seed=2, dtype=F32), device_randn(width, seed=3, dtype=F32)
    y, h, mean, rstd = tb.layer_norm_fwd(x, w, b, residual=r)
    want = tb.layer_norm_fwd(head, w, b, residual=head * 0.5 if add else None)
    for got, some in zip((y, h, mean, rstd), want):
        assert torch.equal(got[:5_001], some) and torch.equal(got[-5_001:], some)
    assert torch.equal(y[5_001:-5_001].amin(0), b.to(BF16)) and torch.equal(y[5_001:-5_001].amax(0), b.to(BF16))
    assert not mean[5_001:-5_001].any()


@pytest.mark.parametrize("ptype,gtype,offset", [(F32, F32, 1), (F32, BF16, 0), (BF16, BF16, 3), (F16, F32, 0)])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_past_the_caches(tb, bits, ptype, gtype, offset):
    """Steps of over 128 MiB, tensors of odd sizes one after another in their buffers."""
    from test_gpu_learned_ops import HYPER, adam_bound, same_codes
    sizes = [9_000_003, 5, 70_001, 6_000_002]

    def held(seed, dtype, scale=1.0, blocks=False):
        n = [-(-k // 256) for k in sizes] if blocks else sizes
        flat = (scale * device_randn(offset + sum(n), seed=seed, dtype=F32)).to(dtype)
        return list(flat[offset:].split(n))

    p, g = held(1, F32), held(2, gtype, 0.01)
    master = None if ptype == F32 else p
    param = [t.clone() for t in p] if ptype == F32 else [t.to(ptype) for t in p]
    start = [t.clone() for t in p]
    more = {}
    if bits == 32:
        m, v = held(3, F32, 0.003), [t.square() for t in held(4, F32, 0.01)]
        m0, v0 = [t.clone() for t in m], [t.clone() for t in v]
    else:  # (any codes are moments: m of either sign, roots without one)
        code = lambda seed, top: [(t.abs() * 40).clamp_max(top).byte() for t in held(seed, F32)]  # noqa: E731
        m = [c | (s < 0).byte() << 7 for c, s in zip(code(3, 126), held(5, F32))]
        v = code(4, 126)
        ms, vs = ([t.abs() * 1e-4 + 1e-6 for t in held(k, F32, blocks=True)] for k in (6, 7))
        values = ref.code_values().cuda()
        full = lambda c, s: values[c.long()] * s.double().repeat_interleave(256)[:c.numel()]  # noqa: E731
        m0, v0 = [full(c, s) for c, s in zip(m, ms)], [full(c, s).square() for c, s in zip(v, vs)]
        more = dict(exp_avg_scale=ms, exp_avg_sq_scale=vs, seed=77)
    lr, step = 1e-2, 5
    tb.adamw_step(param, g, m, v, step=step, lr=lr, weight_decay=0.02, master=master, **more, **HYPER)
    for i, n in enumerate(sizes):
        new = ref.adamw(start[i], g[i], m0[i], v0[i], step=step, lr=lr, weight_decay=0.02, **HYPER)
        ep, em, ev = adam_bound(start[i], g[i], m0[i], v0[i], new, lr, step)
        inside(param[i] if master is None else master[i], new[0], 2 * ep, f"param {i}")
        if master is not None:
            assert torch.equal(param[i], master[i].to(ptype))
        if bits == 32:
            inside(m[i], new[1], em, f"m {i}")
            inside(v[i], new[2], ev, f"v {i}")
            continue
        random = ref.random_bits(77, step, i, n)
        for at in {0, n // 512 * 256, max(n - 1, 0) // 256 * 256}:  # three places, whole blocks
            k = slice(at, min(n, at + 25_600))
            codes, scale = ref.encode(new[1][k].cpu(), random[k] & 0xFFFF, False)
            same_codes(m[i][k], codes, "exp_avg")
            within(ms[i][at // 256:at // 256 + scale.numel()], scale, 8 * ref.U32 * scale, "exp_avg_scale")
            codes, scale = ref.encode(new[2][k].sqrt().cpu(), random[k] >> 16, True)
            same_codes(v[i][k], codes, "exp_avg_sq")
            within(vs[i][at // 256:at // 256 + scale.numel()], scale, 8 * ref.U32 * scale, "exp_avg_sq_scale")


@pytest.mark.parametrize("width", [1, 3, 45, 64, 300, 1024, 5000, 20_000])
def test_layer_norm_statistics_of_rows_that_are_not_finite(tb, width):
    """Neither the mean nor rstd of such a row is finite (an infinity of an element that two vectors hold may leave no number), and
    the other rows' are theirs."""
    x = randn(9, width, seed=1)
    last = width - 1
    x[1, 0], x[2, last], x[3, 0], x[4, 0], x[4, last], x[5, 0] = math.inf, -math.inf, math.nan, math.inf, -math.inf if width > 1 else math.inf, 1e30
    want = x.double().sum(1) / width
    mean, rstd = (t.cpu().double() for t in tb.layer_norm_fwd(x.cuda())[2:])
    finite = torch.isfinite(want)
    assert not torch.isfinite(mean[~finite]).any() and torch.isnan(rstd[~finite]).all()
    assert ((mean - want).abs()[finite] <= (width / 32 + 16) * ref.U32 * x.double().abs().amax(1)[finite]).all()
