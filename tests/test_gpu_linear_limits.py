"""Linear layers at the limits of their plans: weights that fill a workgroup's LDS, rows of the most elements."""
import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

from test_gpu_linear import BF16, F16, F32, TYPES, compare, held, randn, tb, whole, within  # noqa: F401

pytestmark = pytest.mark.gpu


# Of a forward of 4096 rows and more: on both sides of where eight waves' outputs fit beside the weight, and where four waves' just do.
@pytest.mark.parametrize("rows,sizes", [(4096, None), (100_000, None), (4500, [1000, 0, 3100, 1, 300])])
@pytest.mark.parametrize("dtype,n_in,n_out", [
    *((t, *s) for t in (BF16, F16) for s in ((128, 384), (256, 192), (192, 256), (64, 768), (96, 512))),
    (BF16, 128, 320), (F16, 40, 900), (BF16, 16, 3584), (F16, 13, 3500), (BF16, 200, 130), (F32, 8, 3584), (F32, 5, 3530), (F32, 8, 3520), (F32, 64, 384)])
def test_weights_that_fill_the_lds(tb, dtype, n_in, n_out, rows, sizes):  # noqa: F811
    compare(tb, rows, n_in, n_out, dtype, "silu", add=True, pad=n_in % 3, sizes=sizes, seed=n_in)


# Rows of as many elements as a layer may have: a tile's lines lie 2^25 bytes (16 bits) and 2^26 (floats) apart, 256 and 128 of them
# (64 floats' already 2^32 bytes).
@pytest.mark.parametrize("dtype,rows,n_in,n_out", [(F32, 33, 1 << 24, 100), (BF16, 40, 1 << 24, 200), (F16, 260, (1 << 23) + 8, 40), (F32, 100, 5, 1 << 24),
                                                   (BF16, 264, 3, (1 << 24) - 8)])
def test_rows_of_the_most_elements(tb, dtype, rows, n_in, n_out):  # noqa: F811
    """Whole numbers, -1 to 1: every partial sum is exact. Compared a range of the long dimension at a time."""
    print(dtype, rows, n_in, n_out, flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    part = 1 << 20

    def ones(n, m):
        t = torch.empty(n, m, dtype=dtype, device="cuda")
        for c in range(0, m, part):
            t[:, c:c + part] = torch.randint(-1, 2, (n, min(part, m - c)), generator=g, device="cuda", dtype=torch.int8)
        return t

    x, w, dy = ones(rows, n_in), (ones(n_out, n_in) if n_out < n_in else ones(n_in, n_out).t().contiguous()), ones(rows, n_out)
    y, _ = tb.linear_fwd(x, w)
    dx, dw, db = tb.linear_bwd(dy, x, w)
    wide = range(0, max(n_in, n_out), part)
    if n_in > n_out:
        z = sum(x[:, c:c + part].double() @ w[:, c:c + part].double().t().contiguous() for c in wide)
        assert torch.equal(y, z.to(dtype))
        for c in wide:
            assert torch.equal(dx[:, c:c + part], (dy.double() @ w[:, c:c + part].double()).to(dtype))
            assert torch.equal(dw[:, c:c + part], (dy.double().t().contiguous() @ x[:, c:c + part].double()).to(dtype))
        assert torch.equal(db, dy.double().sum(0).to(dtype))
        return
    d = sum(dy[:, c:c + part].double() @ w[c:c + part].double() for c in wide)
    assert torch.equal(dx, d.to(dtype))
    for c in wide:
        assert torch.equal(y[:, c:c + part], (x.double() @ w[c:c + part].double().t().contiguous()).to(dtype))
        assert torch.equal(dw[c:c + part], (dy[:, c:c + part].double().t().contiguous() @ x.double()).to(dtype))
        assert torch.equal(db[c:c + part], dy[:, c:c + part].double().sum(0).to(dtype))


# The lines of a sum are shared by eight waves, x's rows are taken eight at a time, and rows begin anywhere, between NaN.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_in", [31, 63, 64, 65, 255, 257, 511, 512, 513, 1025, 2111, 4099, 8321])
def test_few_rows_off_their_lines(tb, n_in, dtype):  # noqa: F811
    for rows, sizes in ((1, None), (8, None), (9, None), (16, None), (17, None), (32, None), (41, [8, 0, 33]), (20, [17])):
        compare(tb, rows, n_in, 77, dtype, "gelu", add=True, pad=1 + rows % 2, off=rows % 3, sizes=sizes, seed=rows)


# Floats between few rows and many, in lines off 16 bytes and on them: 33 to 128 rows by the few rows' kernel, more by tiles through registers.
@pytest.mark.parametrize("n_in,n_out", [(31, 600), (33, 1000), (64, 300), (127, 700), (257, 513), (1025, 200), (2047, 129)])
@pytest.mark.parametrize("rows,sizes", [(33, None), (64, None), (65, None), (128, None), (129, None), (515, None), (600, [100, 0, 65, 400]), (100, [64, 36])])
def test_floats_off_their_lines(tb, rows, sizes, n_in, n_out):  # noqa: F811
    for pad, off in ((0, 0), (1, 1), (4, 0), (3, 2)):
        compare(tb, rows, n_in, n_out, F32, "silu", add=True, pad=pad, off=off, sizes=sizes, seed=rows)


# Floats: rows of several lines, the last of any length, and one or two tiles of outputs.
@pytest.mark.parametrize("n_in,n_out", [(129, 1), (130, 33), (131, 64), (160, 32), (178, 2), (193, 31), (257, 5), (283, 4), (300, 64), (512, 32), (601, 17), (990, 3),
                                        (496, 64), (497, 64)])
@pytest.mark.parametrize("rows,sizes", [(32_768, None), (32_801, None), (70_001, None), (40_000, [1000, 0, 3, 30_100, 1, 33, 300]), (33_000, [31, 32, 33, 0, 0, 1, 1, 32_000])])
def test_long_rows_of_floats(tb, rows, sizes, n_in, n_out):  # noqa: F811
    compare(tb, rows, n_in, n_out, F32, "gelu", bias=n_in % 2 == 0, add=n_out % 2 == 0, pad=n_out % 3, off=n_in % 2, sizes=sizes, seed=n_in)


@pytest.mark.parametrize("dtype,rows,n_in,n_out,sizes", [(F32, 33_000, 201, 5, None), (F32, 35_000, 161, 40, [20_000, 0, 14_000]), (BF16, 70_000, 64, 768, None),
                                                         (F16, 9, 2049, 300, None), (F32, 100, 515, 333, None), (F32, 300, 1001, 333, None)])
def test_captured_and_on_two_streams(tb, dtype, rows, n_in, n_out, sizes):  # noqa: F811
    """A graph of both passes, replayed with new inputs in place between other work, and the same on two streams at once."""
    lead, ends = ((len(sizes),), torch.cumsum(torch.tensor(sizes), 0).cuda()) if sizes else ((), None)
    x, dy, w, b = randn(rows, n_in, seed=1, dtype=dtype), randn(rows, n_out, seed=2, dtype=dtype), randn(*lead, n_out, n_in, seed=3, dtype=dtype), randn(*lead, n_out, seed=4, dtype=dtype)

    def work():
        if ends is None:
            y, pre = tb.linear_fwd(x, w, b, "gelu", dy, True)
            return (y, pre, *tb.linear_bwd(dy, x, w, pre, "gelu"))
        y, pre = tb.grouped_linear_fwd(x, w, ends, b, "gelu", dy, True)
        return (y, pre, *tb.grouped_linear_bwd(dy, x, w, ends, pre, "gelu"))

    want = work()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(work())
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for o in outs for a, e in zip(o, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(3):
        x.copy_(randn(rows, n_in, seed=30 + k, dtype=dtype))
        if sizes:
            ends[:2] += k  # (the second group has no rows: they go on ascending)
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, e) for a, e in zip(out, want)), k
        (torch.randn(1000, device="cuda") ** 2).sum().item()


@pytest.mark.parametrize("dtype,rows,n_in,n_out,groups", [(F32, 40_000, 16, 16, 32768), (BF16, 50_000, 40, 24, 32768), (F16, 20_000, 200, 33, 32768), (F32, 9_000, 70, 33, 4000),
                                                          (BF16, 100, 8, 8, 32768), (F32, 60_000, 130, 20, 1000)])
def test_the_most_groups(tb, dtype, rows, n_in, n_out, groups):  # noqa: F811
    """Whole numbers: every row of every group counts. Rows behind the last group are zero."""
    print(dtype, rows, n_in, n_out, groups, flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    ends = torch.randint(0, rows - 10, (groups,), generator=g, device="cuda").sort()[0]
    of = torch.searchsorted(ends, torch.arange(rows, device="cuda"), right=True)  # the first group that ends behind the row
    ours = of < groups
    of = of[ours]
    x, w, dy, b = whole(rows, n_in, seed=1, dtype=dtype, most=1), whole(groups, n_out, n_in, seed=2, dtype=dtype, most=1), whole(rows, n_out, seed=3, dtype=dtype), whole(groups, n_out, seed=4, dtype=dtype)
    y, _ = tb.grouped_linear_fwd(x, w, ends, b)
    z = torch.cat([(x[i].double()[:, None] * w[o].double()).sum(-1) + b[o].double() for i, o in zip(torch.arange(rows, device="cuda")[ours].split(5000), of.split(5000))])
    assert torch.equal(y[ours], z.to(dtype)) and not y[~ours].any()
    dx, dw, db = tb.grouped_linear_bwd(dy, x, w, ends)
    d = torch.cat([(dy[i].double()[:, :, None] * w[o].double()).sum(1) for i, o in zip(torch.arange(rows, device="cuda")[ours].split(5000), of.split(5000))])
    assert torch.equal(dx[ours], d.to(dtype)) and not dx[~ours].any()
    want = torch.zeros(groups, n_out, n_in, device="cuda")
    for i, o in zip(torch.arange(rows, device="cuda")[ours].split(5000), of.split(5000)):
        want.index_add_(0, o, dy[i].float()[:, :, None] * x[i].float()[:, None])
    assert torch.equal(dw, want.to(dtype))
    assert torch.equal(db, torch.zeros(groups, n_out, device="cuda").index_add_(0, of, dy[ours].float()).to(dtype))
