"""Linear layers and linear layers of groups of rows, forward and backward, against their definitions in 64 bits (linear_ref)."""
import math

import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

import linear_ref as ref
import splatx_hip as sh

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = (F32, BF16, F16)


@pytest.fixture(scope="module")
def tb():
    import splatx_torch
    b = splatx_torch.TorchBackend(0)
    yield b
    b.close()


def randn(*shape, seed=0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def whole(*shape, seed=0, dtype=F32, most=3):
    """Whole numbers: their sums are exact, so that results have to be equal."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def held(t, pad, off=0):
    """t with its rows `pad` elements further apart than they are long, `off` elements into its buffer, between NaN."""
    if not pad and not off:
        return t
    rows, width = t.shape
    flat = torch.full((off + rows * (width + pad),), float("nan"), dtype=t.dtype, device="cuda")
    v = flat[off:].view(rows, width + pad)[:, :width]
    v.copy_(t)
    return v


def within(got, want, bound, what):
    assert got.shape == want.shape, what
    d = (got.double() - want).abs()
    bad = ~((d <= bound) | (got == want))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}, worst {(d / bound)[bad].max():.3g} of the bound"


def compare(tb, rows, n_in, n_out, dtype, act="none", bias=True, add=False, pad=0, off=0, sizes=None, seed=0):
    print(f"rows {rows} {n_in} -> {n_out} {dtype} {act} bias {bias} add {add} pad {pad} off {off} groups {sizes if sizes is None else sizes[:8]}", flush=True)
    lead, ends = (), None
    if sizes is not None:
        lead, ends = (len(sizes),), torch.cumsum(torch.tensor(sizes), 0).cuda()
    x, w = randn(rows, n_in, seed=seed, dtype=dtype), (randn(*lead, n_out, n_in, seed=seed + 1) / math.sqrt(n_in)).to(dtype)
    b = randn(*lead, n_out, seed=seed + 2, dtype=dtype) if bias else None
    r = randn(rows, n_out, seed=seed + 3, dtype=dtype) if add else None
    (y, pre), (ey, epre) = ref.fwd(x, w, b, act, r, ends)
    held_ = lambda t: None if t is None else held(t, pad, off)  # noqa: E731
    if sizes is None:
        gy, gpre = tb.linear_fwd(held_(x), w, b, act, held_(r), True)
        alone, none = tb.linear_fwd(held_(x), w, b, act, held_(r))
    else:
        gy, gpre = tb.grouped_linear_fwd(held_(x), w, ends, b, act, held_(r), True)
        alone, none = tb.grouped_linear_fwd(held_(x), w, ends, b, act, held_(r))
    assert gy.dtype == gpre.dtype == dtype and none is None and torch.equal(alone, gy)
    within(gy, y, ey, "y")
    within(gpre, pre, epre, "pre")
    dy, z = randn(rows, n_out, seed=seed + 4, dtype=dtype), None if act == "none" else randn(rows, n_out, seed=seed + 5, dtype=dtype)
    want, bounds = ref.bwd(dy, x, w, z, act, ends)
    if sizes is None:
        f = lambda **k: tb.linear_bwd(held_(dy), held_(x), w, held_(z), act, **k)  # noqa: E731
    else:
        f = lambda **k: tb.grouped_linear_bwd(held_(dy), held_(x), w, ends, held_(z), act, **k)  # noqa: E731
    got = f()
    for g, v, e, name in zip(got, want, bounds, ("dx", "dweight", "dbias")):
        assert g.dtype == dtype
        within(g, v, e, name)
    for g, a in zip(got, f()):
        assert torch.equal(g, a)
    return got, f


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out", [
    (1, 1, 1), (1, 16, 64), (2, 3, 5), (31, 7, 9), (33, 8, 8), (65, 45, 64), (300, 48, 64), (257, 64, 3), (129, 64, 64), (1000, 65, 33),
    (640, 128, 128), (513, 100, 131), (200, 129, 127), (77, 256, 300), (300, 300, 260), (9, 1024, 512), (1, 2048, 130), (40, 130, 2050),
    (130, 1000, 1001), (1025, 512, 768)])
def test_whole_numbers_are_exact(tb, rows, n_in, n_out, dtype):
    """Every index counts: with whole numbers the results are the definition's, rounded once."""
    print(rows, n_in, n_out, dtype, flush=True)
    most = 1 if dtype == F16 and max(rows, n_in, n_out) > 900 else 3
    x, w, b = whole(rows, n_in, seed=1, dtype=dtype, most=most), whole(n_out, n_in, seed=2, dtype=dtype, most=most), whole(n_out, seed=3, dtype=dtype)
    r, dy = whole(rows, n_out, seed=4, dtype=dtype), whole(rows, n_out, seed=5, dtype=dtype, most=most)
    z = x.double() @ w.double().t().contiguous() + b.double()
    y, pre = tb.linear_fwd(x, w, b, "relu", r, True)
    assert torch.equal(pre, z.to(dtype)) and torch.equal(y, (z.clamp_min(0) + r.double()).to(dtype))
    dz = torch.where(pre > 0, dy, torch.zeros_like(dy)).double()
    for act, d in (("relu", dz), ("none", dy.double())):
        dx, dw, db = tb.linear_bwd(dy, x, w, pre if act == "relu" else None, act)
        assert torch.equal(dx, (d @ w.double()).to(dtype))
        assert torch.equal(dw, (d.t().contiguous() @ x.double()).to(dtype))
        assert torch.equal(db, d.sum(0).to(dtype))


SHAPES = [(1, 16, 64), (3, 5, 7), (64, 48, 64), (2000, 45, 64), (777, 64, 3), (1001, 64, 64), (500, 64, 128), (300, 96, 65), (70, 128, 256),
          (515, 200, 136), (9, 2048, 520), (33, 700, 300), (1030, 520, 264), (129, 257, 383)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear(tb, i, act, dtype):
    k = i + ref.ACTS.index(act)
    compare(tb, *SHAPES[i], dtype, act, bias=k % 4 != 3, add=k % 2 == 1, pad=(0, 0, 8, 3)[k % 4], off=(0, 0, 0, 1, 5)[k % 5], seed=10 * i)


SIZES = [[5], [0], [0, 0, 7, 0], [1] * 70, [64, 64, 64], [63, 1, 65, 0, 127, 129, 300], [1000, 0, 3], [0, 2, 0, 900, 31, 0, 33, 257, 0],
         [17, 200, 0, 1, 1, 90] * 23]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_in,n_out,act", [(48, 64, "relu"), (64, 64, "gelu"), (45, 3, "sigmoid"), (128, 40, "none"), (96, 200, "silu"), (300, 260, "gelu")])
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_grouped_linear(tb, i, n_in, n_out, act, dtype):
    sizes, behind = SIZES[i], (0, 1, 70, 200)[(i + n_in) % 4]
    k = i + n_out
    compare(tb, sum(sizes) + behind, n_in, n_out, dtype, act, bias=k % 3 != 2, add=k % 2 == 0, pad=(0, 8, 1)[k % 3], off=k % 2, sizes=sizes, seed=i)


WIDE = [(13_000, 520, 1040), (13_001, 515, 1037), (700, 2056, 2200), (1300, 2049, 2051), (70_000, 264, 264), (3000, 1024, 4104), (257, 4096, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(WIDE)))
def test_wide_linear(tb, i, dtype):
    """Tiles of every size, whole lines and others, the sums' length no multiple of a tile's."""
    compare(tb, *WIDE[i], dtype, ref.ACTS[i % 5], add=i % 2 == 0, pad=(0, 0, 8)[i % 3], seed=i)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out", [(13_000, 520, 1040), (1300, 2049, 2051), (2000, 4096, 264), (70_001, 300, 500)])
def test_wide_whole_numbers_are_exact(tb, rows, n_in, n_out, dtype):
    print(rows, n_in, n_out, dtype, flush=True)
    x, w, dy = (whole(*s, seed=i, dtype=dtype, most=1) for i, s in enumerate(((rows, n_in), (n_out, n_in), (rows, n_out))))
    b = whole(n_out, seed=3, dtype=dtype)
    y, _ = tb.linear_fwd(x, w, b)
    assert torch.equal(y, (x.double() @ w.double().t().contiguous() + b.double()).to(dtype))
    dx, dw, db = tb.linear_bwd(dy, x, w)
    assert torch.equal(dx, (dy.double() @ w.double()).to(dtype))
    assert torch.equal(dw, (dy.double().t().contiguous() @ x.double()).to(dtype))
    assert torch.equal(db, dy.double().sum(0).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_in,n_out,sizes", [(520, 1040, [3000, 0, 4100, 1, 2000, 257, 3000]), (515, 1037, [1000, 4001]), (1024, 1408, [700, 1300, 0, 5, 2600]),
                                              (264, 64, [90, 0, 30_000, 3])])
def test_wide_grouped_linear(tb, n_in, n_out, sizes, dtype):
    compare(tb, sum(sizes) + 300, n_in, n_out, dtype, "silu", sizes=sizes, seed=n_in)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out,sizes", [
    (1, 2048, 8192, None), (9, 2048, 2050, None), (32, 4096, 700, None), (33, 4096, 700, None), (7, 1000, 333, None), (3, 515, 129, None), (31, 9000, 65, None),
    (30, 201, 1486, [1] * 28), (60, 700, 515, [0, 33, 1, 0, 2, 20]), (100, 1024, 300, [65] + [0] * 40 + [1] * 10), (12, 640, 640, [0, 0]),
    (500, 300, 300, [3] * 150 + [0] * 50)])
def test_few_rows(tb, rows, n_in, n_out, sizes, dtype):
    """The weights' bytes are all of it: one row to some for each weight."""
    compare(tb, rows, n_in, n_out, dtype, "gelu", add=rows % 2 == 0, pad=rows % 3, sizes=sizes, seed=rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_in", [5, 7, 9, 20, 40, 70, 79, 81, 100, 111, 113, 139, 145, 150, 161, 177, 193, 209, 211, 225, 230, 241, 250])
@pytest.mark.parametrize("rows,n_out,sizes", [(130, 33, None), (4200, 40, None), (150, 70, [60, 0, 80])])
def test_nothing_of_the_padding_is_taken(tb, rows, n_out, sizes, n_in, dtype):
    """Rows between NaN, of widths at and about every count of steps: an element past a row's end would show."""
    compare(tb, rows, n_in, n_out, dtype, "relu", add=True, pad=8 + n_in % 3, off=n_in % 2, sizes=sizes, seed=n_in)
    compare(tb, rows, n_out, n_in, dtype, "relu", add=True, pad=8 + n_in % 3, off=n_in % 2, sizes=sizes, seed=n_in)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out,sizes", [(377, 1500, 290, None), (372, 700, 246, None), (1850, 319, 738, None), (60, 704, 558, [20, 36]), (50, 1000, 64, None),
                                                   (64, 515, 100, None), (100, 515, 200, [64, 0, 1, 32])])
def test_odd_widths_and_few_rows(tb, rows, n_in, n_out, sizes, dtype):
    compare(tb, rows, n_in, n_out, dtype, "silu", pad=8 if n_in % 2 else 0, sizes=sizes, seed=rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out,sizes", [(1, 7544, 1384, None), (3, 1856, 992, None), (36, 5692, 796, None), (64, 300, 9000, None), (65, 300, 1000, None), (17, 5, 700, None),
                                                   (6, 1984, 1536, [2, 1, 3]), (64, 600, 333, [0] * 20 + [40] + [1] * 20), (50, 1000, 77, [16, 17, 0, 1]), (2, 130, 20_000, [0, 1])])
def test_few_rows_backward(tb, rows, n_in, n_out, sizes, dtype):
    for act in ("none", "gelu"):
        compare(tb, rows, n_in, n_out, dtype, act, pad=rows % 3, off=rows % 2, sizes=sizes, seed=rows)


@pytest.mark.parametrize("rows,n_in,n_out,sizes", [(70, 64, 65, None), (3000, 33, 128, None), (5001, 32, 80, [2000, 0, 3, 2998]), (65, 65, 64, None), (3000, 128, 33, None),
                                                   (4099, 97, 20, [64, 65, 1, 3960]), (200, 64, 129, None), (9000, 32, 144, None), (9000, 16, 300, [4000, 5000])])
def test_middle_layers_of_floats(tb, rows, n_in, n_out, sizes):
    for act in ("none", "silu"):
        compare(tb, rows, n_in, n_out, F32, act, pad=rows % 3, off=rows % 2, sizes=sizes, seed=rows)


# Where dx or dweight has under 1024 elements dz's rounding is kept out of them: what is left of it is a second term's own, half a step of
# at most 2^-5 (bfloat16; half 2^-8) of dz, far under an eighth of dz's.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n_in,n_out,sizes", [(11, 26, 62, None), (33, 7, 9, None), (33, 20, 128, None), (40, 3, 64, [20, 0, 20]), (2000, 1, 1, None), (5000, 5, 100, None),
                                                   (3000, 31, 33, [1000, 0, 1, 1999]), (20, 40, 200, None), (3, 200, 60, None), (700, 250, 4, None)])
def test_few_elements_keep_more_of_dz(tb, rows, n_in, n_out, sizes, dtype, monkeypatch):
    monkeypatch.setitem(ref.DZ_UNIT, dtype, ref.UNIT[dtype] / 8)
    for act in ("gelu", "silu", "sigmoid", "relu", "none"):
        compare(tb, rows, n_in, n_out, dtype, act, pad=rows % 3, off=rows % 2, sizes=sizes, seed=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_values_among_few_elements(tb, dtype):
    dy, x, w, pre = (randn(40, 8, seed=i, dtype=dtype) for i in range(4))
    w = w[:8].clone()
    x[3, 2], x[9, 5], w[4, 6], dy[7, 1] = math.inf, math.nan, -math.inf, math.inf
    got = tb.linear_bwd(dy, x, w, pre, "silu")
    want, _ = ref.bwd(dy, x, w, pre, "silu", None)
    for g, v in zip(got, want):
        assert torch.equal(g.isnan(), v[0].isnan() if v.dim() > g.dim() else v.isnan())
        assert torch.equal(g.isposinf(), v.isposinf()) and torch.equal(g.isneginf(), v.isneginf())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out,sizes", [(24, 4281, 200, None), (31, 2274, 90, None), (2, 8000, 33, None), (1, 4097, 1, None), (3, 2049, 7, [1, 0, 1]), (32, 9001, 64, [30]),
                                                   (16, 16_385, 20, [5, 6])])
def test_few_rows_of_long_sums(tb, rows, n_in, n_out, sizes, dtype):
    for pad in (0, 8):
        compare(tb, rows, n_in, n_out, dtype, "silu", add=True, pad=pad, sizes=sizes, seed=rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_in,n_out", [(40, 200), (7, 9), (9001, 64), (64, 128)])
@pytest.mark.parametrize("sizes", [None, [0, 0, 0]])
def test_no_rows(tb, sizes, n_in, n_out, dtype):
    compare(tb, 0, n_in, n_out, dtype, "gelu", sizes=sizes)
