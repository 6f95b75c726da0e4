"""Linear layers of values that are not finite: infinities and NaN come out where the definition has them, by every kernel."""
import math

import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

import linear_ref as ref
from test_gpu_linear import TYPES, randn, tb  # noqa: F401

pytestmark = pytest.mark.gpu


def alike(got, want, what):
    for name in ("isnan", "isposinf", "isneginf"):
        g, w = getattr(got, name)(), getattr(want, name)()
        assert torch.equal(g, w), f"{what} {name}: {int((g != w).sum())} places, first {(g != w).nonzero()[0].tolist()}"


# few rows, their sums in slices, groups of few rows; narrow; tiles
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n_in,n_out,sizes", [
    (3, 700, 333, None), (20, 1856, 37, None), (32, 300, 1000, None), (5, 1000, 17, None), (4, 9001, 301, None), (7, 515, 259, [2, 0, 4]), (60, 704, 323, [20, 36]),
    (40, 8, 8, None), (5000, 64, 64, None), (5000, 45, 33, [2000, 0, 2500]), (300, 520, 300, None), (700, 515, 333, [300, 0, 400]), (9000, 33, 130, None), (33_000, 201, 5, None), (35_000, 161, 40, [20_000, 0, 14_000]),
    (70_000, 40, 1200, None), (100, 515, 333, None)])
def test_infinities_are_the_definitions(tb, rows, n_in, n_out, sizes, dtype):  # noqa: F811
    print(rows, n_in, n_out, sizes, dtype, flush=True)
    lead, ends = ((len(sizes),), torch.cumsum(torch.tensor(sizes), 0).cuda()) if sizes else ((), None)
    x, w, dy, pre = randn(rows, n_in, seed=1, dtype=dtype), randn(*lead, n_out, n_in, seed=2, dtype=dtype), randn(rows, n_out, seed=3, dtype=dtype), randn(rows, n_out, seed=4, dtype=dtype)
    w[..., n_out - 1, 2], w[..., 0, 5], w[..., 3, n_in - 1] = math.inf, -math.inf, math.nan
    (y, _), _ = ref.fwd(x, w, None, "none", None, ends)
    got = tb.linear_fwd(x, w)[0] if ends is None else tb.grouped_linear_fwd(x, w, ends)[0]
    alike(got, y, "y")
    for act in ("none", "silu"):
        z = None if act == "none" else pre
        (dx, _, _), _ = ref.bwd(dy, x, w, z, act, ends)
        got = tb.linear_bwd(dy, x, w, z, act) if ends is None else tb.grouped_linear_bwd(dy, x, w, ends, z, act)
        alike(got[0], dx, f"dx {act}")
        assert torch.isfinite(got[1]).all() and torch.isfinite(got[2]).all()
    x2, dy2 = x.clone(), dy.clone()
    x2[1, n_in - 1], x2[2, 0], dy2[0, n_out - 1], dy2[min(rows - 1, 30), 0] = math.inf, math.nan, -math.inf, math.inf
    (y, _), _ = ref.fwd(x2, w, None, "none", None, ends)
    alike(tb.linear_fwd(x2, w)[0] if ends is None else tb.grouped_linear_fwd(x2, w, ends)[0], y, "y of x")
    want, _ = ref.bwd(dy2, x2, w, pre, "silu", ends)
    got = tb.linear_bwd(dy2, x2, w, pre, "silu") if ends is None else tb.grouped_linear_bwd(dy2, x2, w, ends, pre, "silu")
    for g, v, name in zip(got, want, ("dx", "dweight", "dbias")):
        alike(g, v, name)
