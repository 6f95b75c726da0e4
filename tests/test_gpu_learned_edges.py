"""Layer norm, gradient norm and AdamW where sums are exact, rows and launches are many, or a program changes things between
calls (the operators over their ordinary range: test_gpu_learned_ops)."""
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
