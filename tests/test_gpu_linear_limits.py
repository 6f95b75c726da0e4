"""Linear layers at the limits of their plans: weights that fill a workgroup's LDS."""
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
