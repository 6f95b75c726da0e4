"""Grouped linear layers whose ends do not ascend: nothing outside the outputs and the workspace is written."""
import ctypes as C

import pytest
import torch  # before anything loads the library: its HIP runtime is the process's

from test_gpu_linear import BF16, F16, F32, randn, tb  # noqa: F401

pytestmark = pytest.mark.gpu

CODE = {F32: 0, BF16: 1, F16: 2}
GUARD = 1 << 16  # bytes before and behind


class Guarded:
    """Bytes between two ranges of a known value."""

    def __init__(self, size):
        self.size = size
        self.all = torch.full((2 * GUARD + (size + 255) // 256 * 256,), 0xA5, dtype=torch.uint8, device="cuda")
        self.at = self.all.data_ptr() + GUARD

    def intact(self):
        return bool((self.all[:GUARD] == 0xA5).all()) and bool((self.all[GUARD + self.size:] == 0xA5).all())


# narrow, narrow in two terms, tiles in parts, few rows, rows in lines, many groups
@pytest.mark.parametrize("dtype,rows,n_in,n_out,groups", [
    (F32, 5000, 48, 64, 4), (BF16, 5000, 64, 64, 4), (BF16, 5000, 20, 30, 4), (F16, 5000, 300, 260, 4), (F32, 5000, 300, 260, 4), (BF16, 700, 520, 300, 4),
    (F32, 33_000, 201, 5, 4), (F16, 30, 700, 333, 4), (F32, 90, 515, 333, 4), (BF16, 60, 700, 300, 30), (F32, 5000, 33, 130, 4), (BF16, 3000, 16, 16, 500)])
def test_bad_ends_write_nothing_else(tb, dtype, rows, n_in, n_out, groups):  # noqa: F811
    import splatx_torch as st
    e, t = dtype.itemsize, CODE[dtype]
    x, w, dy = randn(rows, n_in, seed=1, dtype=dtype), randn(groups, n_out, n_in, seed=2, dtype=dtype), randn(rows, n_out, seed=3, dtype=dtype)
    pre, bias = randn(rows, n_out, seed=4, dtype=dtype), randn(groups, n_out, seed=5, dtype=dtype)
    g = torch.Generator().manual_seed(6)
    for bad in ([9000, 100, rows, 3000], [-5, 2 ** 62, 7, -2 ** 62], [rows, rows // 2, rows // 3, 1], [2 ** 40] * 4, [-1] * 4, [2 ** 63 - 1, -2 ** 63, rows - 1, rows + 1],
                torch.randint(-rows, 2 * rows, (groups,), generator=g).tolist()):
        bad = (bad * groups)[:groups]
        print(dtype, rows, n_in, n_out, groups, bad[:4], flush=True)
        ends = torch.tensor(bad, device="cuda")
        y, z = Guarded(rows * n_out * e), Guarded(rows * n_out * e)
        a = st.LinearInputs(x.data_ptr(), w.data_ptr(), bias.data_ptr(), None, ends.data_ptr(), rows, n_in, n_out, groups, n_in, 0, t, 3, 1)
        work = Guarded(tb.lib.sxh_linear_fwd_workspace(C.byref(a)))
        torch.cuda.synchronize()
        rc = tb.lib.sxh_linear_fwd(tb.handle, C.byref(a), C.byref(st.LinearOutputs(y.at, z.at, n_out, n_out, work.at, work.size)), None)
        assert rc == 0, tb.lib.sxh_last_error()
        assert y.intact() and z.intact() and work.intact(), "forward"
        dx, dw, db = Guarded(rows * n_in * e), Guarded(groups * n_out * n_in * e), Guarded(groups * n_out * e)
        a = st.LinearGradsIn(dy.data_ptr(), pre.data_ptr(), x.data_ptr(), w.data_ptr(), ends.data_ptr(), rows, n_in, n_out, groups, n_out, n_out, n_in, t, 3, 1)
        work = Guarded(tb.lib.sxh_linear_bwd_workspace(C.byref(a)))
        torch.cuda.synchronize()
        rc = tb.lib.sxh_linear_bwd(tb.handle, C.byref(a), C.byref(st.LinearGrads(dx.at, dw.at, db.at, n_in, work.at, work.size)), None)
        assert rc == 0, tb.lib.sxh_last_error()
        assert dx.intact() and dw.intact() and db.intact() and work.intact(), "backward"


def test_a_guard_sees_a_write():
    """(what the test above goes by)"""
    for at in (GUARD - 1, GUARD + 100):
        k = Guarded(100)
        assert k.intact()
        k.all[at] = 0
        assert not k.intact()
