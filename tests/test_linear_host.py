"""The linear layers' C structs, workspace sizes and what is refused before a device is touched (no GPU use)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import linear_ref as ref

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def st():
    import splatx_torch
    return splatx_torch


@pytest.fixture(scope="module")
def lib():
    import splatx_hip
    lib = splatx_hip.load_library()
    for name in ("sxh_linear_fwd_workspace", "sxh_linear_bwd_workspace"):
        f = getattr(lib, name)
        f.argtypes, f.restype = [C.c_void_p], C.c_int64
    return lib


def test_struct_layouts_match_the_header(st, tmp_path):
    pairs = {"sxh_linear_inputs": st.LinearInputs, "sxh_linear_outputs": st.LinearOutputs, "sxh_linear_grads_in": st.LinearGradsIn,
             "sxh_linear_grads": st.LinearGrads}
    field = lambda f: f[0].rstrip("_")  # noqa: E731
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {field(f)}));' for f in t._fields_)
             for c, t in pairs.items()]
    lines += [f'printf("%d\\n", SXH_ACT_{name.upper()});' for name in st.ACTIVATIONS]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "splatx_hip.h"\nint main(void) {' + "\n".join(lines) + "return 0;}")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(REPO, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = [v for t in pairs.values() for v in [C.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]]
    assert got == want + list(st.ACTIVATIONS.values())


def test_refusals_without_a_device(st, lib):
    x = 1 << 20  # never read: every call below is refused for something else first

    def refused(rc, word):
        assert rc == 1 and word.encode() in lib.sxh_last_error(), lib.sxh_last_error()

    i = st.LinearInputs(x, x, None, None, None, 4, 8, 8, 0, 8, 0, 0, 0, 0)
    o = st.LinearOutputs(x, None, 8, 0, None, 0)
    g = st.LinearGradsIn(x, None, x, x, None, 4, 8, 8, 0, 8, 0, 8, 0, 0, 0)
    go = st.LinearGrads(x, x, x, 8, None, 0)
    fwd = lambda a: lib.sxh_linear_fwd(None, C.byref(a), C.byref(o), None)  # noqa: E731
    bwd = lambda a, b=go: lib.sxh_linear_bwd(None, C.byref(a), C.byref(b), None)  # noqa: E731
    refused(fwd(i), "null backend")
    refused(bwd(g), "null backend")
    refused(lib.sxh_linear_fwd(None, None, C.byref(o), None), "null inputs")
    refused(lib.sxh_linear_bwd(None, C.byref(g), None, None), "null inputs")
    for name, v, word in (("type", 3, "type"), ("activation", 5, "activation"), ("in_", 0, "in and out"), ("out", 0, "in and out"),
                          ("in_", 1 << 25, "in and out"), ("rows", -1, "rows"), ("rows", 1 << 50, "larger"), ("groups", -1, "groups"),
                          ("groups", 32769, "groups"), ("groups", 2, "ends"), ("ends", x, "ends"), ("clear", 2, "clear")):
        for cls, call, base in ((st.LinearInputs, fwd, i), (st.LinearGradsIn, bwd, g)):
            bad = cls.from_buffer_copy(base)
            setattr(bad, name, v)
            refused(call(bad), word)
    wide = st.LinearInputs.from_buffer_copy(i)
    wide.in_ = wide.out = 1 << 24
    refused(fwd(wide), "larger")
    refused(bwd(g, st.LinearGrads(None, None, None, 8, None, 0)), "no gradient")
    for pre, act in ((x, 0), (None, 2)):
        bad = st.LinearGradsIn.from_buffer_copy(g)
        bad.pre, bad.activation = pre, act
        refused(bwd(bad), "pre is given")


def test_workspaces(st, lib):
    at = 1 << 20  # never read

    def f(rows, n_in, n_out, groups, t, x=at, stride=None):
        a = st.LinearInputs(x, at, None, None, at if groups else None, rows, n_in, n_out, groups, n_in if stride is None else stride, 0, t, 0, 0)
        return lib.sxh_linear_fwd_workspace(C.byref(a))

    def g(rows, n_in, n_out, groups, t, x=at, stride=None):
        a = st.LinearGradsIn(at, at, x, at, at if groups else None, rows, n_in, n_out, groups, n_out, n_out, n_in if stride is None else stride, t, 2, 0)
        return lib.sxh_linear_bwd_workspace(C.byref(a))

    for rows in (0, 1, 13, 1000, 10 ** 6, 10 ** 9):
        for n_in, n_out in ((1, 1), (16, 64), (64, 64), (2048, 8192), (8192, 1), (1, 1 << 20)):
            for groups in (0, 1, 7, 300, 32768):
                for t in (0, 1, 2):
                    # some tens of MiB for partial sums, and a copy of what does not lie as the products read it: of x and the
                    # weights; for the backward also of dz
                    rows_bytes, weights = 4 * rows * (n_in + 16), 4 * max(groups, 1) * n_out * (n_in + 16)
                    assert 0 <= f(rows, n_in, n_out, groups, t) <= (64 << 20) + rows_bytes + weights
                    assert 0 <= g(rows, n_in, n_out, groups, t) <= (300 << 20) + rows_bytes + 4 * rows * (n_out + 16) + 2 * weights + 2048 * 8 * n_in * min(n_out, 256)
    # whole lines are read where they lie, others copied: rows of x, and for widths that are no multiple of 16 bytes the weights
    assert f(100_000, 1024, 1024, 0, 1) == 0
    assert f(100_000, 1024, 1024, 0, 1, x=at + 2) >= 100_000 * 2048 and f(100_000, 1024, 1024, 0, 1, stride=1025) >= 100_000 * 2048
    assert f(100_000, 1023, 1024, 0, 1, stride=1024) >= 2 * 1024 * 1024 and f(100_000, 1024, 1024, 0, 1, stride=0) == 0
    assert g(100_000, 1024, 1024, 0, 1, stride=1025) >= g(100_000, 1024, 1024, 0, 1) + 100_000 * 2048 - (300 << 20)
    for bad in ((-1, 4, 4, 0, 0), (4, 0, 4, 0, 0), (4, 4, 0, 0, 0), (4, 4, 4, -1, 0), (4, 4, 4, 32769, 0), (4, 4, 4, 0, 3), (1 << 60, 4, 4, 0, 0)):
        assert f(*bad) == g(*bad) == 0
    assert lib.sxh_linear_fwd_workspace(None) == lib.sxh_linear_bwd_workspace(None) == 0


def test_tensor_calls_refuse_host_memory(st):
    import splatx_hip as sh
    ops = st._extension()
    x, w = torch.ones(4, 8), torch.ones(3, 8)
    for f, args in ((ops.linear_fwd, (x, w, None, None, 0, None, False)), (ops.linear_fwd, (None, w, None, None, 0, None, False)),
                    (ops.linear_fwd, (x, w, None, None, "relu", None, False)), (ops.linear_fwd, ()),
                    (ops.linear_bwd, (x, x, w, None, None, 0, True, True, True)), (ops.linear_bwd, (x, x, w, None, None, 0, True, True))):
        with pytest.raises(sh.SxInvalidArgument):
            f(0, 0, 0, *args)
    for name in ("tanh", None, 1, []):
        with pytest.raises(sh.SxInvalidArgument, match="activation must be one of"):
            st._act(name)
    with pytest.raises(sh.SxInvalidArgument, match="ends"):
        st._ends(None)


@pytest.mark.parametrize("name", ref.ACTS)
def test_reference_slopes_are_the_activations(name):
    """Against differences in 64 bits, about no corner."""
    z = torch.linspace(-6, 6, 997, dtype=torch.float64) + 1e-3
    h = 1e-5
    want = (ref.act(z + h, name) - ref.act(z - h, name)) / (2 * h)
    assert (ref.slope(z, name) - want).abs().max() <= 1e-9
    if name != "none":
        t = {"relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid}[name]
        assert (ref.act(z, name) - t(z)).abs().max() <= 1e-15 * 8


def test_reference_gradients_are_torchs():
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((7, 4), (2, 3, 4), (2, 3)))
    dy = torch.randn(7, 3, generator=g, dtype=torch.float64)
    z = torch.cat([x[:2] @ w[0].t() + b[0], x[2:6] @ w[1].t() + b[1]])
    torch.nn.functional.gelu(z).backward(dy[:6])
    ends = torch.tensor([2, 6])
    from unittest import mock
    with mock.patch.dict(ref.UNIT, {torch.float64: 0.0}), mock.patch.dict(ref.TINY, {torch.float64: 0.0}), mock.patch.dict(ref.ACT, {torch.float64: 0.0}):
        pre = torch.zeros(7, 3, dtype=torch.float64)
        pre[:6] = z.detach()
        got, _ = ref.bwd(dy, x.detach(), w.detach(), pre, "gelu", ends)
    for a, want in zip(got, (x.grad, w.grad, b.grad)):
        assert (a - want).abs().max() <= 1e-12
