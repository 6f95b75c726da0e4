"""The learned heads' C structs, their workspace sizes and what is refused before a device is touched (no GPU use), and the
reference the GPU tests compare with, checked against torch's own float8 type."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

import learned_ref as ref

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def st():
    import splatx_torch
    return splatx_torch


@pytest.fixture(scope="module")
def lib():
    import splatx_hip
    return splatx_hip.load_library()


def test_struct_layouts_match_the_header(st, tmp_path):
    pairs = {"sxh_queue": st.Queue, "sxh_layer_norm_inputs": st.LayerNormInputs, "sxh_layer_norm_outputs": st.LayerNormOutputs,
             "sxh_layer_norm_grads_in": st.LayerNormGradsIn, "sxh_layer_norm_grads": st.LayerNormGrads,
             "sxh_norm_tensor": st.NormTensor, "sxh_adamw_tensor": st.AdamWTensor, "sxh_adamw_params": st.AdamWParams}
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in t._fields_)
             for c, t in pairs.items()]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "splatx_hip.h"\nint main(void) {' + "\n".join(lines) + "return 0;}")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(REPO, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = [v for t in pairs.values() for v in [C.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]]
    assert got == want


def test_refusals_without_a_device(st, lib):
    x = 1 << 20  # never read: every call below is refused for something else first
    i = st.LayerNormInputs(x, None, None, None, 4, 8, 8, 0, 1e-5, 0, 0)
    o = st.LayerNormOutputs(x, None, None, None, 8, 0)

    def refused(rc, word):
        assert rc == 1 and word.encode() in lib.sxh_last_error(), lib.sxh_last_error()

    refused(lib.sxh_layer_norm_fwd(None, C.byref(i), C.byref(o), None), "null backend")
    refused(lib.sxh_layer_norm_fwd(None, None, C.byref(o), None), "null inputs")
    for name, v, word in (("type", 3, "type"), ("weight_type", 1, "weight_type"), ("eps", 0.0, "eps"), ("eps", math.nan, "eps"),
                          ("residual", x, "h is written")):
        bad = st.LayerNormInputs.from_buffer_copy(i)
        setattr(bad, name, v)
        refused(lib.sxh_layer_norm_fwd(None, C.byref(bad), C.byref(o), None), word)
    g = st.LayerNormGradsIn(x, x, None, x, x, None, 4, 8, 8, 8, 0, 0, 0)
    refused(lib.sxh_layer_norm_bwd(None, C.byref(g), C.byref(st.LayerNormGrads(None, None, None, 8, None, 0)), None), "no gradient")
    p = st.AdamWParams(1, 0, 0.9, 0.999, 1e-8, None, 0.0, 1.0, 32)
    lib.sxh_adamw.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]
    refused(lib.sxh_adamw(None, None, 0, C.byref(p), None), "null backend")
    refused(lib.sxh_adamw(None, None, 1, C.byref(p), None), "null tensors")
    for name, v, word in (("step", 0, "step"), ("state_bits", 16, "state_bits"), ("b1", 1.0, "b1"), ("b2", -0.1, "b2"), ("eps", 0.0, "eps"),
                          ("max_norm", 1.0, "grad_norm"), ("max_norm", -1.0, "max_norm"), ("grad_scale", 0.0, "grad_scale"),
                          ("grad_scale", math.inf, "grad_scale")):
        bad = st.AdamWParams.from_buffer_copy(p)
        setattr(bad, name, v)
        refused(lib.sxh_adamw(None, None, 0, C.byref(bad), None), word)
    lib.sxh_grad_norm.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    refused(lib.sxh_grad_norm(None, None, 0, None, None, 0, None), "null backend")
    refused(lib.sxh_grad_norm(None, None, -1, None, None, 0, None), "tensors")


def test_workspaces(lib):
    f, g = lib.sxh_layer_norm_bwd_workspace, lib.sxh_grad_norm_workspace
    f.argtypes, f.restype, g.argtypes, g.restype = [C.c_int64] * 2, C.c_int64, [C.c_int64], C.c_int64
    for rows in (0, 1, 1000, 10 ** 6, 10 ** 12):
        for width in (1, 48, 4096, 1 << 24):
            assert 8 * width <= f(rows, width) <= max(64 << 20, 16 * width)  # both sums of a part of the rows at least
    assert f(-1, 4) == f(4, 0) == f(4, (1 << 24) + 1) == 0
    assert 0 < g(0) <= g(1) <= g(1000) and g(-1) == 0


def test_reference_codes_are_e4m3():
    v = ref.code_values()
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(v, 999.0), torch.nan_to_num(t, 999.0))


def test_reference_rounding_is_unbiased_and_bits_are_even():
    """A value's codes average to it over the elements' bits; each of the 32 bits is one half the time and two of a word do
    not go together (5 sigma of 2^18 draws, 1 %)."""
    n = 1 << 18
    bits = ref.random_bits(12345, 7, 3, n)
    ones = torch.stack([(bits >> k & 1).double() for k in range(32)])
    assert (ones.mean(1) - 0.5).abs().max() < 0.005
    joint = (ones @ ones.t() / n - 0.25).fill_diagonal_(0)
    assert joint.abs().max() < 0.005
    after = ones[:, 1:] @ ones[:, :-1].t() / (n - 1) - 0.25  # a word and the next element's
    assert after.abs().max() < 0.005
    for value in (0.3, 0.0101, 3e-5):
        x = torch.full((n,), value, dtype=torch.float64)
        x[::256] = 1.0
        codes, scale = ref.encode(x, bits & 0xFFFF, False)
        got = ref.decode(codes, scale)[torch.arange(n) % 256 != 0]
        assert abs(float(got.mean()) - value) <= 5 * float(got.std()) / math.sqrt(n) + value * 2.0 ** -15


def test_the_nearest_code_would_hold_a_second_moment_still():
    """Why the roots are not rounded to nearest: a step moves one by a two-thousandth, the codes are a sixteenth apart."""
    v = torch.full((256,), 0.25, dtype=torch.float64)
    v[0] = 1.0
    half = torch.full((256,), 0x8000)
    codes, scale = ref.encode(v.sqrt(), half, True)
    for _ in range(100):  # decays to 0.25 * 0.999^100 = 0.226 in truth
        root = ref.decode(codes, scale)
        new = 0.999 * root.square()
        new[0] = 1.0
        codes, scale = ref.encode(new.sqrt(), half, True)
    assert float(ref.decode(codes, scale)[1]) ** 2 == pytest.approx(0.25, rel=0.01)


def test_tensor_calls_refuse_host_memory(st, lib):
    """The calls on tensors raise the binding's exceptions, also for arguments that are no tensors or no numbers."""
    import splatx_hip as sh
    import torch
    ops = st._extension()
    x = torch.ones(4, 8)
    for f, args in ((ops.layer_norm_fwd, (x, None, None, 1e-5, None, True)), (ops.layer_norm_fwd, (None, None, None, 1e-5, None, True)),
                    (ops.layer_norm_bwd, (x, x, x, x, None, None, True, True, True)), (ops.grad_norm, ([x],)), (ops.grad_norm, (x,)),
                    (ops.grad_norm, ([x.numpy()],)), (ops.grad_norm, ()),
                    (ops.adamw, ([x], [x], [x], [x], 1, 1e-3, 0.0, 0.9, 0.999, 1e-8, None, 1.0, None, 0.0, None, None, 0)),
                    (ops.adamw, ([], [], [], [], 1.5, 1e-3, 0.0, 0.9, 0.999, 1e-8, None, 1.0, None, 0.0, None, None, 0)),
                    (ops.adamw, ([], [], [], [], 1, "x", 0.0, 0.9, 0.999, 1e-8, None, 1.0, None, 0.0, None, None, 0)),
                    (ops.adamw, ([], [], [], [x], 1, 1e-3, 0.0, 0.9, 0.999, 1e-8, None, 1.0, None, 0.0, None, None, 0)),
                    (ops.adamw, ([], [], [], [], 1, 1e-3, 0.0, 0.9, 0.999, 1e-8, None, 1.0, None, 0.0, [], None, 0)),
                    (ops.adamw, ([], [], [], [], 1, 1e-3, 0.0, 0.9, 0.999, 1e-8, None, 1.0, None, 0.0, None, None, 2 ** 64))):
        with pytest.raises(sh.SxInvalidArgument):
            f(0, 0, 0, *args)
    with pytest.raises(sh.SxInvalidArgument, match="null backend"):
        ops.adamw(0, 0, 0, [], [], [], [], 1, 1e-3, 0.0, 0.9, 0.999, 1e-8, None, 1.0, None, 0.0, None, None, 0)
