"""The learned heads' calls on tensors where a program does what a call does not expect (no GPU use)."""
import pytest
import torch


@pytest.fixture(scope="module")
def st():
    import splatx_torch
    return splatx_torch


class Raising:
    """A number or a truth value whose conversion raises."""

    def __init__(self, error):
        self.error = error

    def _raise(self):
        raise self.error

    __float__ = __bool__ = __index__ = _raise


def adamw(ops, **k):
    a = dict(params=[], grads=[], m=[], v=[], step=1, lr=1e-3, weight_decay=0.0, b1=0.9, b2=0.999, eps=1e-8, master=None, grad_scale=1.0,
             grad_norm=None, max_norm=0.0, m_scale=None, v_scale=None, seed=0)
    assert k.keys() <= a.keys()
    return ops.adamw(0, 0, 0, *{**a, **k}.values())


@pytest.mark.parametrize("error", [KeyboardInterrupt, ZeroDivisionError, MemoryError, RuntimeError])
def test_exceptions_of_a_conversion_are_the_callers(st, error):
    ops, x, bad = st._extension(), torch.ones(4, 8), Raising(error)
    for k in ("step", "lr", "weight_decay", "b1", "b2", "eps", "grad_scale", "max_norm", "seed"):
        with pytest.raises(error):
            adamw(ops, **{k: bad})
    with pytest.raises(error):
        ops.layer_norm_fwd(0, 0, 0, x, None, None, bad, None, True)
    with pytest.raises(error):
        ops.layer_norm_fwd(0, 0, 0, x, None, None, 1e-5, None, bad)
    for k in range(3):
        with pytest.raises(error):
            ops.layer_norm_bwd(0, 0, 0, x, x, x, x, None, None, *[bad if i == k else True for i in range(3)])


def test_what_is_no_number_is_refused(st):
    import splatx_hip as sh
    ops = st._extension()
    for bad in (Raising(TypeError), Raising(ValueError), Raising(OverflowError), "x", None, 10 ** 400):
        for k in ("lr", "step", "seed"):
            with pytest.raises(sh.SxInvalidArgument):
                adamw(ops, **{k: bad})


def test_eps_of_any_size_that_the_arithmetic_holds(st):
    """Refused for the missing backend alone, or for eps."""
    import splatx_hip as sh
    ops = st._extension()
    for eps, word in ((1e-30, "null backend"), (0.9, "null backend"), (1.0, "null backend"), (10.0, "null backend"), (1e30, "null backend"),
                      (0.0, "eps"), (9e-31, "eps"), (1.1e30, "eps"), (float("inf"), "eps"), (float("nan"), "eps"), (-1.0, "eps")):
        with pytest.raises(sh.SxInvalidArgument, match=word):
            adamw(ops, eps=eps)


def test_states_of_other_types_are_refused(st):
    """8-bit moments held as whole numbers would be taken for those numbers, not for the codes."""
    import splatx_hip as sh
    p = [torch.nn.Parameter(torch.randn(300)), torch.nn.Parameter(torch.randn(20, dtype=torch.bfloat16))]
    for bits in (32, 8):
        opt = st.AdamW(None, p, state_bits=bits)
        good = opt.state_dict()
        opt.load_state_dict(good)
        for k, dtype in (("exp_avg", torch.uint8), ("exp_avg_sq", torch.float64), ("master", torch.bfloat16)):
            bad = opt.state_dict()
            bad["state"][1][k] = bad["state"][1][k].float().to(dtype)
            with pytest.raises(sh.SxInvalidArgument):
                opt.load_state_dict(bad)
        with pytest.raises(sh.SxInvalidArgument):
            opt.load_state_dict({**good, "state_bits": 40 - bits})
        assert opt.steps == 0


@pytest.mark.parametrize("missing", ["TORCH=", "TORCH=/nowhere/torch", "PYTHON_INCLUDE=/nowhere", "PYTHON_INCLUDE=", "PYTHON=/nowhere/python3", None])
def test_the_library_is_built_without_the_extension_where_it_cannot_be(missing):
    """`make all` where torch, its headers or Python's are not there, looked over without running it."""
    import os
    import subprocess
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "splatx-metal_amd")
    r = subprocess.run(["make", "-n", "-B", "all"] + ([missing] if missing else []), cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lines = r.stdout.splitlines()
    assert any("-o build/libsplatx_hip.so" in x for x in lines)
    assert any("host/torch_ops.cpp" in x and "-o build/_splatx_torch.so" in x for x in "\n".join(lines).replace("\\\n", " ").splitlines()) == (missing is None)
