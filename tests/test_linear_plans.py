"""The linear layers' plans (csrc/sx_linear_plan.h) over all sizes: what each launch asks for is what a workgroup can have (no GPU
use)."""
import os
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plans") / "plans")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wno-unused-function", "-I", os.path.join(REPO, "splatx-metal_amd", "csrc"),
                    os.path.join(REPO, "tests", "linear_plans.cpp"), "-o", exe], check=True)
    return subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines()


def test_every_plan_fits(lines):
    assert lines[-1].startswith("looked at ") and int(lines[-1].split()[-1]) > 1_000_000
    assert not lines[:-1], f"{len(lines) - 1} plans do not fit, first {lines[0]}"


@pytest.mark.parametrize("t,size", [(0, 4), (1, 2), (2, 2)])
def test_the_widest_rows_are_not_copied(t, size):
    """A copy has rows as wide: it would put none of them nearer to each other."""
    import ctypes as C

    import splatx_hip
    import splatx_torch as st
    lib, at = splatx_hip.load_library(), 1 << 20  # (never read)
    f, g = lib.sxh_linear_fwd_workspace, lib.sxh_linear_bwd_workspace
    for k in (f, g):
        k.argtypes, k.restype = [C.c_void_p], C.c_int64
    wide, rows, n = 1 << 24, 200, 128
    assert f(C.byref(st.LinearInputs(at, at, None, None, None, rows, wide, n, 0, wide, 0, t, 0, 0))) <= 64 << 20
    assert g(C.byref(st.LinearGradsIn(at, None, at, at, None, rows, wide, n, 0, n, 0, wide, t, 0, 0))) <= 64 << 20
    # rows of 16 bits further apart than that are (floats are read where they lie)
    assert t == 0 or f(C.byref(st.LinearInputs(at, at, None, None, None, rows, 1024, n, 0, 1 << 25, 0, t, 0, 0))) >= rows * 1024 * size
