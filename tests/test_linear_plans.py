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
