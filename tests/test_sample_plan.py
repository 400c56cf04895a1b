"""The arithmetic of sampling without a device (gollama_b200/csrc/sample_plan.h,
compiled for the host)."""
import ctypes as C
import math
import subprocess
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).parent


@pytest.fixture(scope="module")
def host():
    src, lib = HERE / "native" / "sample_host.cpp", HERE / "native" / "_build" / "libsample_host.so"
    lib.parent.mkdir(exist_ok=True)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True, capture_output=True)
    h = C.CDLL(str(lib))
    h.sample_goal_of.restype = C.c_uint64
    h.sample_goal_of.argtypes = [C.c_uint64, C.c_float]
    return h


@pytest.mark.parametrize("p", [1e-45, 1e-38, 1e-30, 1e-20, 5.4e-20, 5.5e-20, 1e-9, 0.5, 0.9, float(np.nextafter(np.float32(1), np.float32(0)))])
@pytest.mark.parametrize("all_", [1, 2**31, 3 * 2**31 + 1, 344064 << 31])
def test_a_share_of_a_sum_is_reached_by_some_token(host, p, all_):
    """The least whole number not below the share, one at least: a goal of zero has no token."""
    goal = host.sample_goal_of(all_, p)
    assert 1 <= goal <= all_
    exact = math.ceil(Fraction(float(np.float32(p))) * all_)
    assert goal == max(exact, 1)
