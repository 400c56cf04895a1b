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


def weights(host, top, t, x):
    x = np.ascontiguousarray(x, np.float32)
    w, bins, lead = np.zeros(len(x), np.uint32), np.zeros(len(x), np.int32), np.zeros(len(x), np.uint32)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    host.sample_weights_of(C.c_float(top), C.c_float(t), p(x), len(x), p(w), p(bins), p(lead))
    return w, bins, lead


# a temperature whose inverse no float holds makes many bins of differences that are next to nothing
@pytest.mark.parametrize("t", [1e-45, 1e-42, 1e-40, 2.9e-39, 3e-39, 1e-30, 0.01, 1.0, 1e30, np.inf])
@pytest.mark.parametrize("size", [1e-44, 1e-41, 1e-39, 6e-38, 1e-20, 1.0, 1e5, 3e38])
def test_every_weight_has_a_bin_and_is_that_of_its_logit(host, t, size):
    r = np.random.default_rng(1)
    far = np.concatenate([r.random(4000), [0.0, 1.0], 10.0 ** r.uniform(-8, 0, 1000)])
    x = (-far * size).astype(np.float32)
    top = float(x.max())
    x = np.concatenate([x, np.array([np.nan, -np.inf], np.float32)])
    w, bins, lead = weights(host, top, t, x)
    assert (bins >= 0).all() and (bins < host.sample_bins()).all()
    assert (w[-2:] == 0).all() and (lead[-2:] == 0).all()
    d = (np.float64(top) - x[:-2].astype(np.float64)) / np.float64(np.float32(t))
    assert (np.abs(w[:-2] - 2.0**31 * np.exp(-d)) <= 1.5 + 2.0**-9).all()  # half a unit of the table's entry, the correction, the shift


def test_no_store_to_another_cta_before_the_cluster_has_started():
    """Every thread arrives at the cluster's barrier first thing and waits for it before the first store to the
    shared memory of the row's other CTAs; each barrier is arrived at once and waited for once."""
    text = (HERE.parent / "gollama_b200" / "csrc" / "sample.cu").read_text()
    kernel = text[text.index("sample_kernel(const Sample a) {"):text.index('extern "C"')]
    arrive, wait = kernel.index("cluster.barrier_arrive();"), kernel.index("cluster.barrier_wait();")
    stores = [kernel.index(x) for x in ("o.tops[rank] =", "o.sums[rank] =", "o.finites[rank] =")]
    assert arrive < kernel.index("const float* src") < wait < min(stores)
    assert kernel.count("barrier_arrive") == kernel.count("barrier_wait") == 1
    # before the wait nothing goes through a peer's address, returns, or uses the barrier for itself
    before = kernel[:wait]
    assert before.count("map_shared_rank") == 1 and "lead." not in before and "return" not in before and "cluster.sync" not in before
