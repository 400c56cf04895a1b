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
    h.sample_code_of.argtypes = [C.c_double]
    h.sample_weight_of.restype = C.c_uint64
    for f in (h.sample_code_of, h.sample_bin_top_of):
        f.restype = C.c_uint32
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
    w, bins = np.zeros(len(x), np.uint64), np.zeros(len(x), np.int32)
    lead, code = np.zeros(len(x), np.uint32), np.zeros(len(x), np.uint32)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    host.sample_weights_of(C.c_float(top), C.c_float(t), p(x), len(x), p(w), p(bins), p(lead), p(code))
    return w, bins, lead, code


# a temperature whose inverse no float holds makes many bins of differences that are next to nothing
@pytest.mark.parametrize("t", [1e-45, 1e-42, 1e-40, 2.9e-39, 3e-39, 1e-30, 0.01, 1.0, 1e30, np.inf])
@pytest.mark.parametrize("size", [1e-44, 1e-41, 1e-39, 6e-38, 1e-20, 1.0, 1e5, 3e38])
def test_every_weight_has_a_bin_and_is_that_of_its_logit(host, t, size):
    r = np.random.default_rng(1)
    far = np.concatenate([r.random(4000), [0.0, 1.0], 10.0 ** r.uniform(-8, 0, 1000)])
    x = (-far * size).astype(np.float32)
    top = float(x.max())
    x = np.concatenate([x, np.array([np.nan, -np.inf], np.float32)])
    w, bins, lead, _ = weights(host, top, t, x)
    assert (bins >= 0).all() and (bins < host.sample_bins()).all()
    assert (w[-2:] == 0).all() and (lead[-2:] == 0).all()
    d = (np.float64(top) - x[:-2].astype(np.float64)) / np.float64(np.float32(t))
    one = 2.0 ** host.sample_unit()
    # a unit cut off, and half of the 27th bit, 2^-27 of itself; before it, half a 2^-31 of at least 2^-1 each for the
    # table's entry, the correction and 2^-9 more
    assert (np.abs(w[:-2] - one * np.exp(-d)) <= 1 + one * np.exp(-d) * (2.0**-27 + 2.1 * 2.0**-31)).all()


@pytest.mark.parametrize("vocab", [1000, 131075, 344064])
@pytest.mark.parametrize("below", [1, 5, 15, 19.7, 20, 21, 22, 22.1, 22.2, 23, 25, 28, 31, 31.8, 31.9, 33, 60])
def test_a_flat_tail_has_its_share_of_the_sum(host, vocab, below):
    """One token over vocab - 1 equal ones: the errors are all of one sign."""
    w = weights(host, 0.0, 1.0, np.full(8, -below, np.float32))[0]
    assert (w == w[0]).all()
    exact = (vocab - 1) * math.exp(-float(np.float32(below)))
    got = (vocab - 1) * int(w[0]) / 2.0 ** host.sample_unit()
    assert abs(got - exact) <= vocab * 2.0**-45 + exact * 2.0**-26.7
    assert 2 ** host.sample_unit() * vocab < 2**64


def test_codes_hold_and_order_the_weights(host):
    r = np.random.default_rng(2)
    unit = host.sample_unit()
    # every weight of up to 27 bits has a code, the weight comes back, and codes order as weights do
    xs = sorted({1, 2, 3, 2**26, 2**27 - 1, 2**27, 2**unit} | {int(m) << int(s) for m, s in zip(r.integers(1, 2**27, 3000), r.integers(0, unit - 26, 3000))})
    codes = [host.sample_code_of(float(x)) for x in xs]
    assert codes == sorted(set(codes)) and codes[0] == 1 << 26
    assert [host.sample_weight_of(c) for c in codes] == xs and host.sample_weight_of(0) == 0
    # bins follow on one another, from the largest weight down to none
    tops = [host.sample_bin_top_of(b) for b in range(host.sample_bins() + 1)]
    assert tops[0] == host.sample_code_of(2.0**unit) and tops[-1] == 0 and tops == sorted(tops, reverse=True)


def test_weights_lie_in_their_bins_and_their_leading_bits_say_nearly_what_they_are(host):
    r = np.random.default_rng(3)
    x = -r.random(20000).astype(np.float32) * 33
    w, bins, lead, code = weights(host, 0.0, 1.0, x)
    tops = np.array([host.sample_bin_top_of(b) for b in range(host.sample_bins() + 1)], np.int64)
    near, some = host.sample_near(), w > 0
    assert (code <= tops[bins] + near)[some].all() and (code + near > tops[bins + 1])[some].all()
    # 2^(unit - 15) = 2^30 to 2^31 times the leading bits, cut off, at 2^-(bin's power)
    said = lead.astype(np.float64) * 2.0 ** (host.sample_unit() - 16) / 2.0 ** (bins // 256)
    assert (np.abs(said - w) <= 1 + w * 2.0**-14 + 2.0 ** (host.sample_unit() - 16 - 31) * (bins == host.sample_bins() - 1))[some].all()


def test_neighbours_are_out_of_order_by_no_more_than_counts_as_near(host):
    for at in (0.5, 3.3, 9.9, 14.0, 20.5, 27.7, 30.5):
        x = np.float32(-at) + np.arange(40000, dtype=np.float32) * np.float32(2.0**-23 * max(1.0, 2.0 ** np.floor(np.log2(at))))
        code = weights(host, 0.0, 1.0, x)[3].astype(np.int64)
        highest = np.maximum.accumulate(code)
        assert (highest - code <= host.sample_near() // 2).all()


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
