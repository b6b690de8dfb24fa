"""The bounds on float32 keys by which the routing decides what 64 bits have to
decide again (csrc/route_bounds.h), compiled for the host: whatever the keys' errors
within their own bounds are, what counts as decided is."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "aethermoe_b200", "csrc")
SOURCE = """
#include "route_bounds.h"
extern "C" {
float key_slack(int sigmoid, float score, float key) { return aem::key_slack(sigmoid, score, key); }
float score_slack(int sigmoid, float top) { return aem::score_slack(sigmoid, top); }
float group_slack(float score, float largest) { return aem::group_slack(score, largest); }
int open_at_end(float key, float slack, float then, float score) { return aem::open_at_end(key, slack, then, score); }
int to_decide(int open) { return aem::to_decide(open); }
}
"""
U = 2.0 ** -24


@pytest.fixture(scope="module")
def bounds(tmp_path_factory):
    d = tmp_path_factory.mktemp("bounds")
    (d / "b.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-shared", "-fPIC", "-I", CSRC, str(d / "b.cpp"),
                    "-o", str(d / "b.so")], check=True)
    lib = ctypes.CDLL(str(d / "b.so"))
    lib.key_slack.argtypes = [ctypes.c_int, ctypes.c_float, ctypes.c_float]
    lib.score_slack.argtypes = [ctypes.c_int, ctypes.c_float]
    lib.group_slack.argtypes = [ctypes.c_float, ctypes.c_float]
    lib.open_at_end.argtypes = [ctypes.c_float] * 4
    lib.key_slack.restype = lib.score_slack.restype = lib.group_slack.restype = ctypes.c_float
    return lib


@pytest.mark.parametrize("sigmoid", [1, 0])
def test_scores(bounds, sigmoid):
    """No score's part of a key's bound is above the row's."""
    s = np.linspace(0.0, 1.0, 100001).astype(np.float32)
    of = np.array([bounds.key_slack(sigmoid, v, 0.0) for v in s])
    for top in (0.01, 0.3, 0.7525, 1.0):
        assert of[s <= top].max() <= bounds.score_slack(sigmoid, top)


@pytest.mark.parametrize("sigmoid", [1, 0])
@pytest.mark.parametrize("summed", [1, 2])
def test_groups(bounds, sigmoid, summed):
    """Two groups' values, each a key or the sum of two, in a row that has a larger score
    with a smaller key: their errors and the sums' roundings stay within the slack."""
    rng = np.random.default_rng(summed)
    for i in range(4000):
        if sigmoid:
            s = rng.choice([0.5, 0.7, 0.75, 0.8, 1.0], 2 * summed) * rng.choice([1.0, rng.uniform(0.9, 1.0)])
        else:
            s = rng.uniform(0.0, 0.2, 2 * summed)
        key = s + rng.choice([0.0, -0.4, -0.74, 0.3, 5.0])
        top = max(s.max(), rng.choice([s.max(), 0.9, 1.0]) if sigmoid else rng.choice([s.max(), 0.5]))
        largest = np.abs(key).max() * rng.choice([1.0, 1.5])
        errors = sum(bounds.key_slack(sigmoid, a, k) for a, k in zip(s, key))
        values = np.abs(key[:summed].sum()), np.abs(key[summed:].sum())
        need = errors + (sum(values) * U if summed == 2 else 0.0)
        assert bounds.group_slack(bounds.score_slack(sigmoid, top), largest) >= need, (s, key, top, largest)


@pytest.mark.parametrize("sigmoid", [1, 0])
def test_the_chosen_ones(bounds, sigmoid):
    """Where nothing is left to decide the keys' order is that of the real ones, and
    where only the order of the chosen ones is, none of them can lie below an expert
    that was not chosen."""
    rng = np.random.default_rng(4 + sigmoid)
    seen = [0, 0, 0]
    for i in range(20000):
        k, n = 3, 5
        s = (rng.choice([1e-6, 0.3, 0.75, 0.95, 1.0], n) if sigmoid else rng.choice([1e-6, 0.01, 0.4], n)).astype(np.float32)
        top = s.max()
        key = np.float32(rng.choice([0.0, 0.4, 1.5]))
        gaps = rng.choice([0.0, 0.5, 2.3, 2.6, 4.7, 6.0, 10.0], n) * rng.choice([1.0, 0.02 if sigmoid else 20.0])
        key = (key - np.cumsum(gaps) * U).astype(np.float32)
        slack = [bounds.key_slack(sigmoid, a, b) for a, b in zip(s, key)]
        score = bounds.score_slack(sigmoid, top)
        open_ = 0
        for j in range(k):
            if j + 1 < k:
                open_ |= 0 if np.float32(key[j] - key[j + 1]) > np.float32(slack[j]) + np.float32(slack[j + 1]) else 1
            else:
                open_ |= bounds.open_at_end(key[j], slack[j], key[j + 1], score)
        what = bounds.to_decide(open_)
        seen[what] += 1
        real = np.array(slack) / 1.001, key.astype(np.float64)  # (the comparisons round too)
        if what < 2:
            assert min(real[1][:k] - real[0][:k]) > max(real[1][k:] + real[0][k:]), (s, key, open_)
        if what == 0:
            for j in range(k - 1):
                assert real[1][j] - real[0][j] > max(real[1][j + 1:] + real[0][j + 1:]), (s, key)
    assert min(seen) > 100, seen
