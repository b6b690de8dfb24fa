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
