"""The 8-bit products index rows in 32 bits, a tile of 256 past the last one included:
more rows than that leave room for are refused before anything else is looked at.
On any host; the handle and the pointers stand for ones that are never followed."""
import ctypes

import pytest

from aethermoe_b200 import _lib

P = 4096


class Weight(ctypes.Structure):
    """A weight of one group of 1 x 1."""
    _fields_ = [("device", ctypes.c_int), ("sizes", ctypes.c_int64 * 5), ("data", ctypes.c_void_p),
                ("scale", ctypes.c_void_p)]


@pytest.mark.parametrize("M", [2 ** 31 - 256, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
def test_rows_past_32_bits(M):
    w = Weight(0, (1, 1, 1, 1, 1), P, P)
    h, L = ctypes.addressof(w), _lib.lib()
    assert L.aem_fp8gemm(h, 0, 0, P, _lib.E4M3, 16, P, 4, M, P, _lib.F32, 1, None, 0, None) == _lib.AEM_EINVAL
    assert b"too many" in L.aem_last_error()
    assert L.aem_grouped_fp8gemm(h, P, 0, P, _lib.E4M3, 16, P, 4, M, P, _lib.F32, 1, 0, 0, None, 0,
                                 None) == _lib.AEM_EINVAL
    assert b"too many" in L.aem_last_error()
