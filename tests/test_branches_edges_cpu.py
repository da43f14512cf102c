"""Argument checks of the calls that keep page bounds beside drafted tokens and
shared pages, without a GPU: every call here fails (or has nothing to do)
before the device is touched; the pointers are fake."""
import ctypes

import pytest

from test_branches_cpu import P
from test_paged_cpu import INVALID, LIB, LL3, MISALIGNED, OK, PagedCache, cache


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    p, i, ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
    lib.launch_kv_compact_bounds.argtypes = [ctypes.POINTER(PagedCache), p, p, ll, i, p, p, p, p]
    return lib


def _compact(lib, bounds=P, strides=LL3(256, 128, 64), **kw):
    return lib.launch_kv_compact_bounds(ctypes.byref(cache(**kw)), P, P, 4, 4, P, bounds, strides, None)


def test_compact_bounds_checks(lib):
    assert _compact(lib, strides=None) == INVALID
    for bad in (LL3(-1, 128, 64), LL3(256, -1, 64), LL3(256, 128, -1)):
        assert _compact(lib, strides=bad) == INVALID
    assert _compact(lib, bounds=0x1001) == MISALIGNED and _compact(lib, bounds=0x1002, dtype=2) == MISALIGNED
    assert _compact(lib, B=0) == OK and _compact(lib, heads=0) == INVALID
