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
    c = ctypes.POINTER(PagedCache)
    lib.launch_kv_compact_bounds.argtypes = [c, p, p, ll, i, p, p, p, p]
    lib.launch_kv_fork_bounds.argtypes = [c, p, p, p, i, p, p, p, p, p, p, p, ctypes.c_size_t, p]
    return lib


def _compact(lib, bounds=P, strides=LL3(256, 128, 64), **kw):
    return lib.launch_kv_compact_bounds(ctypes.byref(cache(**kw)), P, P, 4, 4, P, bounds, strides, None)


def _fork(lib, bounds=P, strides=LL3(256, 128, 64), space=P, size=1 << 20, **kw):
    return lib.launch_kv_fork_bounds(ctypes.byref(cache(**kw)), P, P, P, 2, P, P, P, P, bounds, strides, space, size, None)


@pytest.mark.parametrize("call", [_compact, _fork])
def test_bounds_checks(lib, call):
    assert call(lib, strides=None) == INVALID
    for bad in (LL3(-1, 128, 64), LL3(256, -1, 64), LL3(256, 128, -1)):
        assert call(lib, strides=bad) == INVALID
    assert call(lib, bounds=0x1001) == MISALIGNED and call(lib, bounds=0x1002, dtype=2) == MISALIGNED
    assert call(lib, heads=0) == INVALID


def test_calls_without_work_or_room(lib):
    assert _compact(lib, B=0) == OK
    assert _fork(lib, space=None) == INVALID and _fork(lib, size=8) == INVALID
