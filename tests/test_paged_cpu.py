"""Argument checks of the paged-cache entry points, without a GPU: every call
here fails (or has nothing to do) before the device is touched; the pointers
are fake."""
import ctypes
import os

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "rocm_attn_b200", "librocm_attn.so")
OK, INVALID, UNSUPPORTED, MISALIGNED = 0, 1, 2, 3
LL3 = ctypes.c_longlong * 3


class PagedCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("num_pages", ctypes.c_int), ("heads", ctypes.c_int),
                ("page_size", ctypes.c_int), ("D", ctypes.c_int), ("dtype", ctypes.c_int), ("k_strides", LL3),
                ("v_strides", LL3), ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_longlong),
                ("table_width", ctypes.c_int), ("seq_lens", ctypes.c_void_p), ("B", ctypes.c_int)]


def cache(**kw):
    d = dict(k=0x1000, v=0x1000, num_pages=4, heads=2, page_size=16, D=64, dtype=0, k_strides=LL3(2048, 1024, 64),
             v_strides=LL3(2048, 1024, 64), block_table=0x1000, table_stride=4, table_width=4, seq_lens=0x1000, B=1)
    d.update(kw)
    return PagedCache(**d)


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    p, i, ll, sz, b = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t, ctypes.c_bool
    c = ctypes.POINTER(PagedCache)
    lib.attn_decode_workspace_bytes.argtypes = [c, i, b, i, b, ctypes.POINTER(sz)]
    lib.launch_attn_decode.argtypes = [c, p, p, p, i, ctypes.c_float, p, i, p, p, p, sz, p]
    lib.launch_kv_append.argtypes = [c, p, p, p, p, i, p, p, p, p]
    lib.launch_kv_page_bounds.argtypes = [c, p, p, p]
    lib.kv_select_pages_workspace_bytes.argtypes = [c, ctypes.POINTER(sz)]
    lib.launch_kv_select_pages.argtypes = [c, p, p, i, p, p, i, p, p, sz, p]
    lib.launch_kv_evict.argtypes = [c, p, p, p, ll, i, i, i, p, p, p, p]
    return lib


CALLS = {
    "decode": lambda lib, c: lib.launch_attn_decode(c, 0x1000, None, 0x1000, 4, -1.0, None, 0, None, None, 0x1000,
                                                    1 << 30, None),
    "append": lambda lib, c: lib.launch_kv_append(c, 0x1000, LL3(), 0x1000, LL3(), 1, None, None, None, None),
    "bounds": lambda lib, c: lib.launch_kv_page_bounds(c, 0x1000, LL3(), None),
    "select": lambda lib, c: lib.launch_kv_select_pages(c, 0x1000, None, 4, 0x1000, LL3(), 2, 0x1000, 0x1000, 1 << 30,
                                                        None),
    "evict": lambda lib, c: lib.launch_kv_evict(c, 0x1000, LL3(), 0x1000, 4, 4, 8, 2, 0x1000, 0x1000, 0x1000, None),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("bad,status", [
    (dict(dtype=3), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(D=257), UNSUPPORTED), (dict(D=0), INVALID),
    (dict(heads=0), INVALID), (dict(page_size=0), INVALID), (dict(num_pages=-1), INVALID), (dict(B=-1), INVALID),
    (dict(table_width=-1), INVALID), (dict(table_stride=-4), INVALID), (dict(block_table=None), INVALID),
    (dict(seq_lens=None), INVALID), (dict(page_size=1 << 20, table_width=1 << 11), INVALID),
    (dict(seq_lens=0x1002), MISALIGNED), (dict(block_table=0x1001), MISALIGNED), (dict(B=0), OK)], ids=str)
def test_cache_checks(lib, name, bad, status):
    assert CALLS[name](lib, ctypes.byref(cache(**bad))) == status


@pytest.mark.parametrize("name,bad,status", [
    (n, bad, st) for n in ("decode", "append", "evict")
    for bad, st in ((dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k_strides=LL3(-1, 1, 1)), INVALID),
                    (dict(v_strides=LL3(1, 1, -1)), INVALID), (dict(k=0x1001), MISALIGNED),
                    (dict(v=0x1002, dtype=2), MISALIGNED))] + [("bounds", dict(k=None), INVALID)])
def test_cache_tensor_checks(lib, name, bad, status):
    assert CALLS[name](lib, ctypes.byref(cache(**bad))) == status


def test_null_cache(lib):
    for call in CALLS.values():
        assert call(lib, None) == INVALID


def _decode(lib, Hq=4, q=0x1000, out=0x1000, pages=None, n=0, weights=None, ws=None, space=0x1000, strides=None, **kw):
    return lib.launch_attn_decode(ctypes.byref(cache(**kw)), q, strides, out, Hq, -1.0, pages, n, weights, ws, space, 0,
                                  None)


def test_decode_checks(lib):
    two = (ctypes.c_longlong * 2)
    assert _decode(lib, Hq=3) == INVALID and _decode(lib, Hq=-2) == INVALID
    assert _decode(lib, q=None) == INVALID and _decode(lib, out=None) == INVALID and _decode(lib, space=None) == INVALID
    assert _decode(lib, strides=two(-1, 64)) == INVALID
    assert _decode(lib, pages=0x1000, n=-1) == INVALID
    assert _decode(lib, pages=0x1000, n=1 << 28) == INVALID
    assert _decode(lib, pages=0x1000, n=2, weights=0x1000, ws=two(64, 64)) == UNSUPPORTED
    assert _decode(lib, weights=0x1000) == INVALID
    assert _decode(lib, weights=0x1000, ws=two(-1, 1)) == INVALID
    assert _decode(lib, weights=0x1002, ws=two(128, 64)) == MISALIGNED
    assert _decode(lib, q=0x1001) == MISALIGNED and _decode(lib, out=0x1001) == MISALIGNED
    assert _decode(lib, space=0x1008) == MISALIGNED and _decode(lib, pages=0x1002, n=1) == MISALIGNED
    assert _decode(lib, Hq=0) == OK and _decode(lib, B=0) == OK
    assert _decode(lib, B=1 << 16, Hq=1 << 16) == INVALID
    assert _decode(lib, B=1 << 16, weights=0x1000, ws=two(64, 64)) == UNSUPPORTED
    n = ctypes.c_size_t(7)
    assert lib.attn_decode_workspace_bytes(ctypes.byref(cache()), 4, False, 0, False, None) == INVALID
    assert lib.attn_decode_workspace_bytes(ctypes.byref(cache()), 3, False, 0, False, ctypes.byref(n)) == INVALID
    assert lib.attn_decode_workspace_bytes(ctypes.byref(cache(B=0)), 4, False, 0, False, ctypes.byref(n)) == OK
    assert n.value == 0


def test_append_checks(lib):
    def call(k=0x1000, ks=LL3(), v=0x1000, vs=LL3(), S=1, new=None, bounds=None, bs=None, **kw):
        return lib.launch_kv_append(ctypes.byref(cache(**kw)), k, ks, v, vs, S, new, bounds, bs, None)
    assert call(S=-1) == INVALID and call(S=0) == OK
    assert call(k=None) == INVALID and call(v=None) == INVALID and call(ks=None) == INVALID and call(vs=None) == INVALID
    assert call(ks=LL3(0, -1, 0)) == INVALID
    assert call(bounds=0x1000) == INVALID and call(bounds=0x1000, bs=LL3(0, 0, -1)) == INVALID
    assert call(k=0x1001) == MISALIGNED and call(bounds=0x1001, bs=LL3()) == MISALIGNED and call(new=0x1002) == MISALIGNED


def test_select_checks(lib):
    def call(q=0x1000, qs=None, Hq=4, bounds=0x1000, bs=LL3(), top=2, pages=0x1000, space=0x1000, size=1 << 20, **kw):
        return lib.launch_kv_select_pages(ctypes.byref(cache(**kw)), q, qs, Hq, bounds, bs, top, pages, space, size, None)
    assert call(top=0) == INVALID and call(Hq=5) == INVALID and call(q=None) == INVALID and call(bounds=None) == INVALID
    assert call(bs=None) == INVALID and call(bs=LL3(-1, 0, 0)) == INVALID and call(pages=None) == INVALID
    assert call(space=None) == INVALID and call(size=8) == INVALID and call(heads=65536, Hq=0) == INVALID
    assert call(q=0x1001) == MISALIGNED and call(pages=0x1001) == MISALIGNED and call(space=0x1004) == MISALIGNED
    n = ctypes.c_size_t()
    assert lib.kv_select_pages_workspace_bytes(ctypes.byref(cache(k=None, v=None, B=3)), ctypes.byref(n)) == OK
    assert n.value >= 3 * 2 * 4 * 8
    assert lib.kv_select_pages_workspace_bytes(ctypes.byref(cache()), None) == INVALID


def test_evict_checks(lib):
    def call(w=0x1000, ws=LL3(), table=0x1000, stride=4, width=4, budget=8, recent=2, nw=0x1000, kept=0x1000, nl=0x1000,
             **kw):
        return lib.launch_kv_evict(ctypes.byref(cache(**kw)), w, ws, table, stride, width, budget, recent, nw, kept, nl,
                                   None)
    assert call(budget=0) == INVALID and call(budget=65) == INVALID and call(recent=-1) == INVALID
    assert call(recent=9) == INVALID and call(stride=-1) == INVALID and call(width=-1) == INVALID
    for name in ("w", "ws", "table", "nw", "kept", "nl"):
        assert call(**{name: None}) == INVALID
    assert call(w=0x1002) == MISALIGNED and call(nl=0x1001) == MISALIGNED
    assert call(ws=LL3(-1, 0, 0)) == INVALID


def test_python_names_and_devices():
    import rocm_attn_b200 as ra
    import rocm_attn_op

    for name in ("attn_decode", "kv_append", "kv_page_bounds", "kv_select_pages", "kv_evict"):
        assert getattr(rocm_attn_op, name) is getattr(ra, name) and name in ra.__all__
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    t, n, w = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, 32)
    for call in (lambda: ra.attn_decode(q, k, k, t, n), lambda: ra.kv_append(q, q, k, k, t, n),
                 lambda: ra.kv_page_bounds(k, t, n), lambda: ra.kv_select_pages(q, k, t, n, 16, 1),
                 lambda: ra.kv_evict(k, k, t, n, w, t, 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
