"""Argument checks of the operators for drafted tokens and shared pages, without
a GPU: every call here fails (or has nothing to do) before the device is
touched; the pointers are fake."""
import ctypes

import pytest
import torch

from test_paged_cpu import INVALID, LIB, LL3, MISALIGNED, OK, UNSUPPORTED, PagedCache, cache

P = 0x1000  # a pointer


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    p, i, ll, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t
    c, out = ctypes.POINTER(PagedCache), ctypes.POINTER(ctypes.c_size_t)
    lib.attn_tree_workspace_bytes.argtypes = [c, i, i, out]
    lib.launch_attn_tree.argtypes = [c, p, p, p, i, i, ctypes.c_float, p, ll, p, p, sz, p]
    lib.launch_kv_compact.argtypes = [c, p, p, ll, i, p, p]
    lib.kv_resize_workspace_bytes.argtypes = [c, out]
    lib.launch_kv_resize.argtypes = [c, p, p, p, p, p, sz, p]
    lib.kv_fork_workspace_bytes.argtypes = [c, i, out]
    lib.launch_kv_fork.argtypes = [c, p, p, p, i, p, p, p, p, p, sz, p]
    return lib


def _tree(lib, q=P, qs=None, out=P, Hq=4, S=3, parents=None, stride=0, new=None, space=P, size=0, c=True, **kw):
    return lib.launch_attn_tree(ctypes.byref(cache(**kw)) if c else None, q, qs, out, Hq, S, -1.0, parents, stride, new,
                                space, size, None)


def _compact(lib, new=P, kept=P, stride=4, n=4, lens=P, c=True, **kw):
    return lib.launch_kv_compact(ctypes.byref(cache(**kw)) if c else None, new, kept, stride, n, lens, None)


def _resize(lib, table=P, held=P, refs=P, missing=P, space=P, size=1 << 20, c=True, **kw):
    return lib.launch_kv_resize(ctypes.byref(cache(**kw)) if c else None, table, held, refs, missing, space, size, None)


def _fork(lib, held=P, refs=P, parents=P, n=2, table=P, new_held=P, lens=P, missing=P, space=P, size=1 << 20, c=True,
          **kw):
    return lib.launch_kv_fork(ctypes.byref(cache(**kw)) if c else None, held, refs, parents, n, table, new_held, lens,
                              missing, space, size, None)


CALLS = {"tree": _tree, "compact": _compact, "resize": _resize, "fork": _fork}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("bad,status", [
    (dict(dtype=3), UNSUPPORTED), (dict(D=257), UNSUPPORTED), (dict(D=0), INVALID), (dict(heads=0), INVALID),
    (dict(page_size=0), INVALID), (dict(num_pages=-1), INVALID), (dict(B=-1), INVALID), (dict(table_width=-1), INVALID),
    (dict(table_stride=-4), INVALID), (dict(block_table=None), INVALID), (dict(seq_lens=None), INVALID),
    (dict(page_size=1 << 20, table_width=1 << 11), INVALID), (dict(seq_lens=0x1002), MISALIGNED),
    (dict(block_table=0x1001), MISALIGNED)], ids=str)
def test_cache_checks(lib, name, bad, status):
    assert CALLS[name](lib, **bad) == status
    assert CALLS[name](lib, c=False) == INVALID


@pytest.mark.parametrize("name", ["tree", "compact", "fork"])
@pytest.mark.parametrize("bad,status", [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k_strides=LL3(-1, 1, 1)), INVALID),
    (dict(v_strides=LL3(1, 1, -1)), INVALID), (dict(k=0x1001), MISALIGNED), (dict(v=0x1002, dtype=2), MISALIGNED)])
def test_cache_tensor_checks(lib, name, bad, status):
    assert CALLS[name](lib, **bad) == status


def test_tree_checks(lib):
    assert _tree(lib, Hq=3) == INVALID and _tree(lib, Hq=-2) == INVALID and _tree(lib, S=-1) == INVALID
    assert _tree(lib, S=1025) == INVALID and _tree(lib, B=1 << 16, Hq=1 << 16) == INVALID
    assert _tree(lib, q=None) == INVALID and _tree(lib, out=None) == INVALID and _tree(lib, space=None) == INVALID
    assert _tree(lib, qs=LL3(-1, 64, 64)) == INVALID and _tree(lib, qs=LL3(1, 64, -64)) == INVALID
    assert _tree(lib, parents=P, stride=-3) == INVALID
    assert _tree(lib, q=0x1001) == MISALIGNED and _tree(lib, out=0x1001) == MISALIGNED
    assert _tree(lib, parents=0x1002) == MISALIGNED and _tree(lib, new=0x1002) == MISALIGNED
    assert _tree(lib, space=0x1008) == MISALIGNED
    assert _tree(lib, Hq=0) == OK and _tree(lib, S=0) == OK and _tree(lib, B=0) == OK
    n = ctypes.c_size_t(7)
    assert lib.attn_tree_workspace_bytes(ctypes.byref(cache()), 4, 3, None) == INVALID
    assert lib.attn_tree_workspace_bytes(ctypes.byref(cache()), 3, 3, ctypes.byref(n)) == INVALID
    assert lib.attn_tree_workspace_bytes(ctypes.byref(cache()), 4, 1025, ctypes.byref(n)) == INVALID
    assert lib.attn_tree_workspace_bytes(ctypes.byref(cache()), 4, 0, ctypes.byref(n)) == OK and n.value == 0


def test_compact_checks(lib):
    assert _compact(lib, n=-1) == INVALID and _compact(lib, stride=-1) == INVALID
    for name in ("new", "kept", "lens"):
        assert _compact(lib, **{name: None}) == INVALID
        assert _compact(lib, **{name: 0x1002}) == MISALIGNED
    assert _compact(lib, B=0) == OK


def test_resize_checks(lib):
    for name in ("held", "refs", "missing"):
        assert _resize(lib, **{name: None}) == INVALID
        assert _resize(lib, **{name: 0x1002}) == MISALIGNED
    assert _resize(lib, table=0x2000) == INVALID  # not the cache's table
    assert _resize(lib, space=None) == INVALID and _resize(lib, space=0x1008) == MISALIGNED
    assert _resize(lib, size=16) == INVALID and _resize(lib, B=0) == OK
    n = ctypes.c_size_t()
    assert lib.kv_resize_workspace_bytes(ctypes.byref(cache(k=None, v=None, B=3)), ctypes.byref(n)) == OK
    assert n.value >= 4 * (3 + 3 + 4)
    assert lib.kv_resize_workspace_bytes(ctypes.byref(cache()), None) == INVALID


def test_fork_checks(lib):
    assert _fork(lib, n=-1) == INVALID
    for name in ("held", "refs", "parents", "table", "new_held", "lens", "missing"):
        assert _fork(lib, **{name: None}) == INVALID
        assert _fork(lib, **{name: 0x1002}) == MISALIGNED
    assert _fork(lib, space=None) == INVALID and _fork(lib, space=0x1008) == MISALIGNED and _fork(lib, size=8) == INVALID
    n = ctypes.c_size_t()
    assert lib.kv_fork_workspace_bytes(ctypes.byref(cache(B=3)), 5, ctypes.byref(n)) == OK
    assert n.value >= 4 * (3 + 3 + 5 + 4)
    assert lib.kv_fork_workspace_bytes(ctypes.byref(cache()), -1, ctypes.byref(n)) == INVALID
    assert lib.kv_fork_workspace_bytes(ctypes.byref(cache()), 2, None) == INVALID


def test_python_names_and_devices():
    import rocm_attn_b200 as ra
    import rocm_attn_op

    for name in ("attn_tree", "kv_compact", "kv_fork", "kv_resize"):
        assert getattr(rocm_attn_op, name) is getattr(ra, name) and name in ra.__all__ and name in rocm_attn_op.__all__
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    q = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: ra.attn_tree(q, k, k, t, n), lambda: ra.kv_compact(k, k, t, n, t, n),
                 lambda: ra.kv_fork(k, k, t, n, n, t[0], n), lambda: ra.kv_resize(t, n, n, t[0], 16)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-60):
        with pytest.raises(ValueError, match="scale"):
            ra.attn_tree(q, k, k, t, n, scale=scale)
