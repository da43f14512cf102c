"""Drop-in package name of JoursBleu/rocm_attn's operator.

``from rocm_attn_op import attn_forward`` and
``from rocm_attn_op import rocm_attn_ext`` keep working for callers of the
reference (python/rocm_attn_op/__init__.py:29, setup.py:62,68); both resolve
to the sm_100a implementation in ``rocm_attn_b200``.
"""
import sys as _sys

from rocm_attn_b200 import (attn_decode, attn_forward, attn_forward_batch, attn_tree, check_status, kv_append,
                            kv_compact, kv_evict, kv_fork, kv_page_bounds, kv_resize, kv_select_pages, rocm_attn_ext)

_sys.modules[__name__ + ".rocm_attn_ext"] = rocm_attn_ext

__all__ = ["attn_forward", "attn_forward_batch", "attn_decode", "kv_append", "kv_evict", "kv_page_bounds",
           "kv_select_pages", "attn_tree", "kv_compact", "kv_fork", "kv_resize", "check_status", "rocm_attn_ext"]
