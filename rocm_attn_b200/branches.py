"""Drafted tokens and shared pages on the paged key-value cache: the attention
that checks several guesses of the next tokens at once, and the pages that
sequences take, give back, share and copy.

The cache is the one of ``attn_decode`` (paged.py): ``k_cache``, ``v_cache``
``[num_pages, Hkv, page_size, D]``, ``block_table`` int32 ``[B, W]``,
``seq_lens`` int32 ``[B]``.  Two more tensors say who holds which pages:

* ``refs``: int32 ``[num_pages]``, the holders of each page, 0 where it is free;
* ``held``: int32 ``[B]``; sequence b holds the first ``held[b]`` pages of its
  row of the table.

All of them are device tensors that only the kernels read and write, so nothing
here synchronises and captured calls follow them.  Free pages are given out
from the lowest on, in the order of the sequences.  What is out of range
(pages, lengths, parents) is never followed; ``check_status`` then returns 8.

Lengths must not pass the pages that a sequence holds.  Entries of the table
behind ``held[b]`` are what is left of pages that it has given back, and other
sequences may hold those by now; no operator can tell.  So a program grows its
lengths by what it got, not by what it asked for.  A step that drafts tokens::

    kv_resize(table, held, lens + S, refs, page_size)             # room for the drafts
    drafted = (held * page_size - lens).clamp(0, S)               # fewer than S where pages ran out
    lens += drafted
    kv_append(k, v, k_cache, v_cache, table, lens, drafted)       # k/v [B, Hkv, S, D]
    o = attn_tree(q, k_cache, v_cache, table, lens, parents, drafted)  # q [B, Hq, S, D]
    lens = kv_compact(k_cache, v_cache, table, lens, accepted, drafted)
    kv_resize(table, held, lens, refs, page_size)                 # what the others held goes back

and one of a beam search::

    table, held, lens, missing = kv_fork(k_cache, v_cache, table, held, lens, refs, parents)
    kv_resize(table, held, lens + 1, refs, page_size)
    grown = (held * page_size - lens).clamp(0, 1)                 # 0 where pages ran out
    lens += grown
    kv_append(k, v, k_cache, v_cache, table, lens, grown)         # k/v [B, Hkv, 1, D]
    o = attn_decode(q, k_cache, v_cache, table, lens)

Nor may lengths be shortened into a page that other sequences hold (``kv_fork``
shares full pages) and then grow there: appends would write to it.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import rocm_attn_ext


def attn_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
              seq_lens: torch.Tensor, parents: Optional[torch.Tensor] = None,
              new_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of drafted tokens over a sequence's cached tokens:
    ``softmax(scale * q K^T) V``, each over the context and the drafted tokens
    that it follows.

    q: ``[B, Hq, S, D]`` in the cache's type, S at most 1024, Hq a multiple of
    Hkv (query heads ``h * Hq // Hkv`` and following read kv head ``h``).  The
    drafted tokens are the last n of the sequence, n being S or, with
    ``new_lens`` (int32 ``[B]``, at most S), its entry: token s lies at position
    ``seq_lens[b] - n + s``, where ``kv_append`` with the same lengths puts it.

    parents: int32 ``[B, S]`` (one tree for all: ``tree.expand(B, S)``), the
    drafted token that token s follows, below s, or -1 where it follows the
    context.  Token s attends to the context, itself, its parent, the parent's
    parent and so on; not given, token s follows s - 1.

    ``scale`` is positive and finite, 1/sqrt(D) if not given.  Returns O ``[B,
    Hq, S, D]``: zeros for tokens behind the n and for empty sequences; NaN, as
    the formula gives, for a token that has only scores of -inf.  Precision is
    that of ``attn_decode``; fp16 weights below 2^-21 of the largest may be off by
    2^-32 of that where ``Hq / Hkv * S`` is above eight.
    """
    if scale is None:
        scale = -1.0  # the binding's default
    else:
        # as 32 bits, what the kernels get; the binding takes other scales as not given
        scale = ctypes.c_float(scale).value
        if not 0.0 < scale < math.inf:
            raise ValueError("attn_tree: scale must be positive and finite in 32 bits")
    return rocm_attn_ext.attn_tree(q, k_cache, v_cache, block_table, seq_lens, parents, new_lens, scale)


def kv_compact(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               kept: torch.Tensor, new_lens: torch.Tensor, bounds: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Move the drafted tokens that were accepted to the front of the drafted
    ones, in place.

    new_lens: int32 ``[B]``, the drafted tokens of each sequence.  kept: int32
    ``[B, n]``, drafted tokens in ascending order (a path of the tree); the first
    -1 ends a list.  With ``base = seq_lens[b] - new_lens[b]``, K and V of position
    ``base + kept[b, i]`` go to position ``base + i``; rows behind the last kept
    token stay as they are.  Two sequences must not write to one page.

    bounds: optional page bounds (``kv_page_bounds``) that bound the drafted
    tokens where they were, as ``kv_append`` with them leaves them; a page that
    keys come to takes them in.  Where it is not given, a key that moves to
    another page may lie outside that page's bounds, and ``kv_page_bounds`` has
    to make them anew before ``kv_select_pages`` reads them.

    Returns the new lengths, int32 ``[B]``: base plus the tokens kept.
    """
    return rocm_attn_ext.kv_compact(k_cache, v_cache, block_table, seq_lens, kept, new_lens, bounds)


def kv_fork(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, held: torch.Tensor,
            seq_lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor,
            bounds: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The sequences of the next step as continuations of the present ones:
    beams, or several samples of one prompt.

    parents: int32 ``[n]``; new sequence i has the tokens of sequence
    ``parents[i]`` (-1: it is empty).  Full pages are shared.  A last page that is
    partly filled goes to the first sequence that continues the parent, if
    nobody else held it, and is copied to a free page for each other one.  All
    present sequences give up what they hold, so ``refs``, changed in place,
    counts the new ones; pages that this frees are given out from the next call on.

    bounds: optional page bounds (``kv_page_bounds``); those of a copied page go
    with it.  Where it is not given, a copy's bounds are whatever the page had
    before, and ``kv_page_bounds`` has to make them anew before ``kv_append``
    folds keys into them or ``kv_select_pages`` reads them.

    Returns ``(block_table, held, seq_lens, missing)`` of the new sequences, int32
    ``[n, W]`` (-1 behind a row's pages), ``[n]``, ``[n]`` and ``[1]``.  If there are fewer free
    pages than copies, ``missing`` says how many are lacking, nothing is changed
    and the new sequences are empty; the given tensors are still valid then and
    hold all their pages, so they had better be kept until ``missing`` has been
    read.  One pair of cache tensors is served: layers that share a table are kept
    as heads of one.
    """
    return rocm_attn_ext.kv_fork(k_cache, v_cache, block_table, held, seq_lens, refs, parents, bounds)


def kv_resize(block_table: torch.Tensor, held: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor,
              page_size: int) -> torch.Tensor:
    """Make every sequence hold the pages that its length needs: pages behind
    are given back, pages that it lacks are taken from the free ones.  A length
    of zero gives back all.  Changes ``block_table``, ``held`` and ``refs`` in place;
    entries of the table behind those held stay as they are, and lengths must not
    reach them: their pages may be other sequences'.

    Pages that the call frees are given out from the next call on.  A sequence
    for which too few are free, those for the sequences before it counted, takes
    none, and ``held[b] * page_size`` tokens are all it has room for.  Returns int32
    ``[B]``: the pages that such a sequence lacked, else 0.
    """
    return rocm_attn_ext.kv_resize(block_table, held, seq_lens, refs, int(page_size))
