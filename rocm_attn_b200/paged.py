"""Paged key-value cache: the attention of one new token per sequence, the
cache's writer, and the two ways of reading less of it.

The reference has no cache (its op takes whole q/k/v tensors,
python/rocm_attn_op/__init__.py:29-32); these operators are what a program
that generates token by token needs beside ``attn_forward``.

Cache layout, common to all of them:

* ``k_cache``, ``v_cache``: ``[num_pages, Hkv, page_size, D]``, fp16, bf16 or
  fp32, any strides with a contiguous head dim (a ``[num_pages, page_size, Hkv,
  D]`` cache is passed as ``cache.transpose(1, 2)``), 1 <= D <= 256, any page
  size;
* ``block_table``: int32 ``[B, W]``; token t of sequence b lies in page
  ``block_table[b, t // page_size]``, row ``t % page_size``.  Entries behind a
  sequence's last page do not matter;
* ``seq_lens``: int32 ``[B]``, the tokens of each sequence in the cache, the
  newest included.  Zero or less is an empty sequence, such as an unused row of
  a padded batch.

Table and lengths are device tensors that only the kernels read, so nothing
here synchronises and captured calls follow pages and lengths that change.
Entries outside the cache are never followed and tokens beyond ``W *
page_size`` are left out; ``check_status`` then returns 8.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import rocm_attn_ext


def attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, scale: Optional[float] = None, pages: Optional[torch.Tensor] = None,
                weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence over its cached tokens:
    ``softmax(scale * q K^T) V``.

    q: ``[B, Hq, 1, D]`` in the cache's type, Hq a multiple of Hkv (query heads
    ``h * Hq // Hkv`` and following read kv head ``h``).  ``scale`` is positive
    and finite, 1/sqrt(D) if not given.  Returns O ``[B, Hq, 1, D]``; an empty
    sequence gives zeros, one that has tokens and only scores of -inf NaN, as
    the formula does.

    Scores and softmax are held in 32 bits.  With fp16 and bf16 each softmax
    weight is rounded to that type for the product with V, by half a step (2^-11
    and 2^-8 of it) at most, as attention on tensor cores does; the error
    against exact arithmetic is about 1.2 times that of rounding O alone.

    pages: optional int32 ``[B, Hkv, n]`` of logical pages (``t // page_size``),
    as ``kv_select_pages`` returns: only their tokens are attended to.  Entries
    that name no page of the sequence (-1) add nothing; one named twice counts
    twice.

    weights: optional fp32 ``[B, Hkv, >= W * page_size]``, updated in place:
    each token's softmax weight, summed over the query heads of the kv head, is
    added to it (``kv_evict`` takes it).  Needs ``4 * B * Hq * W * page_size``
    bytes of scratch memory, so the table had better be as wide as the lengths
    need.  Not together with ``pages``: steps that read listed pages leave the
    weights as they are, so a loop that evicts by them takes whole steps too.
    """
    if scale is None:
        scale = -1.0  # the binding's default
    else:
        # as 32 bits, what the kernels get; the binding takes other scales as not given
        scale = ctypes.c_float(scale).value
        if not 0.0 < scale < math.inf:
            raise ValueError("attn_decode: scale must be positive and finite in 32 bits")
    return rocm_attn_ext.attn_decode(q, k_cache, v_cache, block_table, seq_lens, scale, pages, weights)


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: Optional[torch.Tensor] = None,
              bounds: Optional[torch.Tensor] = None) -> None:
    """Write new tokens to the cache.

    k, v: ``[B, Hkv, S, D]``.  ``seq_lens`` counts the new tokens already, so
    that one lengths tensor serves this call and the ``attn_decode`` after it:
    token s of the n new ones of sequence b goes to position ``seq_lens[b] - n +
    s``, where n is S or, with ``new_lens`` (int32 ``[B]``, at most S), its
    entry.  Positions below zero are left out (empty sequences take nothing),
    and all other rows of the cache stay as they are.  Two sequences must not
    write to one page.

    bounds: optional page bounds (``kv_page_bounds``); the new keys are folded
    in, and a page whose row 0 is new begins anew.
    """
    rocm_attn_ext.kv_append(k, v, k_cache, v_cache, block_table, seq_lens, new_lens, bounds)


def kv_page_bounds(k_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                   bounds: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Elementwise minimum and maximum of the keys of each page:
    ``bounds[page, h, 0 or 1]`` for the pages of the given sequences, over the
    sequence's tokens in the page.  ``[num_pages, Hkv, 2, D]`` in the cache's
    type; written to ``bounds`` if given (pages of no sequence keep their
    values), else to a new tensor (where they are zero).  A page that sequences
    share should hold the same tokens of each, otherwise it gets the bounds of
    one of them.  Returns it.
    """
    return rocm_attn_ext.kv_page_bounds(k_cache, block_table, seq_lens, bounds)


def kv_select_pages(q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    page_size: int, top: int) -> torch.Tensor:
    """The pages of each (sequence, kv head) that a new token should read:
    int32 ``[B, Hkv, top]``, ascending logical pages, -1 behind them where the
    sequence has fewer than ``top``.

    The newest page is always in.  The others are those of largest score, the
    sum over d of ``max * p + min * m``, p and m being q's positive and negative
    parts summed over the kv head's query heads.  That is the sum of ``max(q *
    min, q * max)``, an upper bound of the summed scores of any token of the
    page.  A part that is zero adds nothing, even beside an infinite bound; a NaN
    bound makes the score NaN.  Ties go to the lower page and NaN counts as
    largest.  Scores are summed in 64 bits.
    """
    return rocm_attn_ext.kv_select_pages(q, bounds, block_table, seq_lens, int(page_size), int(top))


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
             weights: torch.Tensor, new_block_table: torch.Tensor, budget: int,
             recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Evict tokens by accumulated attention weight.

    Of each (sequence, kv head) the last ``recent`` tokens are kept and, of the
    others, those of largest ``weights`` (as ``attn_decode`` accumulates them),
    ``budget`` tokens in all; ties go to the lower position and NaN counts as
    largest.  The kept tokens are copied, in their order, to the pages that
    ``new_block_table`` (int32 ``[B, W']``, ``W' * page_size >= budget``) names
    in the same caches; the old pages stay as they are.  The new pages must be
    distinct and none an old page of the given sequences.  Page bounds of the
    new pages come from ``kv_page_bounds``.

    Returns ``(new_lens, new_weights, kept)``: int32 ``[B]``, min(length,
    budget); fp32 ``[B, Hkv, W' * page_size]``, the kept tokens' weights with
    zeros behind; int32 ``[B, Hkv, budget]``, their old positions with -1 behind.
    """
    return rocm_attn_ext.kv_evict(k_cache, v_cache, block_table, seq_lens, weights, new_block_table, int(budget),
                                  int(recent))
