"""A paged K/V cache: rows into it, rows out of it, and attention of new tokens over it.

A decoder keeps the keys and values of its sequences in pages, which ``fst_attention_paged`` reads as the prefix
of token trees if they are held in 16 bits (a prefix in 8 bits goes there by way of ``fst_cache_read`` and ``fst_attention``).  Here are the calls around it: ``fst_cache_append`` writes the rows of new tokens (a prompt's, a
decoded token's, or the accepted path of a tree) into the pages, ``fst_attention_chunk`` is the attention of those
tokens, and ``fst_cache_read`` brings sequences back as contiguous tensors.

The cache is plain tensors.  ``k_pool`` and ``v_pool`` are ``[n_pages, page_size, H_kv, D]``
(``pool_layout="NHD"``) or ``[n_pages, H_kv, page_size, D]`` (``"HND"``), page_size 16, 32, 64 or 128, D 64 or 128;
``block_table`` is int32 ``[Z, pages]``: row ``r`` of sequence ``z`` lives in page ``block_table[z, r // page_size]``.
The pools are float16 or bfloat16, or float8_e4m3fn for half the memory; then ``k_scale`` and ``v_scale``, contiguous
float8_e8m0fnu ``[n_pages, H_kv, page_size]``, hold a power of two for every row and head, and the row stands for
``pool.float() * scale.float()``.

All calls are asynchronous on torch's current stream and can be captured into a graph; lengths and tables are read
on the GPU.  What only the GPU can see (a page number outside the pool, a length past the table) is
recorded for ``last_status`` and never faults.  (Length and pages are not looked at where a sequence has no queries.)  What an
8-bit cache holds is what ``fst_cache_append`` wrote or zeros: e4m3's NaN bytes do not occur.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def _nhd(pool_layout) -> bool:
    if pool_layout not in ("NHD", "HND"):
        raise ValueError("pool_layout must be 'NHD' or 'HND'")
    return pool_layout == "NHD"


def fst_cache_append(k, v, k_pool, v_pool, block_table, start, *, lens: Optional[torch.Tensor] = None,
                     rows: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                     v_scale: Optional[torch.Tensor] = None, pool_layout: str = "NHD") -> None:
    """Write new K/V rows into a paged cache, quantising them if it holds float8_e4m3fn.

    ``k``, ``v`` are ``[Z, H_kv, N, D]`` (any strides, D contiguous), float16 or bfloat16, the cache's dtype if that
    has 16 bits.  New row ``j < lens[z]`` (default: all) of sequence ``z`` goes to position ``start[z] + j``.  ``rows``
    (int32 ``[Z, M]``) picks the rows of ``k`` and ``v`` and their order, e.g. the nodes of a token tree that
    were accepted.  ``start`` and ``lens`` are int32 ``[Z]``.

    Quantisation of a row of one head: with ``a`` its largest magnitude, the scale is the smallest ``2**e`` with
    ``a <= 448 * 2**e`` (e from -117 to 119); values are rounded to the nearest e4m3 of ``x / 2**e``, ties to even,
    at most 448.  A row with an element that is not finite reads as NaN.

    A row whose position lies outside its table, whose page is not one of the pool's or whose entry of ``rows`` is not
    one of ``k``'s is not written, and of a count ``lens[z]`` above the call's rows only those are (``last_status`` in
    either case); a count below zero is none.  No two rows of a call may go to the same place: pages that
    sequences share are to be copied before one of them writes there."""
    host = _lib._host or _lib.host()
    host.cache_append(k, v, k_pool, v_pool, _nhd(pool_layout), block_table, start, lens, rows, k_scale, v_scale)


def fst_cache_read(k_pool, v_pool, block_table, lens, max_rows: int, *, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None,
                   pool_layout: str = "NHD", out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """The first ``min(lens[z], max_rows)`` rows of every sequence as contiguous ``(k, v)``, each
    ``[Z, H_kv, max_rows, D]``; the rows behind them are zeros.

    A float8_e4m3fn cache is expanded to ``dtype``, bfloat16 (default, exact) or float16 (rounded, at most 65504 in
    magnitude); one of 16 bits is read as what it is.  ``out``: the two tensors to write instead."""
    if dtype not in (None, torch.float16, torch.bfloat16):
        raise TypeError("a cache is read as float16 or bfloat16")
    k_out, v_out = (None, None) if out is None else out
    host = _lib._host or _lib.host()
    return host.cache_read(k_pool, v_pool, _nhd(pool_layout), block_table, lens, int(max_rows), k_scale, v_scale,
                           None if dtype is None else dtype == torch.bfloat16, k_out, v_out)


def fst_attention_chunk(q, k_pool, v_pool, block_table, kv_lens, sm_scale, *, q_lens: Optional[torch.Tensor] = None,
                        causal: bool = True, k_scale: Optional[torch.Tensor] = None,
                        v_scale: Optional[torch.Tensor] = None, pool_layout: str = "NHD",
                        out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of new tokens over a paged cache that holds their own rows too (``fst_cache_append`` first).

    ``q`` is ``[Z, H, N, D]``, float16 or bfloat16 (the cache's dtype if that has 16 bits), ``H`` a multiple of the
    cache's heads.  Sequence ``z`` has ``kv_lens[z]`` rows in the cache and ``q_lens[z]`` queries (default ``N``), which are
    its last positions: query ``i`` attends to the rows up to ``kv_lens[z] - q_lens[z] + i``, or with
    ``causal=False`` to all of them.  One call covers single tokens, drafted runs and chunks of prompts, also
    mixed; which kernel runs goes by ``N``, so that a prompt and many single tokens are faster as two calls (512 tokens beside 63
    over 4500 rows each: 240 instead of 280 us, over an 8-bit cache 176 instead of 650).  Both lengths are int32 ``[Z]``.

    A query that sees no row gets zeros.  Rows ``i >= q_lens[z]`` of ``out`` are left as they are (zeros where the call
    allocates it).  ``out`` may be ``q``.  What the cache holds at rows that a query does not attend to, NaN included, does not reach it.
    An 8-bit cache under float16 queries is meant to hold values that float16 can hold (``fst_cache_read``).
    Sums are float32: V's values times the number of rows times 256 have to stay below 3e38.  Every call allocates a workspace of up to 39 MB where
    tables hold more than 128 rows; with ``N * H / H_kv`` of 2048 or more an 8-bit cache is copied to 16 bits for the
    call, in room for all that the tables can hold, as long as that is at most 2 GB.
    With ``return_lse`` the result is ``(out, lse)``, ``lse`` the base-2 log-sum-exp of the scaled scores,
    ``[Z * H, N]``, -inf where nothing is seen.  ``sm_scale`` must be positive."""
    host = _lib._host or _lib.host()
    return host.attention_chunk(q, out, k_pool, v_pool, _nhd(pool_layout), block_table, kv_lens, q_lens, k_scale, v_scale,
                                sm_scale, bool(causal), bool(return_lse))
