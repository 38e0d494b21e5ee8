"""Keys and values of running sequences in a cache of pages: appending to it, with the rotation on the way, and attention that reads it.

A cache is a tensor [pages, Hkv, page, D]; row b of ``page_table`` (int32 [B, columns]) names the pages of sequence b in order, so that position
p lies in row ``p % page`` of page ``page_table[b, p // page]``.  ``seq_len`` (int32 [B]) counts the tokens of every sequence, its newest
ones included; of T new tokens in a call sequence b has the first ``n_new[b]`` (None: all T), at positions ``seq_len[b] - n_new[b] ..
seq_len[b] - 1``; those behind are padding.  A ``seq_len`` beyond the table's row is a mistake: the append leaves out what does not fit, attention
takes what the row holds.  Both calls take the same ``seq_len`` and ``n_new``, which stay on the device: no call waits for
the host, and a captured graph sees what they hold when it is replayed.  Neither records a graph for autograd, and forward-mode tangents are
refused.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .rope_axes import _layout, _refuse_tangents


class PagedAppend(torch.autograd.Function):
    """``apply(k_cache, v_cache, k, v, page_table, seq_len, n_new, pos, layout number, rotate, q, *tables)`` -> rotated q or None: what calls of ``paged_append_`` that
    are not plain eager ones (trace, transform, dispatch mode) run through, without a graph.  It does not return what it writes: a trace could not run that."""

    @staticmethod
    def forward(ctx, k_cache, v_cache, k, v, page_table, seq_len, n_new, pos, layout, rotate, q, *tables):
        return _lib.native.paged_append(k_cache, v_cache, k, v, page_table, seq_len, n_new, pos, tables if rotate else None, layout, q, True)


class PagedAttention(torch.autograd.Function):
    """``apply(q, k_cache, v_cache, page_table, seq_len, n_new, window, n_sink, sm_scale)``: the same for ``paged_attention``."""

    @staticmethod
    def forward(ctx, q, k_cache, v_cache, page_table, seq_len, n_new, window, n_sink, sm_scale):
        return _lib.native.paged_attention(q, k_cache, v_cache, page_table, seq_len, window, n_sink, sm_scale, n_new, True)


def paged_append_(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, seq_len: torch.Tensor,
                  n_new: torch.Tensor = None, rope=None, q: torch.Tensor = None):
    """Writes k [B, Hkv, T, Dk] and v [B, Hkv, T, Dv] into their caches, in one launch with the rotation of k and q.

    ``rope``: None or ``(pos, tables, layout)`` as ``rope_axes_qk`` takes them; ``pos`` None: a token's place in its sequence on every axis.
    With ``q`` [B, H, T, Dk] rotated queries come back in a new tensor (padded rows as they were), else None.  Padding, positions outside the
    table and page numbers outside the cache write nothing.  No two tokens of a call may have the same place, and q, k and v must not lie in
    the caches.  bfloat16, float16 and float32, any strides and page size."""
    pos, tables, layout = rope if rope is not None else (None, None, "blocks")
    tables, code = None if rope is None else tuple(tables), _layout(layout)
    out = _lib.native.paged_append(k_cache, v_cache, k, v, page_table, seq_len, n_new, pos, tables, code, q, False)
    if out is NotImplemented:
        _refuse_tangents("paged_append_", k_cache, v_cache, k, v, q, *(tables or ()))
        with torch.no_grad():
            out = PagedAppend.apply(k_cache, v_cache, k, v, page_table, seq_len, n_new, pos, code, rope is not None, q, *(tables or ()))
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_len: torch.Tensor, window: int = None,
                    n_sink: int = 0, sm_scale: float = None, n_new: torch.Tensor = None) -> torch.Tensor:
    """``window_attention`` of the newest tokens q [B, H, T, Dk] over the cached keys and values: o [B, H, T, Dv].

    Padded rows, and rows of sequences without a key, give zeros, whatever the keys and values beside them hold.  bfloat16 and float16, head
    dims in multiples of 8 up to 128, pages of a multiple of 16 tokens, cache rows contiguous and 16-byte aligned.  What a page holds behind
    a sequence's last token does not matter; a page number outside the cache is a mistake that is not looked for (some page of the cache is
    read)."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale
    o = _lib.native.paged_attention(q, k_cache, v_cache, page_table, seq_len, window, n_sink, scale, n_new, False)
    if o is NotImplemented:
        _refuse_tangents("paged_attention", q, k_cache, v_cache)
        with torch.no_grad():
            o = PagedAttention.apply(q, k_cache, v_cache, page_table, seq_len, n_new, window, n_sink, scale)
    return o
