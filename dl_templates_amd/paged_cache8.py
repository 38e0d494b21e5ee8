"""Keys and values of running sequences in a cache of pages held in 8 bits: appending to it, with the rotation on the way, and attention that reads it.

A cache is as ``paged_cache`` has it, [pages, Hkv, page, D] with the same ``page_table``, ``seq_len`` and ``n_new``, of 8-bit numbers c: ``torch.float8_e4m3fn`` or
``torch.int8``.  Beside it are scales, ``torch.float8_e8m0fnu`` [pages, Hkv, page / block]: the cache holds c times the scale of its block, ``block`` tokens of a head.  A block
is a multiple of 16 tokens, up to 128, that divides the page.  The type makes scales powers of two, which has two uses: every number times its scale is a number of
bfloat16 (from 2^-124, an append's least being 2^-100), and a scale that grows with the tokens of its block costs the older ones no bit but those that leave the format's range.

Both caches may be uninitialised memory: what is behind a sequence's last token does not matter, and a block's scale is set with its first token.  Half the bytes of a
16-bit cache; e4m3 keeps 4 bits of every number (an error of up to 2^-4 of it), int8 7 to 8 bits of the largest number of a block.  No call records a graph, waits
for the host, or takes forward-mode tangents.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .rope_axes import _layout, _refuse_tangents


class Paged8Append(torch.autograd.Function):
    """``apply(k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_len, n_new, pos, layout number, rotate, q, *tables)`` -> rotated q or None: what calls of
    ``paged8_append_`` that are not plain eager ones run through, without a graph."""

    @staticmethod
    def forward(ctx, k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_len, n_new, pos, layout, rotate, q, *tables):
        return _lib.native.paged8_append(k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_len, n_new, pos, tables if rotate else None, layout, q, True)


class Paged8Attention(torch.autograd.Function):
    """``apply(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_len, n_new, window, n_sink, sm_scale)``: the same for ``paged8_attention``."""

    @staticmethod
    def forward(ctx, q, k_cache, v_cache, k_scale, v_scale, page_table, seq_len, n_new, window, n_sink, sm_scale):
        return _lib.native.paged8_attention(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_len, window, n_sink, sm_scale, n_new, True)


def paged8_append_(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                   seq_len: torch.Tensor, n_new: torch.Tensor = None, rope=None, q: torch.Tensor = None):
    """``paged_append_`` into an 8-bit cache: k [B, Hkv, T, Dk] and v [B, Hkv, T, Dv] rounded to it, in one launch with the rotation of k and q.

    A block whose first token is new takes the least scale at which its new tokens fit (the largest e4m3 number is 448, the largest of int8 127); where new tokens join older
    ones the scale grows if it has to, and then the older ones' numbers are rounded anew.  Rounding is to nearest, even ones at ties, from the rotation's 32 bits.
    Elements that are infinite or NaN become NaN, in int8 with all of their block until a sequence starts the block again.  Numbers of float16 come back finite.

    ``rope`` and ``q`` as in ``paged_append_``: rotated queries come back in a new tensor.  Padding, positions outside the table and page numbers outside the cache write
    nothing.  No two tokens of a call may have the same place, no block may get tokens of two sequences in one call, and k, v and q must not lie in the caches.  bfloat16, float16 and float32; head dims in multiples of 8
    up to 128; cache rows contiguous and 8-byte aligned."""
    pos, tables, layout = rope if rope is not None else (None, None, "blocks")
    tables, code = None if rope is None else tuple(tables), _layout(layout)
    out = _lib.native.paged8_append(k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_len, n_new, pos, tables, code, q, False)
    if out is NotImplemented:
        _refuse_tangents("paged8_append_", k, v, q, *(tables or ()))
        with torch.no_grad():
            out = Paged8Append.apply(k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_len, n_new, pos, code, rope is not None, q, *(tables or ()))
    return out


def paged8_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor,
                     seq_len: torch.Tensor, window: int = None, n_sink: int = 0, sm_scale: float = None, n_new: torch.Tensor = None) -> torch.Tensor:
    """``paged_attention`` over an 8-bit cache: o [B, H, T, Dv] of q [B, H, T, Dk], bfloat16 or float16, keys and values read as numbers of q's type (of int8
    caches, with up to 32 rows a kv head, as they are).  For float16 queries the cache must hold no number beyond 65504; an append of float16 tokens sees to that.

    Padded rows, and rows of sequences without a key, give zeros, whatever the keys and values beside them hold.  Head dims in multiples of 8 up to 128, cache rows contiguous
    and 8-byte aligned.  What a page holds behind a sequence's last token, its scales included, does not matter; a page number outside the cache is a mistake that is not
    looked for (some page of the cache is read)."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale
    o = _lib.native.paged8_attention(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_len, window, n_sink, scale, n_new, False)
    if o is NotImplemented:
        _refuse_tangents("paged8_attention", q)
        with torch.no_grad():
            o = Paged8Attention.apply(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_len, n_new, window, n_sink, scale)
    return o
