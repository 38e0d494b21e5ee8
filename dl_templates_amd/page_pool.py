"""Pages of a cache for running requests, handed out and taken back on the device, from the lengths that the requests are to have.

A pool is an int32 tensor [2 + pages]: the number of free pages, a word that is 0 between calls, and the free pages' numbers, of which the last of those that count
is handed out next.  ``page_assign_`` brings a pool, the requests' page tables and their lengths up to date; the tables and lengths are those that the paged calls
(``paged_cache``, ``paged_cache8``) take.  Nothing waits for the host, and a captured graph sees what the tensors hold when it is replayed.
"""
from __future__ import annotations

import torch

from . import _lib


class PageAssign(torch.autograd.Function):
    """``apply(page_table, seq_len, want, pool, page, n_tokens)`` -> (n_new, slots or None): what calls of ``page_assign_`` that are not plain eager ones run through."""

    @staticmethod
    def forward(ctx, page_table, seq_len, want, pool, page, n_tokens):
        return _lib.native.page_assign(page_table, seq_len, want, pool, page, n_tokens, True)


def page_pool(n_pages: int, device="cuda") -> torch.Tensor:
    """A pool of pages 0 .. n_pages - 1, all of them free; page 0 is handed out first."""
    if n_pages < 1:
        raise ValueError(f"a pool needs a page, got {n_pages}")
    return torch.cat([torch.tensor([n_pages, 0], dtype=torch.int32), torch.arange(n_pages - 1, -1, -1, dtype=torch.int32)]).to(device)


def page_assign_(page_table: torch.Tensor, seq_len: torch.Tensor, want: torch.Tensor, pool: torch.Tensor, page: int, n_tokens: int = None):
    """Requests of ``seq_len`` [B] tokens take or give back pages of ``page`` tokens until they can hold ``want`` [B]: ``(n_new, slots)``, in one launch.

    ``page_table`` [B, columns], ``seq_len`` and ``pool`` are brought up to date in place; all are int32, as is ``want``.  ``want[b]`` 0 ends a request, a smaller one than
    ``seq_len[b]`` shortens it (guessed tokens that were rejected), a negative one leaves it alone.  Pages that are given back can be handed out in the same call.  Requests
    are served in order: from the first whose pages the pool does not hold, those that need a page get nothing and keep their length, and so do requests that want more
    than their row of the table can hold or, with ``n_tokens``, more than that many tokens at once.  ``n_new`` [B] counts the tokens that each request gained; with
    ``n_tokens`` ``slots`` [B, n_tokens] names the place of each, page number times ``page`` plus the row in it, -1 behind the last (else ``slots`` is None).

    Columns behind a request's last page keep what they held.  A call that takes back what the last one gave leaves the pool as it was.  Up to 8192 requests; lengths
    outside the table's row and page numbers outside the cache are mistakes that are not looked for.  Calls on one pool must not overlap."""
    out = _lib.native.page_assign(page_table, seq_len, want, pool, page, n_tokens, False)
    if out is NotImplemented:
        with torch.no_grad():
            out = PageAssign.apply(page_table, seq_len, want, pool, page, n_tokens)
    return out
