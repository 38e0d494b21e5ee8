"""Attention over a 1D window whose first tokens stay visible, with heads of q in groups that share one head of k and v.

The window of ``tiled_swa`` along a sequence: with ``q`` [B, H, Lq, Dk], ``k`` [B, Hkv, Lk, Dk] and ``v`` [B, Hkv, Lk, Dv], query ``i``
stands at position ``p = Lk - Lq + i`` (the queries are the newest tokens) and sees key ``j`` iff ``j <= p`` and ``p - j < window`` or
``j < n_sink``.  A query that sees nothing (``p < 0``) gives zeros.  bfloat16 and float16, head dims up to 128; head dims that are
no multiples of 8 are zero-padded around the kernels, rows that cannot be read in 16-byte pieces are copied first.  Infinities and NaN
reach the rows and keys that see them and no others, at a price: those are summed by one wave each.  The serving form
of it, keys and values in pages, is ``paged_cache.paged_attention``.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .flash_attn import _cut_last, _pad_last


class WindowAttention(torch.autograd.Function):
    """``apply(q, k, v, window, n_sink, sm_scale)``, ``window`` None: no limit.  Plain eager calls run as one compiled node
    (csrc/torch_binding.cpp); under a trace, a ``torch.func`` transform or a dispatch mode, and with forward-mode tangents, the class itself
    runs.  Backward returns ``(dq, dk, dv, None, None, None)``; dk and dv are sums over the heads of a group."""

    @classmethod
    def apply(cls, *args):
        o = _lib.native.window(*args) if cls is WindowAttention else NotImplemented
        return super().apply(*args) if o is NotImplemented else o

    @staticmethod
    def forward(ctx, q, k, v, window, n_sink, sm_scale):
        ctx.dims = (q.shape[-1], v.shape[-1])
        plan = _lib.native.pad_plan(*ctx.dims, q, -1)
        if plan is not None:
            q, k, v = _pad_last(q, plan[0]), _pad_last(k, plan[0]), _pad_last(v, plan[1])
        ctx.scalars = (window, n_sink, sm_scale)
        o, lse2, low = _lib.native.window_forward(q, k, v, *ctx.scalars)
        ctx.save_for_backward(q, k, v, o, lse2, low)
        return _cut_last(o, ctx.dims[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse2, low = ctx.saved_tensors
        dq, dk, dv = _lib.native.window_backward(q, k, v, o, lse2, low, _pad_last(do, v.shape[-1]), *ctx.scalars)
        return _cut_last(dq, ctx.dims[0]), _cut_last(dk, ctx.dims[0]), _cut_last(dv, ctx.dims[1]), None, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = None, n_sink: int = 0, sm_scale: float = None) -> torch.Tensor:
    """o [B, H, Lq, Dv]; ``sm_scale`` None: ``1 / sqrt(Dk)``."""
    args = (q, k, v, window, n_sink, 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale)
    o = _lib.native.window(*args)
    return WindowAttention.apply(*args) if o is NotImplemented else o
