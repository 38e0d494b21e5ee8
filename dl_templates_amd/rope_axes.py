"""Rotary positions with several axes: time, height and width of a clip, say.

The 2D rotation of ``fused_rope2d`` for one to four axes, each with a cos / sin table of its own (fp32 [len, R, 2], as
``FusedRotaryPositionEncodingContext`` makes them) and an int32 position per token, ``pos`` [axes, N], or [axes, B, N] where sequences
differ.  A negative position leaves the axis' dims as they are, others are clamped to the table.  Axis a turns R_a pairs of dims;
with ``off_a = R_0 + .. + R_(a-1)`` and ``P`` the sum of all R, pair i of axis a is

* ``layout="blocks"``: dims ``2 off_a + i`` and ``2 off_a + R_a + i``, the layout of the 2D rotation;
* ``layout="halves"``: dims ``off_a + i`` and ``P + off_a + i``.

Dims from ``2 P`` on pass through.  bfloat16, float16 and float32, any strides; one launch for q and k together.
"""
from __future__ import annotations

import torch

from . import _lib
from .rope2d import FusedRotaryPositionEncodingContext

LAYOUTS = {"blocks": 0, "halves": 1}


def _layout(name: str) -> int:
    try:
        return LAYOUTS[name]
    except (KeyError, TypeError):
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got {name!r}") from None


class RopeAxes(torch.autograd.Function):
    """``apply(q, k, pos, layout number, inverse, *tables)`` -> (rotated q, rotated k); k may be None.  Plain eager calls of
    ``rope_axes_qk`` run as one compiled node (csrc/torch_binding.cpp), any other (trace, transform, dispatch mode, forward-mode tangent)
    through this class."""

    @staticmethod
    def forward(ctx, q, k, pos, layout, inverse, *tables):
        ctx.layout, ctx.inverse, ctx.n = layout, inverse, len(tables)
        ctx.save_for_backward(pos, *tables)
        ctx.set_materialize_grads(False)
        return _lib.native.rope_axes(q, k, pos, tables, layout, inverse, 1)

    @staticmethod
    def backward(ctx, dq, dk=None):
        pos, *tables = ctx.saved_tensors
        rest = (None,) * (3 + ctx.n)
        if dq is None and dk is None:
            return (None, None) + rest
        if dq is None:
            return (None, RopeAxes.apply(dk, None, pos, ctx.layout, not ctx.inverse, *tables)[0]) + rest
        return tuple(RopeAxes.apply(dq, dk, pos, ctx.layout, not ctx.inverse, *tables)) + rest


def rope_axes_qk(q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor, tables, layout: str = "blocks", inverse: bool = False):
    """Rotated copies of q [B, Hq, N, C] and k [B, Hk, N, C] (None: q alone), one launch in each direction."""
    code, tables = _layout(layout), tuple(tables)
    out = _lib.native.rope_axes(q, k, pos, tables, code, inverse, 0)
    return RopeAxes.apply(q, k, pos, code, inverse, *tables) if out is NotImplemented else out


class RopeAxesInPlace(torch.autograd.Function):
    """``apply(q, k, pos, layout number, inverse, *tables)`` -> None, q and k rotated in place: what calls of ``rope_axes_qk_`` that are not plain eager ones (trace,
    transform, dispatch mode) run through, without a graph.  It does not return what it writes: a trace could not run that."""

    @staticmethod
    def forward(ctx, q, k, pos, layout, inverse, *tables):
        _lib.native.rope_axes(q, k, pos, tables, layout, inverse, 3)


def _refuse_tangents(name: str, *tensors) -> None:
    """A call that writes in place, or records no graph, would leave a forward-mode tangent behind."""
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no derivative in forward mode")


def rope_axes_qk_(q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor, tables, layout: str = "blocks", inverse: bool = False):
    """The same in place and without a graph; tensors that need a gradient, and forward-mode tangents, are refused."""
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        raise RuntimeError("rope_axes_qk_ records no graph: use rope_axes_qk for tensors that need a gradient")
    code, tables = _layout(layout), tuple(tables)
    out = _lib.native.rope_axes(q, k, pos, tables, code, inverse, 2)
    if out is NotImplemented:
        _refuse_tangents("rope_axes_qk_", q, k, pos, *tables)
        with torch.no_grad():
            RopeAxesInPlace.apply(q, k, pos, code, inverse, *tables)
        out = q, k
    return out


class RotaryPositionEncodingAxes(torch.nn.Module):
    """Tables of every axis and the rotation of q and k by them.  ``n_components[a]``: dims that axis a turns (even), ``max_lens[a]``:
    positions on it."""

    @staticmethod
    def encode_pos(*lens: int) -> torch.Tensor:
        """int32 [axes, N]: positions of the cells of a grid of the given lengths, the last axis fastest."""
        grids = torch.meshgrid(*(torch.arange(n) for n in lens), indexing="ij")
        return torch.stack([g.flatten() for g in grids]).to(torch.int32)

    def __init__(self, n_components, max_lens, layout: str = "blocks", base: float = 10000.0):
        super().__init__()
        if len(n_components) != len(max_lens):
            raise ValueError("n_components and max_lens must have an entry for every axis")
        _layout(layout)
        self.layout = layout
        self.axes = torch.nn.ModuleList(FusedRotaryPositionEncodingContext(n, m, base) for n, m in zip(n_components, max_lens))

    @property
    def tables(self):
        return [a.cs_components for a in self.axes]

    def forward(self, q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor):
        return rope_axes_qk(q, k, pos, self.tables, self.layout)
