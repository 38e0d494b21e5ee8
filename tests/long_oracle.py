"""Plain 64-bit forms of the long-sequence operators, on the CPU or the GPU, and how far the kernels' outputs may be from them.

Bounds count roundings.  u = finfo(dtype).eps / 2 is half a step of a 16-bit type, relative to the value.  Products of 16-bit values are exact in
32 bits; a 32-bit sum of n terms is off by at most n 2^-24 times the sum of their magnitudes, and scores, exponentials and logarithms in
32 bits add to that: SLACK covers them for the lengths tested (n <= 2^12 terms, |score| <= 2^5: 2^-12 + 2^5 2^-24 2^1 < 2^-11).
"""
import math

import torch

SLACK = 2.0 ** -11


def seen(qpos, Lk, window, n_sink):
    """bool [Lq, Lk]"""
    p, j = qpos[:, None], torch.arange(Lk, device=qpos.device)[None]
    near = torch.ones_like(j > p) if window is None else p - j < window
    return (j <= p) & (near | (j < n_sink))


def probabilities(q, k, vis, scale):
    """softmax over what is seen [.., Lq, Lk]; rows that see nothing: zeros.  q, k in 64 bits."""
    if k.shape[-2] == 0:
        return (q @ k.transpose(-1, -2))
    s = torch.where(vis, q @ k.transpose(-1, -2) * scale, -math.inf)
    e = torch.where(vis, torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300)), 0.0)
    return e / e.sum(-1, keepdim=True).clamp_min(1e-300)


def window(q, k, v, window_, n_sink, scale, do=None, off=None):
    """{name: (value, bound)} of o, and with `do` of dq, dk, dv; tensors [B, heads, L, D] of a 16-bit type."""
    u = torch.finfo(q.dtype).eps / 2
    G = q.shape[1] // k.shape[1]
    Lq, Lk = q.shape[2], k.shape[2]
    qpos = torch.arange(Lq, device=q.device) + (Lk - Lq if off is None else off)
    vis = seen(qpos, Lk, window_, n_sink)
    f = lambda x: x.double()  # noqa: E731
    wide = lambda x: f(x).repeat_interleave(G, 1)  # noqa: E731
    qd, kd, vd = f(q), wide(k), wide(v)
    p = probabilities(qd, kd, vis, scale)
    o, mag = p @ vd, p @ vd.abs()
    # P and the sum it is divided by are formed from rounded exponentials (u each), the output is rounded once
    o_tol = u * (mag + 2 * o.abs()) + SLACK * mag
    out = {"o": (o, o_tol)}
    if do is None:
        return out
    dod = f(do)
    group = lambda x: x.reshape(x.shape[0], k.shape[1], G, *x.shape[2:]).sum(2)  # noqa: E731
    # P from the stored sum (u) and rounded for the product (u)
    dv, dv_mag = p.transpose(-1, -2) @ dod, p.transpose(-1, -2) @ dod.abs()
    dv, dv_mag = group(dv), group(dv_mag)
    out["dv"] = (dv, (2 * u + SLACK) * dv_mag + u * dv.abs())
    dp, dp_mag = dod @ vd.transpose(-1, -2), dod.abs() @ vd.abs().transpose(-1, -2)
    delta = (dod * o).sum(-1, keepdim=True)
    # delta is formed from the rounded output
    delta_tol = (dod.abs() * (o_tol + u * o.abs())).sum(-1, keepdim=True) + SLACK * (dod * o).abs().sum(-1, keepdim=True)
    ds = p * (dp - delta)
    ds_tol = 2 * u * ds.abs() + p * (delta_tol + SLACK * dp_mag)
    dq, dk = scale * (ds @ kd), scale * (ds.transpose(-1, -2) @ qd)
    out["dq"] = (dq, scale * (ds_tol @ kd.abs() + SLACK * (ds.abs() @ kd.abs())) + u * dq.abs())
    dk, dk_tol = group(dk), scale * group(ds_tol.transpose(-1, -2) @ qd.abs() + SLACK * (ds.abs().transpose(-1, -2) @ qd.abs()))
    out["dk"] = (dk, dk_tol + u * dk.abs())
    return out


def tiny(dtype):
    """Half a step of the type's subnormal numbers: what a rounding may be off by next to zero."""
    return float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps / 2


def check(got, want, what):
    """`got` against (value, bound)."""
    value, bound = (x.to(got.device) for x in want)
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(value.shape)}"
    off = (got.double() - value).abs()
    bad = ~(off <= bound + tiny(got.dtype))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values outside, e.g. {got[bad][:4].tolist()} for {value[bad][:4].tolist()}"


def pairs_of(sections, layout):
    """[(first dim, second dim, axis, pair of the axis)]"""
    out, off, total = [], 0, sum(sections)
    for a, r in enumerate(sections):
        for i in range(r):
            first = (2 * off if layout == "blocks" else off) + i
            out.append((first, first + (r if layout == "blocks" else total), a, i))
        off += r
    return out


def rotate(x, pos, tables, layout, inverse=False):
    """x [B, H, N, C], pos [axes, N] or [axes, B, N]: (value, bound) in 64 bits."""
    y, tol = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    pos = pos if pos.dim() == 3 else pos[:, None].expand(-1, x.shape[0], -1)
    u = torch.finfo(x.dtype).eps / 2
    for d0, d1, a, i in pairs_of([t.shape[1] for t in tables], layout):
        p = pos[a].long()
        cs = tables[a].double()[p.clamp(0, tables[a].shape[0] - 1), i]   # [B, N, 2]
        c = torch.where(p >= 0, cs[..., 0], torch.ones_like(cs[..., 0]))[:, None]
        s = torch.where(p >= 0, cs[..., 1], torch.zeros_like(cs[..., 0]))[:, None] * (-1 if inverse else 1)
        x0, x1 = x[..., d0].double(), x[..., d1].double()
        y[..., d0], y[..., d1] = x0 * c - x1 * s, x0 * s + x1 * c
        for d, m in ((d0, (x0 * c).abs() + (x1 * s).abs()), (d1, (x0 * s).abs() + (x1 * c).abs())):
            # two products and a sum in 32 bits, one rounding to the type; nothing where nothing is rotated
            tol[..., d] = torch.where((p >= 0)[:, None], 2 * 2.0 ** -24 * m + (2.0 ** -24 + u) * y[..., d].abs(), torch.zeros_like(m))
    return y, tol


def table(length, pairs, base=10000.0):
    inv = base ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    ang = torch.arange(length, dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float()
