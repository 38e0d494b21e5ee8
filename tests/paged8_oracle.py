"""Plain forms of the operators of an 8-bit cache, on the host: pages handed out by a loop over requests, blocks formed one by one in 64 bits, and how far numbers may be off.

A rounding is off by at most half a step: 2^-4 of the value in e4m3, or half of its smallest number, 2^-10, times the scale; half of the scale in int8.  Values before it
are rotated in 32 bits: two products and a sum of values of magnitude m are off by at most 3 2^-24 m, which can move a value across a border, but no further than that."""
import numpy as np
import torch

FP8, I8 = torch.float8_e4m3fn, torch.int8
MOST = {FP8: 448.0, I8: 127.0}
LEAST = -100


def exponent(big, fmt):
    """Least e with big <= MOST 2^e, LEAST at least."""
    e = LEAST
    if big > 0:
        e = max(LEAST, int(np.floor(np.log2(big / MOST[fmt]))) - 1)
        while big > MOST[fmt] * 2.0 ** e:
            e += 1
    return e


def most(e, fmt, dtype):
    """The largest number of the format whose value at 2^e is finite in fp16 (other types: the largest)."""
    if dtype != torch.float16:
        return MOST[fmt]
    return min(448.0, 61440 * 2.0 ** -e) if fmt == FP8 else min(127.0, np.floor(65504 * 2.0 ** -e))


def rounded(x, fmt):
    """Nearest number of the format, in 64 bits, ties to even; no number: NaN."""
    if fmt == I8:
        return torch.where(torch.isfinite(x), torch.round(x), 0.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, 1e300))) - 3)
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, float("nan"))


def scales(bits):
    """float8_e8m0fnu or its bytes -> 64 bits."""
    b = bits.view(torch.uint8).double() if bits.dtype != torch.float64 else bits
    return torch.where(b == 255, float("nan"), torch.exp2(b - 127))


def values(cache, scale):
    """What a cache holds: 64 bits."""
    n, h, page, d = cache.shape
    s = scales(scale).repeat_interleave(page // scale.shape[2], 2)[..., None]
    return cache.to(torch.float32).double() * s


def append(cache, scale, x, m, table, seq, new, dtype):
    """x [B, H, T, d] in 64 bits (m: magnitudes of what it was formed from) into copies of cache and scale: (numbers in 64 bits, bytes of the scales, bound of the numbers,
    blocks whose largest element lies at a border of two scales)."""
    fmt, page, block = cache.dtype, cache.shape[2], cache.shape[2] // scale.shape[2]
    c, e = cache.to(torch.float32).double(), scale.view(torch.uint8).int().clone()
    tol, near = torch.zeros_like(c), torch.zeros_like(e, dtype=torch.bool)
    room = table.shape[1] * page
    for b in range(len(seq)):
        held = seq[b] - new[b]
        lo, hi = max(held, 0), min(seq[b], room)
        for base in range(lo // block * block, hi, block):
            n0, n1 = max(lo, base), min(hi, base + block)
            p = int(table[b, base // page])
            if not 0 <= p < cache.shape[0] or n0 >= n1:
                continue
            row = base % page
            for h in range(x.shape[1]):
                y, mag = x[b, h, n0 - held:n1 - held], m[b, h, n0 - held:n1 - held]
                fin = y[torch.isfinite(y)].abs()
                big = float(fin.max()) if fin.numel() else 0.0
                need, old = exponent(big, fmt) + 127, int(e[p, h, row // block])
                if mag.abs().max() > 0 and not torch.equal(mag, torch.zeros_like(mag)):
                    slack = 3 * 2.0 ** -24 * float(mag[torch.isfinite(mag)].max())
                    near[p, h, row // block] = exponent(big + slack, fmt) != exponent(max(big - slack, 0.0), fmt)
                now = need if n0 == base else max(need, old)
                lim = most(now - 127, fmt, dtype)
                if n0 > base and now > old:
                    was = c[p, h, row:row + n0 - base]
                    c[p, h, row:row + n0 - base] = rounded((was * 2.0 ** (old - now)).clamp(-lim, lim), fmt)
                e[p, h, row // block] = 255 if fmt == I8 and not torch.isfinite(y).all() else now
                v = (y * 2.0 ** (127 - now))
                c[p, h, row + n0 - base:row + n1 - base] = rounded(torch.where(torch.isfinite(v), v.clamp(-lim, lim), v), fmt)
                # a value that 32 bits move across a border: one step at most
                slack = 3 * 2.0 ** -24 * torch.nan_to_num(mag, posinf=0.0, neginf=0.0) * 2.0 ** (127 - now)
                step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(2.0 ** -6, 1e300))) - 3) if fmt == FP8 else torch.ones_like(v)
                moved = (rounded(v + slack, fmt) != rounded(v - slack, fmt)) & (slack > 0)
                tol[p, h, row + n0 - base:row + n1 - base] = torch.where(moved, step, 0.0)
    return c, e, tol, near


def assign(table, seq, want, free, page, T):
    """The loop: table, seq (lists) and free (a stack) are changed; (n_new, slots)."""
    B, cols = len(seq), len(table[0])
    P = lambda n: -(-n // page)  # noqa: E731
    asks = []
    for b in range(B):
        w = want[b]
        asks.append(seq[b] if w < 0 or w > cols * page or (T is not None and w - seq[b] > T) else w)
    for b in reversed(range(B)):
        for col in reversed(range(P(asks[b]), P(seq[b]))):
            free.append(table[b][col])
    n_new, slots, short = [0] * B, [[-1] * (T or 0) for _ in range(B)], False
    for b in range(B):
        held, need = seq[b], max(P(asks[b]) - P(seq[b]), 0)
        short = short or need > len(free)
        if asks[b] > held and (need == 0 or not short):
            for col in range(P(held), P(asks[b])):
                table[b][col] = free.pop()
            n_new[b] = asks[b] - held
            for t in range(min(n_new[b], T or 0)):
                p = held + t
                slots[b][t] = table[b][p // page] * page + p % page
        if asks[b] < held or n_new[b]:
            seq[b] = asks[b]
    return n_new, slots
