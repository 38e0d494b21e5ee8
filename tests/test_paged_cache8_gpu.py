"""The paged cache in 8 bits: append and attention against their 64-bit forms (GPU)."""
import math

import pytest
import torch

from dl_templates_amd.paged_cache8 import paged8_append_, paged8_attention
from tests import long_oracle as orc
from tests import paged8_oracle as orc8

pytestmark = pytest.mark.gpu
BF, HF, F32, FP8, I8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
name = lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c)  # noqa: E731


def pool(gen, B, Hkv, page, block, lens, dk, dv, fmt, cols=None):
    """Caches of any numbers, their scales around 2^-6, and a table that hands pages out in any order."""
    cols = cols or max(1, -(-max(lens) // page))
    n = B * cols + 3
    table = torch.randperm(n, generator=gen)[:B * cols].reshape(B, cols).to(torch.int32)

    def mk(d):
        if fmt == FP8:
            return (torch.randn(n, Hkv, page, d, generator=gen) * 100).clamp(-448, 448).to(FP8)
        return torch.randint(-127, 128, (n, Hkv, page, d), generator=gen).to(I8)
    sc = lambda: torch.randint(118, 124, (n, Hkv, page // block), generator=gen).to(torch.uint8).view(torch.float8_e8m0fnu)  # noqa: E731
    return mk(dk), mk(dv), sc(), sc(), table


APPEND = [
    # B, H, Hkv, T, page, block, lens, n_new, dk, dv, layout, dtype, format
    (1, 1, 1, 1, 16, 16, [1], None, 64, 64, "halves", BF, FP8),
    (3, 4, 2, 5, 16, 16, [5, 40, 17], [5, 3, 0], 64, 64, "blocks", HF, I8),
    (2, 0, 3, 33, 48, 48, [33, 100], None, 24, 40, "halves", F32, FP8),
    (2, 6, 2, 9, 96, 32, [12, 200], [9, 1], 128, 128, None, BF, I8),
    (1, 2, 1, 4, 32, 32, [6], None, 16, 8, "blocks", BF, FP8),
    (4, 8, 2, 1, 64, 64, [64, 65, 1, 100], None, 128, 128, "halves", BF, FP8),
    (4, 8, 2, 1, 128, 128, [64, 65, 129, 100], None, 128, 128, "halves", BF, I8),
    (2, 4, 4, 300, 256, 128, [300, 777], [300, 259], 128, 128, "halves", BF, FP8),
    (2, 4, 4, 300, 64, 16, [300, 777], [1, 300], 80, 96, "blocks", HF, FP8),
    (2, 4, 1, 70, 80, 80, [170, 77], [70, 7], 104, 120, "halves", F32, I8),
    (3, 5, 1, 12, 64, 64, [170, 77, 12], None, 8, 8, "blocks", BF, I8),
    (5, 3, 1, 8, 64, 64, [9, 70, 61, 64, 128], None, 128, 64, "halves", HF, FP8),
]


@pytest.mark.parametrize("sections", ["one", "several"])
@pytest.mark.parametrize("case", APPEND, ids=name)
def test_append_against_64_bits(case, sections):
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, layout, dtype, fmt = case
    if layout is None and sections == "several":
        pytest.skip("no rotation")
    gen = torch.Generator().manual_seed(4)
    kc, vc, ks, vs, table = pool(gen, B, Hkv, page, block, lens, dk, dv, fmt)
    mk = lambda h, d: torch.randn(B, T, h, d, generator=gen).to(dtype).transpose(1, 2)  # noqa: E731
    k, v, q = mk(Hkv, dk), mk(Hkv, dv), mk(H, dk) if H else None
    k[:, :, T // 2:] *= 30   # scales that grow
    # one axis that turns all pairs; three with odd sections that leave dims alone
    r = dk // 2
    tables = [orc.table(1000, r)] if sections == "one" else [orc.table(1000, r // 4 + 1), orc.table(300, 0), orc.table(50, r // 3)]
    new = n_new or [T] * B
    pos = torch.tensor([[lens[b] - new[b] + t if t < new[b] else -1 for t in range(T)] for b in range(B)], dtype=torch.int32)[None].repeat(len(tables), 1, 1)
    zero = lambda x: torch.zeros_like(x, dtype=torch.float64)  # noqa: E731
    if layout is None:
        rq, rk = None if q is None else (q.double(), zero(q)), k.double()
    else:
        rq, rk = None if q is None else orc.rotate(q, pos, tables, layout), orc.rotate(k, pos, tables, layout)[0]
    mag = zero(k) if layout is None else k.double().abs().amax(-1, keepdim=True).expand_as(k) * 2
    wk, wv = orc8.append(kc, ks, rk, mag, table, lens, new, dtype), orc8.append(vc, vs, v.double(), zero(v), table, lens, new, dtype)
    kg, vg, ksg, vsg = (x.cuda() for x in (kc, vc, ks, vs))
    rope = None if layout is None else (None, [t.cuda() for t in tables], layout)
    out = paged8_append_(kg, vg, ksg, vsg, k.cuda(), v.cuda(), table.cuda(), ints(lens), None if n_new is None else ints(n_new), rope, None if q is None else q.cuda())
    for got, got_s, (c, e, tol, near), what in ((kg, ksg, wk, "keys"), (vg, vsg, wv, "values")):
        assert not near.any()
        assert torch.equal(got_s.cpu().view(torch.uint8).int(), e), what
        off = (got.cpu().to(torch.float32).double() - c).abs()
        assert (off <= tol).all(), f"{what}: {int((off > tol).sum())} numbers"
    if q is None:
        assert out is None
    else:
        orc.check(out.cpu(), rq, "queries")


def test_values_after_growth_are_near_what_was_appended():
    """A block filled token by token, each larger than the last: numbers stay within what all roundings can add up to."""
    for fmt in (FP8, I8):
        x = torch.randn(64, 1, 1, 64, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.arange(64) / 8.0)[:, None, None, None]
        x = x.to(BF).cuda()
        kc, vc = (torch.empty(1, 1, 64, 64, dtype=torch.uint8, device="cuda").fill_(200).view(fmt) for _ in range(2))
        ks, vs = (torch.full((1, 1, 1), 255, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
        for t in range(64):
            paged8_append_(kc, vc, ks, vs, x[t][None], x[t][None], ints([[0]]), ints([t + 1]))
        got, want = orc8.values(kc.cpu(), ks.cpu())[0, 0], x[:, 0, 0].double().cpu()
        assert torch.equal(kc.view(torch.uint8), vc.view(torch.uint8))
        s = float(orc8.scales(ks.cpu()))
        assert s == 2.0 ** orc8.exponent(float(want.abs().max()), fmt)
        # int8: half a step at each scale, 1/2 (1 + 1/2 + 1/4 + ..) of the last one; e4m3: one rounding, and half of the smallest number at each scale
        bound = s * torch.ones_like(want) if fmt == I8 else want.abs() * 2.0 ** -4 + s * 2.0 ** -9
        assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("fmt", [FP8, I8])
def test_append_of_odd_numbers(fmt, dtype):
    """Zeros, the type's largest and smallest numbers, infinities and NaN, each in a block of its own."""
    top = torch.finfo(dtype).max
    rows = [torch.zeros(16, 64), torch.full((16, 64), top), torch.full((16, 64), float(torch.finfo(dtype).smallest_normal)), torch.randn(16, 64), torch.randn(16, 64), torch.randn(16, 64)]
    rows[3][5, 7], rows[4][0, 0], rows[5][15] = float("nan"), -math.inf, math.inf
    x = torch.cat(rows).to(dtype)[None, None]
    kc, vc = (torch.zeros(1, 1, 96, 64, dtype=torch.uint8, device="cuda").view(fmt) for _ in range(2))
    ks, vs = (torch.zeros(1, 1, 6, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
    paged8_append_(kc, vc, ks, vs, x.cuda(), x.cuda(), ints([[0]]), ints([96]))
    zero = torch.zeros(1, 1, 96, 64, dtype=torch.uint8).view(fmt)
    c, e, _, _ = orc8.append(zero, torch.zeros(1, 1, 6, dtype=torch.uint8), x.double(), torch.zeros_like(x, dtype=torch.float64), torch.zeros(1, 1, dtype=torch.int32), [96], [96], dtype)
    assert torch.equal(ks.cpu().view(torch.uint8).int(), e) and torch.equal(vs.cpu().view(torch.uint8).int(), e)
    got = kc.cpu().float().double()
    keep = torch.ones(96, dtype=torch.bool) if fmt == FP8 else torch.arange(96) < 48   # numbers at a scale that is NaN are anything
    assert torch.equal(torch.nan_to_num(got[0, 0, keep], nan=1e9), torch.nan_to_num(c[0, 0, keep], nan=1e9))
    if dtype == HF:
        assert torch.isfinite(orc8.values(kc.cpu(), ks.cpu())[0, 0, :48].to(HF)).all()


ATTN = [
    # B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, sinks, dtype, format
    (1, 1, 1, 1, 16, 16, [1], None, 64, 64, None, 0, BF, FP8),
    (3, 4, 2, 1, 16, 16, [0, 5, 100], None, 64, 64, None, 0, HF, I8),
    (2, 8, 1, 1, 64, 32, [300, 64], None, 128, 128, 100, 4, BF, FP8),
    (2, 6, 2, 3, 48, 48, [49, 500], None, 80, 80, 64, 5, HF, FP8),
    (4, 2, 2, 4, 32, 16, [0, 3, 200, 4], [0, 1, 4, 2], 128, 128, None, 0, BF, I8),
    (1, 16, 1, 7, 16, 16, [1000], None, 128, 64, 333, 40, BF, FP8),
    (2, 32, 2, 40, 16, 16, [1000, 41], [40, 33], 64, 64, None, 0, BF, I8),
    (1, 64, 1, 3, 16, 16, [77], None, 32, 32, 16, 1, HF, FP8),
    (1, 2, 1, 200, 128, 128, [3000], None, 96, 96, 700, 9, BF, FP8),
    (1, 8, 8, 1, 16, 16, [4000], None, 64, 64, None, 0, HF, FP8),
    (1, 8, 8, 1, 64, 64, [4000], None, 128, 128, None, 0, BF, I8),
    (5, 8, 1, 2, 16, 16, [317, 326, 356, 352, 293], [1, 0, 2, 1, 2], 104, 104, None, 0, BF, FP8),
    (6, 32, 8, 185, 96, 48, [54, 217, 627, 366, 183, 569], [48, 149, 73, 127, 143, 44], 112, 16, 582, 0, BF, I8),
    (2, 4, 2, 30, 32, 32, [6000, 5000], [3, 30], 64, 64, None, 4, HF, FP8),
    (3, 4, 4, 300, 64, 64, [1500, 900, 300], [20, 300, 0], 128, 128, 700, 2, BF, FP8),
    (40, 8, 4, 1, 32, 32, [37 * (b % 9) + 5000 * (b == 7) for b in range(40)], None, 128, 128, None, 0, BF, FP8),
    (40, 12, 4, 2, 64, 16, [61 * (b % 9) + 4 + 3000 * (b == 9) for b in range(40)], None, 72, 40, 1000, 20, HF, I8),
    (2, 3, 3, 1, 16, 16, [2500, 2499], None, 8, 24, 2000, 0, BF, FP8),
]


def cache_for(case, gen):
    """Caches, scales and table; what lies behind a sequence's last token, and in pages that are nobody's, is NaN, its scales are NaN."""
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, fmt = case
    kc, vc, ks, vs, table = pool(gen, B, Hkv, page, block, lens, dk, dv, fmt)
    used = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for b in range(B):
        for p in range(lens[b]):
            used[table[b, p // page], p % page] = True
    if fmt == FP8:
        for x in (kc, vc):
            x.view(torch.uint8).transpose(1, 2)[~used] = 0x7f
    gone = ~used.reshape(-1, page // block, block).any(-1)
    for x in (ks, vs):
        x.view(torch.uint8).transpose(1, 2)[gone] = 255
    return kc, vc, ks, vs, table


def gathered(cache, scale, table, b, n, dtype):
    """What rows of sequence b hold: [Hkv, n, d]"""
    t = table[b].long()
    x = orc8.values(cache[t], scale[t]).transpose(0, 1)
    return x.reshape(cache.shape[1], -1, cache.shape[3])[:, :n].to(dtype)


@pytest.mark.parametrize("case", ATTN, ids=name)
def test_attention_against_64_bits(case):
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, fmt = case
    gen = torch.Generator().manual_seed(3)
    kc, vc, ks, vs, table = cache_for(case, gen)
    q = torch.randn(B, H, T, dk, generator=gen).to(dtype)
    new = n_new or [T] * B
    scale = 0.3 / math.sqrt(dk)
    o = paged8_attention(q.cuda(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda(), ints(lens), window, n_sink, scale, None if n_new is None else ints(n_new)).cpu()
    for b in range(B):
        n = new[b]
        k, v = gathered(kc, ks, table, b, lens[b], dtype)[None], gathered(vc, vs, table, b, lens[b], dtype)[None]
        orc.check(o[b:b + 1, :, :n], orc.window(q[b:b + 1, :, :n], k, v, window, n_sink, scale)["o"], f"sequence {b}")
        assert (o[b, :, n:] == 0).all()
