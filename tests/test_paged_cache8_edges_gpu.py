"""The paged cache in 8 bits where it can go wrong: odd numbers in hidden places, lengths of nothing, strides, bad pages, large offsets, many sequences, streams, graphs, and a
server's loop over all three operators (GPU)."""
import math
import random

import pytest
import torch

from dl_templates_amd.page_pool import page_assign_, page_pool
from dl_templates_amd.paged_cache8 import paged8_append_, paged8_attention
from tests import long_oracle as orc
from tests import paged8_oracle as orc8
from tests.test_paged_cache8_gpu import BF, F32, FP8, HF, I8, cache_for, gathered, ints, pool

pytestmark = pytest.mark.gpu


def attend(case, gen, **kw):
    """(o on the host, q, caches on the host, new tokens) of a case of test_paged_cache8_gpu.ATTN's form."""
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, fmt = case
    parts = cache_for(case, gen)
    q = torch.randn(B, H, T, dk, generator=gen).to(dtype)
    for f in kw.get("change", ()):
        f(*parts)
    kc, vc, ks, vs, table = parts
    scale = 0.3 / math.sqrt(dk)
    o = paged8_attention(q.cuda(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda(), ints(lens), window, n_sink, scale, None if n_new is None else ints(n_new))
    return o.cpu(), q, parts, n_new or [T] * B, scale


def check(case, o, q, parts, new, scale):
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, fmt = case
    kc, vc, ks, vs, table = parts
    for b in range(B):
        n = new[b]
        k, v = gathered(kc, ks, table, b, lens[b], dtype)[None], gathered(vc, vs, table, b, lens[b], dtype)[None]
        orc.check(o[b:b + 1, :, :n], orc.window(q[b:b + 1, :, :n], k, v, window, n_sink, scale)["o"], f"sequence {b}")
        assert (o[b, :, n:] == 0).all()


def drawn(seed):
    rng = random.Random(seed)
    G, Hkv, T = rng.choice([1, 2, 3, 5, 8]), rng.choice([1, 2, 3]), rng.choice([1, 1, 2, 4, 7, 16, 33, 70])
    page = rng.choice([16, 32, 48, 64, 128])
    block = rng.choice([x for x in range(16, page + 1, 16) if page % x == 0])
    B = rng.choice([1, 2, 5, 70]) if T < 8 else rng.randint(1, 2)
    padded = rng.random() < 0.5
    lens, new = [], []
    for _ in range(B):
        n = rng.randint(0, T) if padded else T
        new.append(n)
        lens.append(max(n, int(math.exp(rng.uniform(0, math.log(rng.choice([40, 700, 4000] if B < 9 else [40, 700])))))))
    return (B, G * Hkv, Hkv, T, page, block, lens, new if padded else None, rng.choice([16, 64, 72, 128]), rng.choice([16, 64, 88, 128]), rng.choice([None, None, 1, 30, 200, 1500]),
            rng.choice([0, 0, 3, 40]), rng.choice([BF, HF]), rng.choice([FP8, I8]))


@pytest.mark.parametrize("seed", range(40))
def test_drawn_cases(seed):
    case = drawn(seed)
    check(case, *attend(case, torch.Generator().manual_seed(seed)))


ODD = [
    # rows of up to 32, in whole heads and in runs; more rows
    (2, 4, 2, 4, 32, 16, [70, 40], None, 64, 64, None, 0, BF, FP8),
    (2, 8, 2, 3, 32, 32, [3000, 1000], None, 128, 128, 900, 20, BF, FP8),
    (1, 2, 1, 5, 16, 16, [5], None, 64, 128, None, 0, HF, FP8),
    (1, 6, 1, 30, 64, 64, [900], None, 128, 128, 300, 10, BF, FP8),
    (2, 4, 2, 4, 32, 16, [70, 40], None, 64, 64, None, 0, HF, I8),
    (2, 8, 2, 3, 32, 32, [3000, 1000], None, 128, 128, 900, 20, BF, I8),
    (1, 6, 1, 30, 64, 64, [900], None, 128, 128, 300, 10, HF, I8),
]


@pytest.mark.parametrize("case", ODD, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
@pytest.mark.parametrize("where", ["newest", "middle", "window"])
def test_nan_reaches_the_rows_that_see_it(case, where):
    """A NaN (e4m3) or a scale of NaN (its block, 16 tokens and more) at a key: rows that see it are NaN, the others what they are without it."""
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, fmt = case
    if where == "window" and window is None:
        pytest.skip("no window")
    at = {"newest": lens[0] - 1, "middle": max(0, lens[0] - T - 3), "window": lens[0] - T - (window or 0) + 1}[where]
    for tensor, number in ((0, False), (1, False)) + (((0, True), (1, True)) if fmt == FP8 else ()):
        hit = []

        def change(kc, vc, ks, vs, table):
            p, r = int(table[0, at // page]), at % page
            if number:
                (kc, vc)[tensor].view(torch.uint8)[p, 0, r] = 0x7f
                hit.append((at, at + 1))
            else:
                (ks, vs)[tensor].view(torch.uint8)[p, 0, r // block] = 255
                hit.append((at // block * block, at // block * block + block))
        o, q, parts, new, scale = attend(case, torch.Generator().manual_seed(5), change=[change])
        clean = attend(case, torch.Generator().manual_seed(5))[0]
        lo, hi = hit[0]
        G = H // Hkv
        for t in range(T):
            p = lens[0] - T + t
            sees = any((j <= p) and (window is None or p - j < window or j < n_sink) for j in range(lo, min(hi, lens[0])))
            got, want = o[0, :G, t], clean[0, :G, t]
            assert torch.isnan(got).all() if sees else torch.allclose(got.float(), want.float(), rtol=2 * torch.finfo(dtype).eps, atol=2e-2 * float(want.abs().max())), (where, t)
        assert torch.equal(o[0, G:], clean[0, G:]) and torch.equal(o[1:], clean[1:])


def test_scales_at_the_ends_of_their_range():
    for fmt in (FP8, I8):
        for e in (1, 40, 127, 200, 246):
            one = torch.ones(1, 1, 16, 64).to(fmt).cuda()
            sc = lambda v: torch.full((1, 1, 1), v, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)  # noqa: E731
            q = torch.zeros(1, 2, 1, 64, dtype=BF, device="cuda")
            o = paged8_attention(q, one, one, sc(127), sc(e), ints([[0]]), ints([9]))
            assert (o.double() == 2.0 ** (e - 127)).all(), (fmt, e)
            # scores: q . k = 64 q 2^(e - 127) for all keys alike, where that is finite
            o = paged8_attention(q + 2.0 ** (100 - e if e > 100 else 0), one, one, sc(e), sc(127), ints([[0]]), ints([9]))
            assert (o == 1).all(), (fmt, e)


def test_nothing_to_do():
    gen = torch.Generator().manual_seed(1)
    for case in ((3, 4, 2, 1, 16, 16, [0, 0, 0], [0, 1, 0], 64, 64, None, 0, BF, FP8), (2, 40, 1, 2, 16, 16, [0, 5], [2, 0], 128, 128, 9, 1, HF, I8)):
        o, *_ = attend(case, gen)
        assert (o == 0).all()
    kc, vc, ks, vs, table = (x.cuda() for x in pool(gen, 2, 2, 16, 16, [16, 16], 64, 64, FP8))
    before = [x.clone() for x in (kc, vc)] + [x.view(torch.uint8).clone() for x in (ks, vs)]
    empty = torch.empty(2, 2, 0, 64, dtype=BF, device="cuda")
    assert paged8_append_(kc, vc, ks, vs, empty, empty, table, ints([5, 0])) is None
    assert paged8_append_(kc, vc, ks, vs, empty, empty, table, ints([5, 0]), None, None, empty).shape == empty.shape
    assert paged8_attention(empty, kc, vc, ks, vs, table, ints([5, 0])).shape == empty.shape
    x = torch.randn(2, 2, 3, 64, dtype=BF, device="cuda")
    paged8_append_(kc, vc, ks, vs, x, x, table, ints([5, 9]), ints([0, -4]))
    none = torch.empty(0, 2, 3, 64, dtype=BF, device="cuda")
    assert paged8_append_(kc, vc, ks, vs, none, none, table[:0], ints([]), None, None, none).shape == none.shape
    assert paged8_attention(none, kc, vc, ks, vs, table[:0], ints([])).shape == none.shape
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((kc, vc, ks, vs), before))


@pytest.mark.parametrize("fmt", [FP8, I8])
def test_strides(fmt):
    """Keys and values in one tensor, tokens before heads, padded rows; q, k and v in layouts that are read as they are and in others."""
    gen = torch.Generator().manual_seed(2)
    B, H, Hkv, T, page, block, d = 3, 6, 2, 5, 32, 16, 72
    lens, new = [70, 5, 33], [5, 4, 1]
    kc, vc, ks, vs, table = pool(gen, B, Hkv, page, block, lens, d, d, fmt)
    n = kc.shape[0]
    both = torch.zeros(n, page, 2, Hkv, 80, dtype=torch.uint8, device="cuda").view(fmt)
    view = lambda i: both[:, :, i, :, :d].permute(0, 2, 1, 3)  # noqa: E731
    both_s = torch.zeros(page // block, n, 2, Hkv, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    view_s = lambda i: both_s[:, :, i].permute(1, 2, 0)  # noqa: E731
    for i, (c, s) in enumerate(((kc, ks), (vc, vs))):
        view(i).view(torch.uint8).copy_(c.view(torch.uint8)) if view(i).is_contiguous() else both.view(torch.uint8)[:, :, i, :, :d].copy_(c.view(torch.uint8).permute(0, 2, 1, 3))
        both_s.view(torch.uint8)[:, :, i].copy_(s.view(torch.uint8).permute(2, 0, 1))
    x = [torch.randn(B, T, h, d, generator=gen).to(BF) for h in (Hkv, Hkv, H)]
    want = [y.cuda() for y in (kc, vc, ks, vs)]
    tables = [orc.table(200, 20).cuda()]
    rope = (None, tables, "halves")
    plain = [y.permute(0, 2, 1, 3).contiguous().cuda() for y in x]
    q_want = paged8_append_(*want, plain[0], plain[1], table.cuda(), ints(lens), ints(new), rope, plain[2])
    o_want = paged8_attention(q_want, *want, table.cuda(), ints(lens), 40, 3, None, ints(new))
    for kind in ("tokens first", "odd rows", "dims first"):
        got = [view(0), view(1), view_s(0), view_s(1)]
        y = [t.cuda().permute(0, 2, 1, 3) for t in x]
        if kind == "odd rows":
            y = [torch.empty(*t.shape[:3], d + 3, dtype=BF, device="cuda")[..., 1:d + 1].copy_(t) for t in y]
        elif kind == "dims first":
            y = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in y]
        q = paged8_append_(*got, y[0], y[1], table.cuda(), ints(lens), ints(new), rope, y[2])
        assert torch.equal(q, q_want), kind
        for a, b in zip(got, want):
            used = a.contiguous().view(torch.uint8)
            assert torch.equal(used, b.view(torch.uint8)), kind
        wide = torch.full((B, 9), 10 ** 8, dtype=torch.int32, device="cuda")
        wide[:, 2:2 + table.shape[1]] = table.cuda()
        o = paged8_attention(q if kind != "odd rows" else torch.empty(*q.shape[:3], d + 3, dtype=BF, device="cuda")[..., 1:d + 1].copy_(q), *got, wide[:, 2:2 + table.shape[1]], ints(lens), 40,
                             3, None, ints(new))
        assert torch.equal(o, o_want), kind
    assert (both.view(torch.uint8)[..., d:] == 0).all()


@pytest.mark.parametrize("fmt", [FP8, I8])
def test_bad_pages_and_lengths(fmt):
    gen = torch.Generator().manual_seed(3)
    kc, vc, ks, vs, table = (x.cuda() for x in pool(gen, 2, 2, 16, 16, [64, 64], 64, 64, fmt))
    before = [x.view(torch.uint8).clone() for x in (kc, vc, ks, vs)]
    x = torch.randn(2, 2, 40, 64, dtype=BF, device="cuda")
    bad = torch.tensor([[-1, 2 ** 30, kc.shape[0], -2 ** 31]] * 2, dtype=torch.int32, device="cuda")
    paged8_append_(kc, vc, ks, vs, x, x, bad, ints([60, 40]))
    assert all(torch.equal(a.view(torch.uint8), b) for a, b in zip((kc, vc, ks, vs), before))
    assert torch.isfinite(paged8_attention(x, kc, vc, ks, vs, bad, ints([60, 40]))).all()
    assert torch.isfinite(paged8_attention(x[:, :, :1], kc, vc, ks, vs, bad, ints([60, 40]))).all()
    # lengths outside the table's row: what fits is written, what the row holds is read
    for lens, new in (([70, 64], [40, 40]), ([5, -3], [20, 3]), ([2 ** 31 - 1, 200], [40, 30])):
        a, w = [t.clone() for t in (kc, vc)] + [t.view(torch.uint8).clone().view(torch.float8_e8m0fnu) for t in (ks, vs)], None
        paged8_append_(*a, x, x, table, ints(lens), ints(new))
        c, e, _, _ = orc8.append(kc.cpu(), ks.cpu(), x.double().cpu(), torch.zeros_like(x, dtype=torch.float64).cpu(), table.cpu(), lens, new, BF)
        assert torch.equal(a[0].cpu().float().double(), c) and torch.equal(a[2].cpu().view(torch.uint8).int(), e), lens
        full = [min(max(n, 0), 64) for n in lens]
        o = paged8_attention(x[:, :, :1], kc, vc, ks, vs, table, ints(lens))
        assert torch.equal(o, paged8_attention(x[:, :, :1], kc, vc, ks, vs, table, ints(full)))


def test_offsets_past_32_bits():
    """Pages whose bytes lie behind 2^32 of the cache's start."""
    gen = torch.Generator().manual_seed(4)
    H, Hkv, page, d, n = 8, 8, 64, 128, 70000
    for fmt in (FP8, I8):
        kc, vc = (torch.zeros(n, Hkv, page, d, dtype=torch.uint8, device="cuda").view(fmt) for _ in range(2))   # 4.6e9 bytes
        ks, vs = (torch.full((n, Hkv, 1), 255, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
        small = [torch.zeros(8, Hkv, page, d, dtype=torch.uint8, device="cuda").view(fmt) for _ in range(2)] + [torch.zeros(8, Hkv, 1, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
                                                                                                                for _ in range(2)]
        far, near = ints([[n - 1, 3, n - 40, n - 7]]), ints([[7, 3, 1, 5]])
        for T in (200, 1, 40):
            x = [torch.randn(1, h, T, d, generator=gen).to(BF).cuda() for h in (Hkv, Hkv, H)]
            lens = ints([{200: 200, 1: 201, 40: 241}[T]])
            paged8_append_(kc, vc, ks, vs, x[0], x[1], far, lens)
            paged8_append_(*small, x[0], x[1], near, lens)
            for i in range(4):
                a, b = int(far[0, i]), int(near[0, i])
                assert torch.equal(kc[a].view(torch.uint8), small[0][b].view(torch.uint8)) and torch.equal(vc[a].view(torch.uint8), small[1][b].view(torch.uint8))
            assert torch.equal(paged8_attention(x[2], kc, vc, ks, vs, far, lens), paged8_attention(x[2], *small, near, lens))
        del kc, vc


@pytest.mark.parametrize("B", [65, 700, 4096, 4097])
def test_many_sequences(B):
    """More sequences than lanes, than a lane's list, and than the lists of runs hold; one context is long."""
    gen = torch.Generator().manual_seed(6)
    lens = [1 + 7 * b % 37 for b in range(B)]
    lens[B // 2], lens[B - 1] = 3000, 0
    page, d = 16, 32
    need = [-(-n // page) for n in lens]
    numbers = torch.randperm(sum(need) + 1, generator=gen)
    table, at = torch.zeros(B, max(need), dtype=torch.int32), 0
    for b in range(B):
        table[b, :need[b]] = numbers[at:at + need[b]].int()
        at += need[b]
    kc, vc, ks, vs, _ = pool(gen, 1, 1, page, 16, [page * (sum(need) - 2)], d, d, FP8)
    q = torch.randn(B, 2, 1, d, generator=gen).to(BF)
    o = paged8_attention(q.cuda(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda(), ints(lens), None, 0, 0.2).cpu()
    for b in [0, 1, 63, 64, B // 2, B - 2, B - 1] + list(range(0, B, 97)):
        k, v = gathered(kc, ks, table, b, lens[b], BF)[None], gathered(vc, vs, table, b, lens[b], BF)[None]
        orc.check(o[b:b + 1], orc.window(q[b:b + 1], k, v, None, 0, 0.2)["o"], f"sequence {b}")


def test_equal_calls_give_equal_bits_on_any_stream():
    gen = torch.Generator().manual_seed(7)
    cases = [(20, 8, 2, 1, 64, 32, [300 * b + 1 for b in range(20)], None, 128, 128, None, 0, BF, FP8), (3, 8, 2, 40, 64, 32, [3000, 50, 900], None, 64, 64, None, 4, HF, I8)]
    for case in cases:
        B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, fmt = case
        parts = [x.cuda() for x in cache_for(case, gen)]
        q = torch.randn(B, H, T, dk, generator=gen).to(dtype).cuda()
        seq = ints(lens)
        first = paged8_attention(q, *parts, seq, window, n_sink)
        side = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        outs = []
        for i in range(12):
            with torch.cuda.stream(side[i % 3]):
                outs.append(paged8_attention(q, *parts, seq, window, n_sink))
        torch.cuda.synchronize()
        assert all(torch.equal(o, first) for o in outs)


def test_inference_mode_and_no_graph():
    gen = torch.Generator().manual_seed(8)
    kc, vc, ks, vs, table = (x.cuda() for x in pool(gen, 2, 2, 16, 16, [40, 40], 64, 64, FP8))
    x = torch.randn(2, 2, 3, 64, dtype=BF, device="cuda", requires_grad=True)
    q = paged8_append_(kc, vc, ks, vs, x, x, table, ints([40, 30]), None, None, x)
    o = paged8_attention(x, kc, vc, ks, vs, table, ints([40, 30]))
    assert not q.requires_grad and not o.requires_grad
    with torch.inference_mode():
        q2 = paged8_append_(kc, vc, ks, vs, x, x, table, ints([40, 30]), None, None, x)
        assert torch.equal(q2, q) and torch.equal(paged8_attention(x, kc, vc, ks, vs, table, ints([40, 30])), o)
        t, s, p = ints([[0, 0]]), ints([0]), page_pool(2)
        assert page_assign_(t, s, ints([20]), p, 16, 32)[0].tolist() == [20]


@pytest.mark.parametrize("layout", ["blocks", "halves"])
@pytest.mark.parametrize("sections", [(8, 16, 8), (5, 11, 0)])
def test_given_positions_of_several_axes(layout, sections):
    """Positions that are handed in, one set for all sequences or one each, some of them negative: keys and queries turn by those, not by their places."""
    gen = torch.Generator().manual_seed(9)
    B, H, Hkv, T, page, d, lens, new = 2, 4, 2, 21, 32, 64, [50, 30], [21, 13]
    kc, vc, ks, vs, table = pool(gen, B, Hkv, page, 16, lens, d, d, FP8)
    k, v, q = (torch.randn(B, h, T, d, generator=gen).to(BF) for h in (Hkv, Hkv, H))
    tables = [orc.table(40, r) for r in sections]
    for shape in ((3, T), (3, B, T)):
        pos = torch.randint(-3, 40, shape, generator=gen).int()
        live = torch.tensor([[t < n for t in range(T)] for n in new])
        each = torch.where(live, pos if pos.dim() == 3 else pos[:, None], -1).int()      # padding does not turn
        rk, rq = orc.rotate(k, each, tables, layout), orc.rotate(q, each, tables, layout)
        got = [x.cuda() for x in (kc, vc, ks, vs)]
        out = paged8_append_(*got, k.cuda(), v.cuda(), table.cuda(), ints(lens), ints(new), (pos.cuda(), [t.cuda() for t in tables], layout), q.cuda())
        c, e, tol, near = orc8.append(kc, ks, rk[0], k.double().abs().amax(-1, keepdim=True).expand_as(k) * 2, table, lens, new, BF)
        assert not near.any() and torch.equal(got[2].cpu().view(torch.uint8).int(), e)
        assert ((got[0].cpu().float().double() - c).abs() <= tol).all()
        orc.check(out.cpu(), rq, "queries")


def test_a_block_of_nan_stays_until_it_is_begun_again():
    """int8: one NaN makes its block's scale NaN; tokens that join keep it so, and the block's next first token ends it."""
    kc, vc = (torch.zeros(1, 1, 32, 64, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((1, 1, 2), 100, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2))
    x = torch.ones(1, 1, 4, 64, dtype=BF, device="cuda")
    bad = x.clone()
    bad[0, 0, 2, 9] = float("inf")
    bits = lambda: ks.view(torch.uint8).flatten().tolist()  # noqa: E731
    paged8_append_(kc, vc, ks, vs, bad, x, ints([[0]]), ints([4]))
    assert bits() == [255, 100] and vs.view(torch.uint8).flatten().tolist()[0] == 127 - 6
    paged8_append_(kc, vc, ks, vs, x, x, ints([[0]]), ints([8]))
    assert bits() == [255, 100]
    q = torch.ones(1, 1, 2, 64, dtype=BF, device="cuda")
    assert torch.isnan(paged8_attention(q, kc, vc, ks, vs, ints([[0]]), ints([8]))).all()
    paged8_append_(kc, vc, ks, vs, x, x, ints([[0]]), ints([4]))
    assert bits() == [127 - 6, 100]
    assert (paged8_attention(q, kc, vc, ks, vs, ints([[0]]), ints([4])) == 1).all()


class Server:
    """Requests that come, take tokens (some of them guessed and taken back) and end, over the three operators.  What a sequence was given is kept beside it."""

    def __init__(self, fmt, dtype, seed, T):
        self.gen, self.rng = torch.Generator().manual_seed(seed), random.Random(seed)
        self.B, self.H, self.Hkv, self.d, self.page, self.block, self.T, self.dtype, self.fmt = 5, 8, 2, 64, 32, 16, T, dtype, fmt
        n, self.cols = 24, 10
        self.kc, self.vc = (torch.randint(0, 256, (n, self.Hkv, self.page, self.d), generator=self.gen).to(torch.uint8).cuda().view(fmt) for _ in range(2))
        self.ks, self.vs = (torch.randint(0, 256, (n, self.Hkv, self.page // self.block), generator=self.gen).to(torch.uint8).cuda().view(torch.float8_e8m0fnu) for _ in range(2))
        self.table, self.seq, self.pool = torch.full((self.B, self.cols), 10 ** 6, dtype=torch.int32, device="cuda"), ints([0] * self.B), page_pool(n)
        self.tables = [orc.table(self.cols * self.page, self.d // 2).cuda()]
        mk = lambda h: torch.zeros(self.B, h, T, self.d, dtype=dtype, device="cuda")  # noqa: E731
        self.k, self.v, self.q, self.want = mk(self.Hkv), mk(self.Hkv), mk(self.H), ints([0] * self.B)
        self.held = [0] * self.B

    def inputs(self):
        for x in (self.k, self.v, self.q):
            x.copy_(torch.randn(x.shape, generator=self.gen))
        want = []
        for n in self.held:
            kind = self.rng.random()
            want.append(-1 if kind < 0.1 else 0 if kind < 0.15 else max(0, n - self.rng.randint(0, 3)) if kind < 0.3 else n + self.rng.randint(1, self.T))
        self.want.copy_(ints(want))

    def step(self):
        n_new, slots = page_assign_(self.table, self.seq, self.want, self.pool, self.page, self.T)
        q = paged8_append_(self.kc, self.vc, self.ks, self.vs, self.k, self.v, self.table, self.seq, n_new, (None, self.tables, "halves"), self.q)
        return n_new, slots, q, paged8_attention(q, self.kc, self.vc, self.ks, self.vs, self.table, self.seq, 100, 5, None, n_new)

    def check(self, out):
        n_new, slots, q, o = (x.cpu() for x in out)
        seq, table = self.seq.tolist(), self.table.cpu()
        for b in range(self.B):
            n = int(n_new[b])
            assert seq[b] == (self.held[b] + n if n else seq[b]) and (n == 0 or seq[b] == int(self.want[b]))
            for t in range(self.T):
                p = seq[b] - n + t
                assert int(slots[b, t]) == (int(table[b, p // self.page]) * self.page + p % self.page if t < n else -1)
            k, v = (gathered(c.cpu(), s.cpu(), table.clamp(0, 23), b, seq[b], self.dtype)[None] for c, s in ((self.kc, self.ks), (self.vc, self.vs)))
            if n:
                # the newest tokens are what was given, to a rounding of 8 bits
                pos = torch.arange(seq[b] - n, seq[b])[None].int()
                x = orc.rotate(self.k[b:b + 1, :, :n].cpu(), pos, [t.cpu() for t in self.tables], "halves")[0]
                off = (k[0, :, seq[b] - n:].double() - x[0]).abs()
                top = x[0].abs().max()
                assert (off <= (x[0].abs() * 2.0 ** -4 + top * 2.0 ** -12 if self.fmt == FP8 else top * 2.0 ** -6)).all()
                assert torch.isfinite(k).all()
            scale = 1.0 / math.sqrt(self.d)
            orc.check(o[b:b + 1, :, :n], orc.window(q[b:b + 1, :, :n], k, v, 100, 5, scale)["o"], f"sequence {b}")
            assert (o[b, :, n:] == 0).all()
        self.held = seq


@pytest.mark.parametrize("fmt, dtype, T", [(FP8, BF, 1), (FP8, HF, 9), (I8, BF, 40), (I8, HF, 3)])
def test_a_servers_loop(fmt, dtype, T):
    s = Server(fmt, dtype, 11, T)
    for _ in range(25):
        s.inputs()
        s.check(s.step())


@pytest.mark.parametrize("fmt, T", [(FP8, 4), (I8, 1), (FP8, 60)])
def test_a_captured_step(fmt, T):
    """The whole step captured once and replayed on what the tensors hold then, with eager work between, against a server that runs it eagerly."""
    a, b = Server(fmt, BF, 12, T), Server(fmt, BF, 12, T)
    for s in (a, b):
        s.inputs()
        s.check(s.step())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = a.step()
    for i in range(12):
        for s in (a, b):
            s.inputs()
        g.replay()
        want = b.step()
        for x, y in zip(out, want):
            assert torch.equal(x, y), i
        for x, y in ((a.kc, b.kc), (a.vc, b.vc), (a.ks, b.ks), (a.vs, b.vs), (a.seq, b.seq), (a.table, b.table), (a.pool, b.pool)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), i
        a.check(out)
        b.check(want)


@pytest.mark.parametrize("T, d, dtype, fmt, window, n_sink", [(40, 64, HF, I8, None, 0), (130, 128, BF, FP8, None, 0), (40, 128, HF, FP8, 4300, 70), (130, 64, BF, I8, 4222, 1)])
def test_a_workgroup_with_more_than_64_chunks(T, d, dtype, fmt, window, n_sink):
    """64 sequences whose tables name the same pages: every workgroup walks the whole context of 4500 tokens."""
    gen = torch.Generator().manual_seed(70)
    case = (1, 8, 8, T, 64, 32, [4500], None, d, d, window, n_sink, dtype, fmt)
    kc, vc, ks, vs, table = cache_for(case, gen)
    q = torch.randn(1, 8, T, d, generator=gen).to(dtype)
    scale = 0.3 / math.sqrt(d)
    o = paged8_attention(q.cuda().expand(64, -1, -1, -1).contiguous(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda().expand(64, -1).contiguous(), ints([4500] * 64), window, n_sink,
                         scale)
    assert (o == o[:1]).all()
    check(case, o[:1].cpu(), q, (kc, vc, ks, vs, table), [T], scale)


@pytest.mark.parametrize("T, lens", [(1, [5000]), (3, [20001]), (1, [3000] * 40), (40, [5000]), (1, [300]), (5, [1000] * 3), (1, [64] * 300)])
@pytest.mark.parametrize("fmt", [FP8, I8])
def test_infinite_values_where_parts_are_joined(T, lens, fmt):
    """A block of values past the type's largest number, in one dim, at a sequence's end: that dim is infinite, the others are what they are."""
    gen = torch.Generator().manual_seed(90)
    B, Hkv, d, page = len(lens), 2, 128, 64
    case = (B, 2 * Hkv, Hkv, T, page, 16, lens, None, d, d, None, 0, BF, fmt)

    def end(kc, vc, ks, vs, table):
        for b, n in enumerate(lens):
            t = n - T - 1   # every row sees it
            block, p = t % page // 16, int(table[b, t // page])
            c = vc[p, 0, 16 * block:16 * block + 16].view(torch.uint8)
            c.zero_()
            c[:, 5] = 0x7e if fmt == FP8 else 127
            vs[p, 0].view(torch.uint8)[block] = 254

    o, q, parts, new, scale = attend(case, gen, change=[end])
    assert torch.isposinf(o[:, :2, :, 5]).all() and torch.isfinite(o[:, 2:]).all()
    kc, vc, ks, vs, table = parts
    for b, n in enumerate(lens):
        k, v = gathered(kc, ks, table, b, n, BF)[None], gathered(vc, vs, table, b, n, BF)[None]
        v[:, 0, :, 5] = 0   # the infinities are looked at above: a dense product in 64 bits multiplies hidden ones by 0
        o[b, :2, :, 5] = 0
        orc.check(o[b:b + 1], orc.window(q[b:b + 1], k, v, None, 0, scale)["o"], f"sequence {b}")


@pytest.mark.parametrize("fmt", [FP8, I8])
def test_traced_calls_depend_on_their_inputs(fmt):
    def inputs(seed):
        s = Server(fmt, BF, seed, 7)
        s.inputs()
        s.want.clamp_(min=1)
        return s.table, s.seq, s.want, s.pool, s.kc, s.vc, s.ks, s.vs, s.k, s.v, s.q
    tables = [orc.table(320, 32).cuda()]

    def step(table, seq, want, pool, kc, vc, ks, vs, k, v, q):
        n_new, slots = page_assign_(table, seq, want, pool, 32, 7)
        r = paged8_append_(kc, vc, ks, vs, k, v, table, seq, n_new, (None, tables, "halves"), q)
        return n_new, slots, r, paged8_attention(r, kc, vc, ks, vs, table, seq, 100, 5, None, n_new)

    def fill(table, seq, want, pool, kc, vc, ks, vs, k, v, q):
        before = seq + 0
        n_new, slots = page_assign_(table, seq, want, pool, 32)
        assert slots is None and paged8_append_(kc, vc, ks, vs, k, v, table, seq, n_new) is None
        return before, seq + 0, n_new, paged8_attention(q, kc, vc, ks, vs, table, seq, None, 0, None, n_new)
    for f in (step, fill):
        traced = torch.jit.trace(f, inputs(30), check_trace=False)
        for seed in (31, 32, 33, 34):
            a, b = inputs(seed), inputs(seed)
            got, want = traced(*a), f(*b)
            assert all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(tuple(got) + a, tuple(want) + b)), (f.__name__, seed)


def test_calls_are_timed():
    """With per-launch timing on, calls do what they do without it, and every launch leaves a record."""
    from dl_templates_amd import _lib
    gen = torch.Generator().manual_seed(40)
    cases = [(1, 8, 2, 1, 64, 64, [300], None, 64, 64, None, 0, BF, FP8), (2, 8, 2, 1, 64, 64, [5000, 700], None, 128, 128, None, 0, HF, I8),
             (1, 8, 2, 100, 32, 32, [700], None, 128, 128, None, 0, BF, I8)]
    for case in cases:
        B, H, Hkv, T, page, block, lens, _, dk, dv, _, _, dtype, fmt = case
        kc, vc, ks, vs, table = (x.cuda() for x in cache_for(case, gen))
        q = torch.randn(B, H, T, dk, generator=gen).to(dtype).cuda()
        want = paged8_attention(q, kc, vc, ks, vs, table, ints(lens))
        _lib.timing_enable(True)
        try:
            got = paged8_attention(q, kc, vc, ks, vs, table, ints(lens))
            records = _lib.timing_collect()
        finally:
            _lib.timing_enable(False)
        assert torch.equal(got, want) and len(records) >= 1


@pytest.mark.parametrize("T, lens, d", [(1, [5, 300, 700], 64), (1, [33, 900], 128), (3, [5003, 2100], 128), (1, [4007], 64), (40, [333, 90], 128)])
@pytest.mark.parametrize("fmt", [FP8, I8])
def test_scales_behind_a_sequence_leave_every_bit(T, lens, d, fmt):
    """Blocks that hold nothing of a sequence share tiles with its last ones.  Whatever their scales and numbers are, no sum is touched (one that was would be formed again, another way)."""
    gen = torch.Generator().manual_seed(50)
    case = (len(lens), 4, 2, T, 128, 16, lens, None, d, d, None, 0, HF, fmt)
    kc, vc, ks, vs, table = cache_for(case, gen)
    q = torch.randn(len(lens), 4, T, d, generator=gen).half().cuda()
    out = []
    for byte in (255, 254, 127, 0):
        parts = [x.clone() for x in (kc, vc, ks, vs)]
        for x in parts[2:]:
            u = x.view(torch.uint8)
            u[u == 255] = byte   # cache_for leaves NaN there and nowhere else
        out.append(paged8_attention(q, *(x.cuda() for x in parts), table.cuda(), ints(lens), None, 0, 0.1))
    assert all(torch.equal(x, out[0]) for x in out) and torch.isfinite(out[0]).all()


def records_of(call):
    """(what the call gives, names of the launches that it leaves on record)"""
    from dl_templates_amd import _lib
    _lib.timing_enable(True)
    try:
        out = call()
        records = _lib.timing_collect()
    finally:
        _lib.timing_enable(False)
    assert all(ms > 0 for _, ms in records)
    return out, [n for n, _ in records]


@pytest.mark.parametrize("T, lens, d, launches", [(1, [300], 64, 1), (1, [5000, 700], 128, 2), (6, [5000, 700], 128, 2), (100, [200], 128, 1), (40, [5000], 64, 2), (100, [5000], 128, 2)])
@pytest.mark.parametrize("fmt", [FP8, I8])
def test_every_launch_leaves_a_record(T, lens, d, launches, fmt):
    """Whole heads and unshared rows are one launch, runs and shared keys two; an append and a call for pages one each."""
    B = len(lens)
    case = (B, 8, 2, T, 64, 64, lens, None, d, d, None, 0, BF, fmt)
    kc, vc, ks, vs, table = (x.cuda() for x in cache_for(case, torch.Generator().manual_seed(41)))
    k, v, q = (torch.randn(B, h, T, d, dtype=BF, device="cuda") for h in (2, 2, 8))
    assert records_of(lambda: paged8_append_(kc, vc, ks, vs, k, v, table, ints(lens), None, None, q))[1] == ["rope2d"]
    o, names = records_of(lambda: paged8_attention(q, kc, vc, ks, vs, table, ints(lens)))
    assert names == ["attn_fwd"] * launches and torch.equal(o, paged8_attention(q, kc, vc, ks, vs, table, ints(lens)))
    pages, seq = page_pool(64), ints([0] * B)
    (n_new, _), names = records_of(lambda: page_assign_(torch.zeros(B, 9, dtype=torch.int32, device="cuda"), seq, ints([77] * B), pages, 16))
    assert names == ["page_assign"] and n_new.tolist() == [77] * B
