"""The paged cache: append and attention against their 64-bit forms (GPU)."""
import math

import pytest
import torch

from dl_templates_amd.paged_cache import paged_append_, paged_attention
from tests import long_oracle as orc

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def pool(gen, B, Hkv, page, lens, dk, dv, dtype, cols=None, fill=None):
    """Caches with unused pages, a table that hands pages out in any order."""
    cols = cols or max(1, -(-max(lens) // page))
    n = B * cols + 3
    table = torch.randperm(n, generator=gen)[:B * cols].reshape(B, cols).to(torch.int32)
    mk = lambda d: (torch.randn(n, Hkv, page, d, generator=gen) if fill is None else torch.full((n, Hkv, page, d), fill)).to(dtype)  # noqa: E731
    return mk(dk), mk(dv), table


def gathered(cache, table, b, n):
    """Rows of sequence b: [Hkv, n, d]"""
    rows = cache[table[b].long()].transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])
    return rows[:, :n]


ATTN = [
    # B, H, Hkv, T, page, lens, n_new, dk, dv, window, sinks, dtype
    (1, 1, 1, 1, 16, [1], None, 64, 64, None, 0, BF),
    (3, 4, 2, 1, 16, [0, 5, 100], None, 64, 64, None, 0, HF),
    (2, 8, 1, 1, 64, [300, 64], None, 128, 128, 100, 4, BF),
    (2, 6, 2, 3, 48, [49, 500], None, 80, 80, 64, 5, HF),
    (4, 2, 2, 4, 32, [0, 3, 200, 4], [0, 1, 4, 2], 128, 128, None, 0, BF),
    (1, 16, 1, 7, 16, [1000], None, 128, 64, 333, 40, BF),
    (2, 32, 2, 40, 16, [1000, 41], [40, 33], 64, 64, None, 0, BF),
    (1, 64, 1, 3, 16, [77], None, 32, 32, 16, 1, HF),
    (1, 2, 1, 200, 128, [3000], None, 96, 96, 700, 9, BF),
    (1, 8, 8, 1, 16, [4000], None, 64, 64, None, 0, HF),
    # padded rows beside rows that see whole chunks
    (5, 8, 1, 2, 16, [317, 326, 356, 352, 293], [1, 0, 2, 1, 2], 104, 104, None, 0, BF),
    (6, 32, 8, 185, 96, [54, 217, 627, 366, 183, 569], [48, 149, 73, 127, 143, 44], 112, 16, 582, 0, BF),
    (2, 4, 2, 30, 32, [6000, 5000], [3, 30], 64, 64, None, 4, HF),
    (3, 4, 4, 300, 64, [1500, 900, 300], [20, 300, 0], 128, 128, 700, 2, BF),
]


@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_attention_against_64_bits(case):
    B, H, Hkv, T, page, lens, n_new, dk, dv, window, n_sink, dtype = case
    gen = torch.Generator().manual_seed(3)
    kc, vc, table = pool(gen, B, Hkv, page, lens, dk, dv, dtype)
    q = torch.randn(B, H, T, dk, generator=gen).to(dtype)
    new = n_new or [T] * B
    # what lies behind a sequence's last token, and in pages that are nobody's, does not matter
    used = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for b in range(B):
        for p in range(lens[b]):
            used[table[b, p // page], p % page] = True
    for x in (kc, vc):
        x.transpose(1, 2)[~used] = float("nan")
    scale = 1.0 / math.sqrt(dk)
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    o = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(lens), window, n_sink, scale, None if n_new is None else ints(n_new)).cpu()
    for b in range(B):
        n = new[b]
        want = orc.window(q[b:b + 1, :, :n], gathered(kc, table, b, lens[b])[None], gathered(vc, table, b, lens[b])[None], window, n_sink, scale)["o"]
        orc.check(o[b:b + 1, :, :n], want, f"sequence {b}")
        assert (o[b, :, n:] == 0).all()


APPEND = [
    # B, H, Hkv, T, page, lens, n_new, dk, dv, layout, dtype
    (1, 1, 1, 1, 16, [1], None, 64, 64, "halves", BF),
    (3, 4, 2, 5, 16, [5, 40, 17], [5, 3, 0], 64, 64, "blocks", HF),
    (2, 0, 3, 33, 7, [33, 100], None, 24, 40, "halves", F32),
    (2, 6, 2, 9, 48, [12, 200], [9, 1], 128, 128, None, BF),
    (1, 2, 1, 4, 1, [6], None, 10, 5, "blocks", BF),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c))
def test_append_against_64_bits(case):
    B, H, Hkv, T, page, lens, n_new, dk, dv, layout, dtype = case
    gen = torch.Generator().manual_seed(4)
    kc, vc, table = pool(gen, B, Hkv, page, lens, dk, dv, dtype)
    mk = lambda h, d: torch.randn(B, T, h, d, generator=gen).to(dtype).transpose(1, 2)  # noqa: E731
    k, v, q = mk(Hkv, dk), mk(Hkv, dv), mk(H, dk) if H else None
    tables = [orc.table(64, dk // 2)]
    new = n_new or [T] * B
    pos = torch.tensor([[lens[b] - new[b] + t if t < new[b] else -1 for t in range(T)] for b in range(B)], dtype=torch.int32)[None]
    if layout is None:
        rq, rk = None if q is None else (q.double(), torch.zeros_like(q, dtype=torch.float64)), (k.double(), torch.zeros_like(k, dtype=torch.float64))
    else:
        rq, rk = None if q is None else orc.rotate(q, pos, tables, layout), orc.rotate(k, pos, tables, layout)
    want = [(kc.double(), torch.zeros_like(kc, dtype=torch.float64)), (vc.double(), torch.zeros_like(vc, dtype=torch.float64))]
    for b in range(B):
        for t in range(new[b]):
            p = lens[b] - new[b] + t
            at = (int(table[b, p // page]), slice(None), p % page)
            for i in range(2):
                want[0][i][at] = rk[i][b, :, t]
            want[1][0][at] = v[b, :, t].double()
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    kg, vg = kc.cuda(), vc.cuda()
    rope = None if layout is None else (None, [t.cuda() for t in tables], layout)
    out = paged_append_(kg, vg, k.cuda(), v.cuda(), table.cuda(), ints(lens), None if n_new is None else ints(n_new), rope, None if q is None else q.cuda())
    orc.check(kg.cpu(), want[0], "keys")
    orc.check(vg.cpu(), want[1], "values")
    if q is None:
        assert out is None
    else:
        orc.check(out.cpu(), rq, "queries")
