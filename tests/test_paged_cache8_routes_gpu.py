"""The paged cache in 8 bits on the routes that real prompts and batches take, against 64 bits: appends whose waves walk several heads, attention of 128 rows a workgroup with
the keys shared, of 17 to 32 rows in whole heads and in runs (GPU).  Every case says which route it is for and asks for it, as the host chooses on 256 CUs."""
import ctypes
import math

import pytest
import torch

from dl_templates_amd import _lib
from dl_templates_amd.paged_cache8 import paged8_append_, paged8_attention
from tests import long_oracle as orc
from tests import paged8_oracle as orc8
from tests.test_paged_cache8_gpu import BF, F32, FP8, HF, I8, cache_for, gathered, ints, name, pool

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def chip():
    if torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("the cases are sized for 256 CUs")


def append_route(B, H, Hkv, T, block, dk, dv):
    """(waves of an item, rounds of their rows, heads that an item walks, heads of q that a wave walks)"""
    rows, most = 64 // (max(dk, dv) // 8), min(T, block)
    nw = 1 if most <= 2 * rows else 4 if most <= 8 * rows else 8
    blocks, hk, hq = B * ((T + block - 2) // block + 1), Hkv, max(H, 1)
    while hk > 1 and blocks * nw * 2 * -(-Hkv // hk) < 8 * 256:
        hk = (hk + 1) // 2
    groups = -(-B * T // (64 // (dk // 8)))
    while hq > 1 and groups * -(-H // hq) < 16 * 256:
        hq = (hq + 1) // 2
    return nw, -(-most // (nw * rows)), hk, hq


# B, H, Hkv, T, page, block, lens, n_new, dk, dv, layout, sections, dtype, (waves, rounds, heads of an item, heads of q)
APPEND = [
    (4, 32, 8, 1000, 64, 16, [1000, 1203, 1001, 1030], None, 64, 64, "halves", "one", HF, (1, 2, 2, 2)),
    (3, 24, 7, 1500, 32, 16, [1510, 1499, 1700], [1500, 1499, 1203], 40, 64, "blocks", "several", BF, (1, 2, 2, 2)),
    (4, 32, 8, 700, 64, 16, [700, 913, 701, 730], None, 128, 128, "halves", "one", BF, (4, 1, 4, 4)),
    (3, 8, 7, 1000, 64, 32, [1000, 1040, 1003], [900, 1000, 3], 128, 128, "blocks", "one", BF, (4, 2, 2, 1)),
    (2, 64, 9, 1000, 64, 32, [1000, 1037], None, 128, 96, "halves", "several", HF, (4, 2, 2, 4)),
    (4, 32, 8, 1500, 64, 64, [1500, 1600, 1517, 1501], None, 128, 128, "halves", "one", BF, (8, 2, 4, 8)),
    (2, 6, 7, 900, 128, 64, [913, 950], [900, 750], 104, 128, "blocks", "several", F32, (8, 2, 2, 1)),
    (3, 16, 14, 800, 128, 128, [890, 800, 1000], None, 128, 128, None, "one", BF, (8, 4, 2, 2)),
    # small ones of the same kernels: an item a head
    (2, 2, 2, 20, 32, 32, [20, 45], None, 128, 128, "halves", "one", BF, (4, 2, 1, 1)),
    (2, 2, 3, 40, 64, 64, [40, 90], [40, 33], 128, 128, "blocks", "one", F32, (8, 2, 1, 1)),
]


def scales_are_certain(y, mag, lens, new, block, fmt):
    """No block's largest element is so near a border of two scales that its rotation in 32 bits (off by 3 2^-24 mag at most, element by element) could cross it."""
    slack = 3 * 2.0 ** -24 * mag
    for b in range(len(lens)):
        held = lens[b] - new[b]
        for base in range(held // block * block, lens[b], block):
            n0, n1 = max(held, base) - held, min(lens[b], base + block) - held
            for h in range(y.shape[1]):
                x, z = y[b, h, n0:n1].abs(), slack[b, h, n0:n1]
                if orc8.exponent(float((x + z).max()), fmt) != orc8.exponent(float((x - z).max()), fmt):
                    return False
    return True


@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: name(c[:6] + c[8:]))
def test_append(case, fmt):
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, layout, sections, dtype, route = case
    assert append_route(B, H, Hkv, T, block, dk, dv) == route
    gen = torch.Generator().manual_seed(14)
    kc, vc, ks, vs, table = pool(gen, B, Hkv, page, block, lens, dk, dv, fmt)
    mk = lambda h, d: torch.randn(B, T, h, d, generator=gen).to(dtype).transpose(1, 2)  # noqa: E731
    k, v, q = mk(Hkv, dk), mk(Hkv, dv), mk(H, dk)
    grow = torch.exp2(torch.randint(-3, 6, (B, Hkv, -(-T // 7)), generator=gen).float()).repeat_interleave(7, 2)[:, :, :T, None]   # scales of neighbouring blocks and heads differ
    k, v = k * grow.to(dtype), v * grow.to(dtype)
    new = n_new or [T] * B
    r = dk // 2
    tables = [orc.table(2000, r)] if sections == "one" else [orc.table(2000, r // 4 + 1), orc.table(300, 0), orc.table(1800, r // 3)]
    pos = torch.tensor([[lens[b] - new[b] + t if t < new[b] else -1 for t in range(T)] for b in range(B)], dtype=torch.int32)[None].repeat(len(tables), 1, 1)
    zero = lambda x: torch.zeros_like(x, dtype=torch.float64)  # noqa: E731
    if layout is None:
        rq, rk, mag = (q.double(), zero(q)), k.double(), zero(k)
    else:
        rq, rk = orc.rotate(q, pos, tables, layout), orc.rotate(k, pos, tables, layout)[0]
        turned = torch.zeros(dk, dtype=torch.bool)   # the other dims are what they were, bit for bit
        for d0, d1, _, _ in orc.pairs_of([t.shape[1] for t in tables], layout):
            turned[d0] = turned[d1] = True
        mag = torch.where(turned, k.double().abs().amax(-1, keepdim=True) * 2, 0.0).expand_as(k)
    assert scales_are_certain(rk, mag, lens, new, block, fmt)
    want = [orc8.append(kc, ks, rk, mag, table, lens, new, dtype), orc8.append(vc, vs, v.double(), zero(v), table, lens, new, dtype)]
    got = [x.cuda() for x in (kc, vc, ks, vs)]
    rope = None if layout is None else (None, [t.cuda() for t in tables], layout)
    out = paged8_append_(*got, k.cuda(), v.cuda(), table.cuda(), ints(lens), None if n_new is None else ints(n_new), rope, q.cuda())
    for i, (c, e, tol, _) in enumerate(want):
        assert torch.equal(got[2 + i].cpu().view(torch.uint8).int(), e), "keys values".split()[i]
        off = (got[i].cpu().to(torch.float32).double() - c).abs()
        assert (off <= tol).all(), f"{'keys values'.split()[i]}: {int((off > tol).sum())} numbers"
    orc.check(out.cpu(), rq, "queries")


def parts_of(case):
    """Copies of all rows' sums that the call's workspace holds: shares of the keys; -1: of runs (their own number each)."""
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, fmt = case
    i64 = lambda *x: (ctypes.c_int64 * len(x))(*x)  # noqa: E731
    shape = _lib.PagedShape(B=B, H=H, Hkv=Hkv, T=T, dk=dk, dv=dv, page=page, n_pages=B * 999, cols=-(-max(lens) // page), window=window or 2 ** 31 - 1, n_sink=n_sink, sm_scale=0.1,
                            dtype=0 if dtype == BF else 1)
    n = ctypes.c_int64()
    _lib.check(_lib.load().dlt_paged8_workspace(shape, _lib.Scales8(0, block, 256, 256, i64(1, 1, 1), i64(1, 1, 1)), ctypes.byref(n)))
    rows = H // Hkv * T
    return (-1 if n.value else 0) if rows <= 32 else n.value // (4 * B * H * T * (dv + 2))


# B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, sinks, dtype; shares
ATTN = [
    # 128 rows a workgroup, keys shared: (512 / (8 heads x blocks)) shares, where blocks of 64 rows would have half as many
    ((1, 32, 8, 120, 64, 32, [8200], None, 128, 128, None, 0, BF), 16),
    ((1, 32, 8, 256, 64, 64, [8200], [201], 128, 128, None, 0, BF), 8),
    ((1, 32, 8, 250, 48, 48, [8111], None, 64, 64, None, 0, HF), 8),
    ((2, 32, 8, 128, 32, 16, [7000, 5003], [128, 77], 96, 80, None, 0, HF), 8),
    ((1, 32, 8, 256, 64, 64, [9000], None, 64, 64, 6000, 9, BF), 8),
    ((1, 32, 8, 200, 128, 128, [8000], None, 104, 128, 7000, 70, BF), 9),
    # the same, not shared
    ((4, 32, 8, 300, 64, 64, [700, 320, 300, 513], None, 128, 128, None, 0, BF), 0),
    ((4, 32, 8, 300, 64, 32, [700, 320, 300, 513], [300, 20, 0, 299], 64, 64, 200, 3, HF), 0),
    # 17 to 32 rows: in runs, and in whole heads
    ((3, 8, 1, 3, 64, 64, [9000, 40, 2700], None, 128, 128, None, 0, BF), -1),
    ((3, 8, 1, 4, 32, 16, [2603, 3, 7001], [4, 2, 3], 64, 64, None, 0, HF), -1),
    ((2, 20, 4, 6, 48, 48, [5000, 6001], None, 80, 128, 4000, 20, BF), -1),
    ((3, 8, 1, 3, 64, 64, [900, 40, 1100], None, 128, 128, None, 0, BF), 0),
    ((3, 8, 1, 4, 32, 16, [603, 3, 1001], [4, 2, 3], 64, 64, None, 0, HF), 0),
    ((2, 20, 4, 6, 48, 48, [5000, 6001], None, 64, 40, 700, 20, BF), 0),
]


@pytest.mark.parametrize("spoilt", ["nothing", "keys", "values"])
@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("case, parts", ATTN, ids=lambda c: name(c) if isinstance(c, tuple) else None)
def test_attention(case, parts, fmt, spoilt):
    """Rows that see a NaN (a token's in e4m3, a block's scale in int8) are NaN; all others, beside them and in other heads, are what they are without it."""
    case = case + (fmt,)
    B, H, Hkv, T, page, block, lens, n_new, dk, dv, window, n_sink, dtype, _ = case
    assert parts_of(case) == parts
    gen = torch.Generator().manual_seed(15)
    kc, vc, ks, vs, table = cache_for(case, gen)
    q = torch.randn(B, H, T, dk, generator=gen).to(dtype).cuda()
    new, scale, G = n_new or [T] * B, 0.3 / math.sqrt(dk), H // Hkv
    lo = hi = -1
    dev = [x.cuda() for x in (kc, vc, ks, vs)]
    if spoilt != "nothing":
        i = ["keys", "values"].index(spoilt)
        j = lens[0] - new[0] // 2 - 1
        p, r = int(table[0, j // page]), j % page
        if fmt == FP8:
            dev[i].view(torch.uint8)[p, 0, r] = 0x7f
            lo, hi = j, j + 1
        else:
            dev[2 + i].view(torch.uint8)[p, 0, r // block] = 255
            lo, hi = j // block * block, min(j // block * block + block, lens[0])
    o = paged8_attention(q, *dev, table.cuda(), ints(lens), window, n_sink, scale, None if n_new is None else ints(n_new))
    again = paged8_attention(q, *dev, table.cuda(), ints(lens), window, n_sink, scale, None if n_new is None else ints(n_new))
    assert torch.equal(o.view(torch.int16), again.view(torch.int16))
    for b in range(B):
        n = new[b]
        assert (o[b, :, n:] == 0).all()
        for h in range(Hkv):
            k, v = (gathered(c[:, h:h + 1], s[:, h:h + 1], table, b, lens[b], dtype)[None].cuda() for c, s in ((kc, ks), (vc, vs)))
            got, rows = o[b:b + 1, h * G:(h + 1) * G, :n], q[b:b + 1, h * G:(h + 1) * G, :n]
            value, bound = orc.window(rows, k, v, window, n_sink, scale)["o"]
            if b == 0 and h == 0 and hi > lo:
                pos = torch.arange(lens[0] - n, lens[0], device="cuda")
                sees = orc.seen(pos, lens[0], window, n_sink)[:, lo:hi].any(-1)
                assert torch.isnan(got[:, :, sees]).all()
                got, value, bound = (x[:, :, ~sees] for x in (got, value, bound))
            orc.check(got, (value, bound), f"sequence {b}, head {h}")


@pytest.mark.parametrize("case", [(2, 4, 2, 1, 32, 16, [700, 90], None, 64, 64, None, 0, HF), (1, 8, 2, 3, 64, 32, [3900], None, 128, 128, None, 0, HF), (1, 8, 2, 30, 64, 64, [900], None, 128, 128, None, 0, HF)],
                         ids=["heads", "runs", "rows"])
@pytest.mark.parametrize("fmt", [FP8, I8])
def test_numbers_below_the_normal_ones_of_float16(case, fmt):
    """fp16 queries read keys and values as numbers of fp16 or better: where those have a step of 2^-24, each is off by half of it at most."""
    case = case + (fmt,)
    B, H, _, T, _, _, lens, _, dk, _, window, n_sink, dtype, _ = case
    for which in ("keys", "values"):
        gen = torch.Generator().manual_seed(16)
        kc, vc, ks, vs, table = cache_for(case, gen)
        u = (ks if which == "keys" else vs).view(torch.uint8)
        u[u != 255] = torch.randint(99, 110, u[u != 255].shape, generator=gen).to(torch.uint8)   # numbers of about 100: 2^-21 to 2^-11
        q = (torch.randn(B, H, T, dk, generator=gen) * (256 if which == "keys" else 1)).to(dtype)
        scale = 0.3 / math.sqrt(dk)
        o = paged8_attention(q.cuda(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda(), ints(lens), window, n_sink, scale).cpu()
        for b in range(B):
            k, v = (gathered(c, s, table, b, lens[b], torch.float64)[None] for c, s in ((kc, ks), (vc, vs)))
            qb = q[b:b + 1]
            wide = lambda x: x.repeat_interleave(H // 2, 1)  # noqa: E731
            p = orc.probabilities(qb.double(), wide(k), orc.seen(torch.arange(lens[b] - T, lens[b]), lens[b], window, n_sink), scale)
            value, mag = p @ wide(v), p @ wide(v).abs()
            half = torch.finfo(dtype).eps / 2
            bound = half * (mag + 2 * value.abs()) + orc.SLACK * mag
            if which == "keys":
                # a score is off by the half step times the sum of its query's magnitudes; a probability by twice that of itself, the numbers here being small (below 2^-8)
                off = scale * 2.0 ** -25 * qb.double().abs().sum(-1, keepdim=True)
                assert off.max() < 2.0 ** -8
                bound = bound + 2 * off * (1 + 2.0 ** -7) * (mag + value.abs())
            else:
                bound = bound + 2.0 ** -25
            orc.check(o[b:b + 1], (value, bound), f"{which}, sequence {b}")
