"""The paged cache in 8 bits where numbers end: scales at both ends of their byte, queries near the type's largest number (GPU)."""
import math

import pytest
import torch

from dl_templates_amd.paged_cache8 import paged8_append_, paged8_attention
from tests import paged8_oracle as orc8
from tests.test_paged_cache8_edges_gpu import check
from tests.test_paged_cache8_gpu import BF, F32, FP8, HF, I8, cache_for, ints, pool

pytestmark = pytest.mark.gpu
bytes_of = lambda x: x.view(torch.uint8)  # noqa: E731


@pytest.mark.parametrize("fmt", [FP8, I8])
def test_ones_at_the_first_and_the_last_scale(fmt):
    one = torch.ones(1, 1, 64, 64).to(fmt).cuda()
    sc = lambda v: torch.full((1, 1, 1), v, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)  # noqa: E731
    for e, n, T in ((0, 1, 1), (0, 9, 1), (0, 64, 40), (254, 1, 1), (254, 1, 40)):   # (two of 2^127 would leave 32 bits)
        q = torch.zeros(1, 2, T, 64, dtype=BF, device="cuda")
        new = ints([min(n, T)])
        o = paged8_attention(q, one, one, sc(127), sc(e), ints([[0]]), ints([n]), n_new=new)[:, :, :min(n, T)]
        assert (o.double() == 2.0 ** (e - 127)).all(), (fmt, e, n, T)


# rows in whole heads, in runs, and more of them; values that differ from key to key by what softmax gives them
LOW = [(2, 4, 2, 1, 32, 16, [700, 90], None, 64, 64, None, 0, BF), (2, 8, 2, 3, 64, 32, [3900, 800], None, 128, 128, None, 0, BF), (1, 8, 2, 30, 64, 64, [900], None, 128, 128, 300, 10, BF)]


@pytest.mark.parametrize("case", LOW, ids=["heads", "runs", "rows"])
@pytest.mark.parametrize("fmt", [FP8, I8])
def test_values_at_the_least_scales(case, fmt):
    """Scales of 2^-127 to 2^-121 on the values: no key's share of a sum is lost, however small its probability."""
    case = case + (fmt,)
    gen = torch.Generator().manual_seed(21)
    kc, vc, ks, vs, table = cache_for(case, gen)
    u = bytes_of(vs)
    u[u != 255] = torch.randint(0, 7, u[u != 255].shape, generator=gen).to(torch.uint8)
    B, H, _, T, _, _, lens, _, dk, _, window, n_sink, dtype, _ = case
    q = torch.randn(B, H, T, dk, generator=gen).to(dtype)
    scale = 1.0 / math.sqrt(dk)
    o = paged8_attention(q.cuda(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda(), ints(lens), window, n_sink, scale).cpu()
    check(case, o, q, (kc, vc, ks, vs, table), [T] * B, scale)


@pytest.mark.parametrize("case", LOW, ids=["heads", "runs", "rows"])
@pytest.mark.parametrize("fmt", [FP8, I8])
def test_keys_at_the_least_scales(case, fmt):
    """The same for keys, under queries so large (2^112 and about) that their scores are ordinary ones."""
    case = case + (fmt,)
    gen = torch.Generator().manual_seed(22)
    kc, vc, ks, vs, table = cache_for(case, gen)
    u = bytes_of(ks)
    u[u != 255] = torch.randint(0, 3, u[u != 255].shape, generator=gen).to(torch.uint8)
    B, H, _, T, _, _, lens, _, dk, _, window, n_sink, dtype, _ = case
    q = (torch.randn(B, H, T, dk, generator=gen).clamp(-3.9, 3.9) * 2.0 ** 112).to(dtype)
    scale = 64.0 / math.sqrt(dk)   # numbers of 100 times 2^-126 times 2^112: 2^-7 a pair of a query's and a key's dims
    o = paged8_attention(q.cuda(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda(), ints(lens), window, n_sink, scale).cpu()
    check(case, o, q, (kc, vc, ks, vs, table), [T] * B, scale)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("old", [0, 1, 26, 250, 253, 254])
def test_tokens_join_a_block_of_any_scale(old, fmt, dtype):
    """Blocks of 32 tokens, 20 of them there at a scale that an append does not give: new ones are rounded to it, or it grows and the older ones are rounded anew."""
    gen = torch.Generator().manual_seed(23)
    kc, vc, ks, vs, table = pool(gen, 2, 2, 64, 32, [64, 64], 64, 72, fmt)
    for s in (ks, vs):
        bytes_of(s).fill_(old)
    lens, T = [20 + 9, 52 + 12], 12
    new = [9, 12]
    top = 1e38 if dtype != HF else 2e4
    mk = lambda d: (torch.randn(2, 2, T, d, generator=gen).clamp(-3, 3) * top).to(dtype)  # noqa: E731
    k, v = mk(64), mk(72)
    zero = lambda x: torch.zeros_like(x, dtype=torch.float64)  # noqa: E731
    want = [orc8.append(c, s, x.double(), zero(x), table, lens, new, dtype) for c, s, x in ((kc, ks, k), (vc, vs, v))]
    got = [x.cuda() for x in (kc, vc, ks, vs)]
    paged8_append_(*got, k.cuda(), v.cuda(), table.cuda(), ints(lens), ints(new))
    for i, (c, e, _, near) in enumerate(want):
        assert torch.equal(bytes_of(got[2 + i].cpu()).int(), e)
        assert torch.equal(got[i].cpu().float().double(), c)


@pytest.mark.parametrize("case", LOW, ids=["heads", "runs", "rows"])
@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_queries_near_the_largest_number(case, fmt, sign):
    """Queries of 2^122 over keys of 2^-121: products without the keys' scales would leave 32 bits.  Scores are about -3 or 3, all of one sign, unequal from key to key."""
    case = case + (fmt,)
    gen = torch.Generator().manual_seed(24)
    kc, vc, ks, vs, table = cache_for(case, gen)
    kc.copy_((kc.float().abs().nan_to_num(1.0) % 64 + 64).to(fmt))
    u = bytes_of(ks)
    u[u != 255] = 0
    B, H, _, T, _, _, lens, _, dk, _, window, n_sink, dtype, _ = case
    q = torch.randn(B, H, T, dk, generator=gen).abs().clamp(0.1, 3.9)
    q[:, ::2] *= 2.0 ** -14   # beside rows that need nothing of the kind
    q = (q * (sign * 2.0 ** 122)).to(dtype)
    scale = 2.0 / dk   # 96 2^-127 2^122 0.8 dk times that: 4.8; rows of even heads: none to speak of
    o = paged8_attention(q.cuda(), *(x.cuda() for x in (kc, vc, ks, vs)), table.cuda(), ints(lens), window, n_sink, scale).cpu()
    check(case, o, q, (kc, vc, ks, vs, table), [T] * B, scale)
