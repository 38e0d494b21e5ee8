"""Window attention with sinks against its 64-bit form (GPU)."""
import math

import pytest
import torch

from dl_templates_amd.window_attn import window_attention
from tests import long_oracle as orc

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(seed, B, Hq, Hkv, Lq, Lk, dk, dv, dtype):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=gen).to(dtype).cuda()  # noqa: E731
    return mk(B, Hq, Lq, dk), mk(B, Hkv, Lk, dk), mk(B, Hkv, Lk, dv), mk(B, Hq, Lq, dv)


def run(q, k, v, do, window, n_sink, scale):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    o = window_attention(q, k, v, window, n_sink, scale)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, (q, k, v), do)))


CASES = [
    # B, Hq, Hkv, Lq, Lk, dk, dv, window, sinks, dtype
    (1, 1, 1, 1, 1, 64, 64, 1, 0, BF),
    (1, 2, 2, 64, 64, 64, 64, None, 0, BF),
    (2, 4, 2, 200, 200, 64, 64, 64, 4, HF),
    (1, 8, 1, 130, 130, 128, 128, 17, 1, BF),
    (1, 6, 2, 257, 301, 80, 80, 100, 5, HF),
    (1, 3, 1, 77, 500, 128, 128, 60, 33, BF),
    (2, 5, 5, 65, 65, 32, 64, 1, 0, BF),
    (1, 4, 4, 90, 40, 64, 64, 16, 2, HF),          # more queries than keys: the first ones see nothing
    (1, 2, 1, 1, 700, 128, 128, None, 0, BF),
    (1, 2, 1, 5, 700, 64, 64, 300, 70, HF),
    (1, 7, 1, 333, 333, 96, 40, 1000, 3, BF),
    (1, 1, 1, 513, 513, 128, 128, 128, 64, HF),
    (1, 1, 1, 513, 513, 128, 128, 129, 65, BF),
    (1, 32, 1, 40, 90, 64, 128, 31, 7, BF),
    (3, 2, 2, 127, 129, 8, 16, 2, 1, BF),
    (1, 2, 2, 700, 700, 64, 64, 64, 600, BF),      # sinks beyond the window's own reach
    (1, 1, 1, 2000, 2000, 64, 64, 500, 4, HF),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_against_64_bits(case):
    B, Hq, Hkv, Lq, Lk, dk, dv, window, n_sink, dtype = case
    q, k, v, do = make(1, B, Hq, Hkv, Lq, Lk, dk, dv, dtype)
    scale = 1.0 / math.sqrt(dk)
    got = run(q, k, v, do, window, n_sink, scale)
    for name, want in orc.window(q, k, v, window, n_sink, scale, do).items():
        orc.check(got[name], want, name)


FAR = [
    (1, 4, 1, 3000, 3000, 64, 64, 33, 4, BF),
    (1, 2, 2, 2500, 2600, 128, 128, 64, 17, HF),      # two groups of sinks, the second one partly filled
    (2, 3, 1, 1500, 1500, 80, 72, 100, 70, BF),       # sinks over two blocks of keys
    (1, 8, 8, 1111, 1111, 128, 128, 1, 1, BF),
    (1, 1, 1, 4000, 4000, 64, 64, 17, 128, HF),
]


@pytest.mark.parametrize("case", FAR, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rows_far_behind_the_sinks(case):
    """Gradients of first keys that the rows of the whole sequence see."""
    test_against_64_bits(case)


SHARED = [
    (1, 4, 2, 20, 3000, 64, 64, None, 4, BF),
    (1, 2, 1, 10, 5000, 128, 128, None, 0, HF),
    (2, 2, 2, 100, 2100, 80, 72, 2000, 9, BF),
    (1, 3, 1, 130, 4000, 128, 40, 3000, 70, HF),
    (1, 1, 1, 1, 9000, 64, 64, None, 0, BF),
]


@pytest.mark.parametrize("case", SHARED, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_few_queries_on_many_keys(case):
    """Keys shared by workgroups, in the forward pass and for dq."""
    test_against_64_bits(case)


@pytest.mark.parametrize("Hq, Hkv, L, dk, dtype", [(2, 2, 70, 64, BF), (6, 2, 300, 128, HF), (4, 1, 1000, 96, BF)])
def test_a_single_key_has_no_gradient_of_scores(Hq, Hkv, L, dk, dtype):
    """The softmax of one score is 1 whatever the score is: dq and dk are zero, not the rest of a cancellation."""
    q, k, v, do = make(2, 1, Hq, Hkv, L, L, dk, dk, dtype)
    got = run(q, k, v, do, 1, 0, 0.3)
    assert torch.equal(got["o"], v.repeat_interleave(Hq // Hkv, 1)) and not got["dq"].any() and not got["dk"].any() and got["dv"].any()
    got = run(q[:, :, :1], k[:, :, :1], v[:, :, :1], do[:, :, :1], None, 3, 0.3)
    assert not got["dq"].any() and not got["dk"].any()
    got = run(q, k, v, do, None, 0, 0.3)
    assert not got["dq"][:, :, 0].any() and got["dq"][:, :, 1].any()   # the query at position 0 sees one key


@pytest.mark.parametrize("window, n_sink, dtype", [(2, 0, BF), (2, 0, HF), (3, 1, HF), (1, 2, BF), (8, 0, BF), (500, 0, HF)])
def test_gradients_of_few_keys(window, n_sink, dtype):
    """Where a row sees few keys, dP and delta nearly cancel, and delta must not suffer from the rounding of o.  The errors of dq and dk, as norms, against those that
    their own rounding makes (1): the rounding of dS makes as much, sqrt(2) together, and P, from sums of rounded exponentials, a third of it: sqrt(2 + 1 / 9) < 1.46, with two keys,
    whose dS are opposite, up to 1.6.  With delta from the rounded o two keys gave 2.3, eight 1.6."""
    q, k, v, do = make(3, 1, 4, 4, 400, 400, 64, 64, dtype)
    got, want = run(q, k, v, do, window, n_sink, 0.125), orc.window(q, k, v, window, n_sink, 0.125, do)
    for name in ("dq", "dk"):
        value = want[name][0]
        own = (value.to(dtype).double() - value).norm()
        assert (got[name].double() - value).norm() <= 1.7 * own, name
