"""Edges of the long-sequence operators that a plan, a padded batch or an unusual caller reaches (GPU)."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad
from torch.utils._python_dispatch import TorchDispatchMode

from dl_templates_amd import _lib
from dl_templates_amd._lib import DltError
from dl_templates_amd.paged_cache import paged_append_, paged_attention
from dl_templates_amd.rope_axes import rope_axes_qk, rope_axes_qk_
from dl_templates_amd.window_attn import window_attention
from tests import long_oracle as orc
from tests.test_paged_cache_gpu import gathered, pool

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")
name_of = lambda c: "-".join(str(x).replace("torch.", "").replace(" ", "") for x in c)  # noqa: E731


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- padded batches ------------------------------------------------------------------------------------------------------------------
# workgroups of 16 rows, of 64 with the keys over two groups of waves, of 64, of 128, and keys shared by workgroups
PADDED = [
    # B, H, Hkv, T, lens, n_new, D, window, sinks, dtype
    (3, 4, 2, 6, (100, 37, 64), (2, 6, 0), 64, None, 0, BF),
    (3, 4, 2, 6, (100, 37, 64), (3, 5, 1), 64, 20, 2, HF),
    (3, 16, 4, 150, (400, 260, 300), (18, 150, 90), 64, None, 0, BF),
    (4, 32, 8, 150, (400, 260, 300, 150), (18, 150, 90, 1), 64, 100, 3, HF),
    (8, 64, 16, 150, (400, 260, 300, 150, 200, 201, 202, 203), (20, 150, 90, 1, 2, 3, 4, 5), 128, 100, 3, BF),
    (1, 2, 1, 30, (3000,), (3,), 64, None, 0, BF),
]


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("where", ["a value that is seen", "a hidden value", "a key that is seen", "a hidden key", "the first value", "the first key"])
@pytest.mark.parametrize("case", PADDED, ids=name_of)
def test_padded_rows_are_zeros_beside_special_values(case, where, bad):
    """Padded rows have no keys: an infinity or a NaN among those of the sequence does not reach them, nor the rows that do not see it."""
    B, H, Hkv, T, lens, new, D, window, n_sink, dtype = case
    kc, vc, table = (x.cuda() for x in pool(torch.Generator().manual_seed(50), B, Hkv, 16, lens, D, D, dtype))
    q = torch.randn(B, H, T, D, generator=torch.Generator().manual_seed(51)).to(dtype).cuda()
    scale, G, n, first = 1.0 / math.sqrt(D), H // Hkv, lens[0], lens[0] - new[0]
    # seen by every new token of sequence 0; hidden: just outside of the first one's window, or ahead of all but the last one
    j = first if "seen" in where else 0 if "first" in where else first - window if window is not None else n - 1
    vis = orc.seen(torch.arange(new[0], device="cuda") + first, n, window, n_sink)[:, j]
    assert vis.all() if "seen" in where else "first" in where or not vis[0]
    keys, values = (gathered(c, table, 0, n)[None] for c in (kc, vc))
    (vc if "value" in where else kc)[int(table[0, j // 16]), 0, j % 16] = bad
    o = paged_attention(q, kc, vc, table, ints(*lens), window, n_sink, scale, ints(*new))
    for b in range(B):
        assert (o[b, :, new[b]:] == 0).all()
        assert b == 0 or o[b].isfinite().all()
    value, bound = orc.window(q[:1, :, :new[0]], keys, values, window, n_sink, scale)["o"]
    clean = torch.ones(1, H, new[0], dtype=torch.bool, device="cuda")
    clean[0, :G] = ~vis
    got = o[:1, :, :new[0]]
    orc.check(got[clean], (value[clean], bound[clean]), "rows that do not see it")
    if bad != bad:
        assert got[~clean].isnan().all()


# ---- shares of keys --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("low", [-400.0, -INF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H, Hkv, Lq, Lk", [(2, 1, 1, 300), (8, 8, 64, 500), (2, 1, 1, 1600), (4, 2, 3, 3008), (4, 1, 20, 8000), (64, 64, 400, 800)])
def test_a_nan_of_no_weight_is_not_lost(H, Hkv, Lq, Lk, dtype, low):
    """The first half of the keys has scores so low that their weights are 0, and one value there is NaN: 0 times NaN is NaN in the formula, however the keys are shared."""
    gen = torch.Generator().manual_seed(52)
    q = torch.rand(1, H, Lq, 64, generator=gen).add(0.1).to(dtype).cuda()
    k, v = (torch.randn(1, Hkv, Lk, 64, generator=gen).to(dtype).cuda() for _ in range(2))
    k[:, :, :Lk // 2] = low
    v[:, :, 5, 3] = NAN
    value, bound = orc.window(q, k, v, None, 0, 0.125)["o"]
    assert value[..., 3].isnan().all() and value[..., :3].isfinite().all()
    outs = {"dense": window_attention(q, k, v, None, 0, 0.125)}
    if Lk % 16 == 0:
        pages = lambda x: x[0].reshape(Hkv, Lk // 16, 16, 64).transpose(0, 1).contiguous()  # noqa: E731
        outs["paged"] = paged_attention(q, pages(k), pages(v), torch.arange(Lk // 16, dtype=torch.int32, device="cuda")[None], ints(Lk), None, 0, 0.125)
    for name, o in outs.items():
        assert o[..., 3].isnan().all(), f"{name}: the NaN is lost"
        keep = [d for d in range(64) if d != 3]
        orc.check(o[..., keep], (value[..., keep], bound[..., keep]), name)


# ---- rows taken again --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
def test_low_parts_of_rows_taken_again(dtype):
    """Rows that meet a hidden NaN are formed once more; o and its low part together are then the value in 32 bits: the low part's own rounding is u^2 |o|, 8 terms and
    scores of 64 products of a sum of magnitudes below 12 are off by 2 (8 + 64 12) 2^-24 < 2^-13 of the terms' magnitude."""
    gen = torch.Generator().manual_seed(53)
    q, k, v = (torch.randn(1, h, 64, 64, generator=gen).to(dtype).cuda() for h in (4, 2, 2))
    value, _ = orc.window(q, k, v, 8, 0, 0.125)["o"]
    mag, _ = orc.window(q, k, v.abs(), 8, 0, 0.125)["o"]
    scores = (q.double().abs() @ k.double().abs().repeat_interleave(2, 1).transpose(-1, -2) * 0.125).amax()
    assert scores < 12
    v[:, :, 20, :32] = NAN   # hidden from tokens 16 to 19, which meet it in their chunk
    o, _, low = _lib.native.window_forward(q, k, v, 8, 0, 0.125)
    at = (slice(None), slice(None), slice(16, 20))
    u = torch.finfo(dtype).eps / 2
    orc.check(o[at], (value[at], u * value[at].abs() + 2.0 ** -13 * mag[at]), "o")
    off = (o[at].double() + low[at].double() - value[at]).abs()
    assert (off <= u * u * value[at].abs() + 2.0 ** -13 * mag[at] + orc.tiny(dtype)).all()


@pytest.mark.parametrize("window, n_sink, dtype", [(2, 0, BF), (2, 0, HF), (3, 1, HF), (8, 0, BF)])
def test_query_gradients_of_rows_taken_again(window, n_sink, dtype):
    """Every 64th key is NaN, and no row but those that see it may tell: the error of dq, as a norm, against that of its own rounding, as for rows that meet none (1.46, up to
    1.6 with two keys; delta from the rounded o alone gives 2.3 with two keys)."""
    gen = torch.Generator().manual_seed(54)
    q, k, v, do = (torch.randn(1, 4, 512, 64, generator=gen).to(dtype).cuda() for _ in range(4))
    value = orc.window(q, k, v, window, n_sink, 0.125, do)["dq"][0]
    k[:, :, 32::64] = NAN
    q.requires_grad_(True)
    dq = torch.autograd.grad(window_attention(q, k, v, window, n_sink, 0.125), q, do)[0]
    t = torch.arange(512, device="cuda") % 64
    clean = (t < 32) | (t >= 32 + window)
    got, want = dq[:, :, clean].double(), value[:, :, clean]
    assert dq[:, :, ~clean].isnan().all() and got.isfinite().all()
    assert (got - want).norm() <= 1.7 * (want.to(dtype).double() - want).norm()


# ---- traces, modes and tangents -------------------------------------------------------------------------------------------------------
def small_cache(seed=55, dtype=BF):
    gen = torch.Generator().manual_seed(seed)
    kc, vc = (torch.randn(6, 2, 16, 64, generator=gen).to(dtype).cuda() for _ in range(2))
    q, k, v = (torch.randn(2, h, 3, 64, generator=gen).to(dtype).cuda() for h in (4, 2, 2))
    return kc, vc, q, k, v, torch.arange(6, dtype=torch.int32, device="cuda").reshape(2, 3), ints(40, 20 + seed % 7)


def test_traced_paged_calls_depend_on_their_inputs():
    tables = [orc.table(64, 32).cuda()]

    def step(kc, vc, q, k, v, pages, seq):
        r = paged_append_(kc, vc, k, v, pages, seq, None, (None, tables, "halves"), q)
        return paged_attention(r, kc, vc, pages, seq, 20, 2)

    def fill(kc, vc, q, k, v, pages, seq):
        before = kc + 0
        assert paged_append_(kc, vc, k, v, pages, seq) is None
        return paged_attention(q, kc, vc, pages, seq), before, kc + 0

    def attend(kc, vc, q, k, v, pages, seq):
        return paged_attention(q, kc, vc, pages, seq, 20, 2, None, seq - 18)
    for f in (step, fill, attend):
        traced = torch.jit.trace(f, small_cache(55), check_trace=False)
        for seed in (56, 57, 58, 59):   # the executor rearranges a graph after its first runs
            a, b = small_cache(seed), small_cache(seed)
            got, want = traced(*a), f(*b)
            got, want = (x if isinstance(x, tuple) else (x,) for x in (got, want))
            assert all(torch.equal(x, y) for x, y in zip(got + a, want + b))


def test_a_traced_rotation_in_place_depends_on_its_inputs():
    tables = [orc.table(64, 32).cuda()]

    def turn(q, k, pos):
        before = q + k
        q, k = rope_axes_qk_(q, k, pos, tables)
        return before, q + k

    def one(q, k, pos):
        return rope_axes_qk_(q, None, pos, tables)[0] * k
    mk = lambda s: tuple(torch.randn(1, 2, 40, 64, generator=torch.Generator().manual_seed(s + i)).cuda() for i in range(2)) + (torch.arange(s, s + 40, dtype=torch.int32, device="cuda")[None],)  # noqa: E731
    for f in (turn, one):
        traced = torch.jit.trace(f, mk(1), check_trace=False)
        for seed in (5, 7, 9, 11):
            a, b = mk(seed), mk(seed)
            got, want = traced(*a), f(*b)
            got, want = (x if isinstance(x, tuple) else (x,) for x in (got, want))
            assert all(torch.equal(x, y) for x, y in zip(got + a, want + b))


def test_tangents_are_refused():
    """No derivative in forward mode: a tangent on any tensor raises before anything is written, as for the operators beside these."""
    kc, vc, q, k, v, pages, seq = small_cache()
    pos, tables = torch.arange(3, dtype=torch.int32, device="cuda")[None], [orc.table(64, 32).cuda()]
    start = [x.clone() for x in (kc, vc, q, k)]
    dual = lambda x: fwd_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
    with fwd_ad.dual_level():
        for call in (lambda: rope_axes_qk_(dual(q), None, pos, tables), lambda: rope_axes_qk_(q, dual(k), pos, tables), lambda: rope_axes_qk_(q, k, pos, [dual(tables[0])]),
                     lambda: paged_attention(dual(q), kc, vc, pages, seq), lambda: paged_attention(q, dual(kc), vc, pages, seq), lambda: paged_attention(q, kc, dual(vc), pages, seq),
                     lambda: paged_append_(kc, vc, dual(k), v, pages, seq), lambda: paged_append_(kc, vc, k, dual(v), pages, seq), lambda: paged_append_(dual(kc), vc, k, v, pages, seq),
                     lambda: paged_append_(kc, dual(vc), k, v, pages, seq), lambda: paged_append_(kc, vc, k, v, pages, seq, None, (None, tables, "halves"), dual(q)),
                     lambda: paged_append_(kc, vc, k, v, pages, seq, None, (None, [dual(tables[0])], "halves"), q)):
            with pytest.raises(NotImplementedError):
                call()
    assert all(torch.equal(x, y) for x, y in zip((kc, vc, q, k), start))


def test_transforms_are_refused():
    kc, vc, q, k, v, pages, seq = small_cache()
    pos, tables = torch.arange(3, dtype=torch.int32, device="cuda")[None], [orc.table(64, 32).cuda()]
    many = lambda x: torch.stack([x, x])  # noqa: E731
    for f, x in ((lambda q: paged_attention(q, kc, vc, pages, seq), many(q)), (lambda k: paged_append_(kc, vc, k, v, pages, seq, q=q), many(k)),
                 (lambda q: rope_axes_qk_(q, None, pos, tables)[0], many(q))):
        with pytest.raises(RuntimeError, match="setup_context"):
            torch.func.vmap(f)(x)


def test_paged_calls_and_rotation_in_place_under_a_mode():
    """A dispatch mode takes the classes: the same bits, no graph, and written tensors that count as written."""
    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    pos, tables = torch.arange(3, dtype=torch.int32, device="cuda")[None], [orc.table(64, 32).cuda()]

    def work():
        kc, vc, q, k, v, pages, seq = small_cache()
        count = [x._version for x in (kc, vc, q)]
        q.requires_grad_(True)
        r = paged_append_(kc, vc, k, v, pages, seq, None, (None, tables, "halves"), q)
        o = paged_attention(r, kc, vc, pages, seq)
        assert paged_append_(kc, vc, k, v, pages, seq) is None
        with torch.no_grad():
            turned = rope_axes_qk_(q, k, pos, tables)
        assert turned[0] is q and turned[1] is k and not o.requires_grad and not r.requires_grad
        assert all(x._version > n for x, n in zip((kc, vc, q), count))
        with pytest.raises(RuntimeError, match="leaf Variable"):
            paged_append_(kc.clone().requires_grad_(True), vc, k, v, pages, seq)
        return kc, vc, r, o, q.detach(), k
    want = work()
    with Seen():
        got = work()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---- empty batches ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 40])
def test_window_attention_of_no_sequence(D):
    """As paged attention has it: empty outputs and gradients; what is wrong with the other arguments is still refused."""
    q, k, v = (torch.zeros(0, h, n, D, dtype=BF, device="cuda", requires_grad=True) for h, n in ((4, 5), (2, 9), (2, 9)))
    o = window_attention(q, k, v, 4, 1)
    assert o.shape == (0, 4, 5, D) and o.dtype == BF
    got = torch.autograd.grad(o, (q, k, v), torch.zeros_like(o))
    assert [g.shape for g in got] == [x.shape for x in (q, k, v)]
    with torch.no_grad():
        assert window_attention(q, k, v).shape == o.shape
    for bad in (lambda: window_attention(q, k, v, 0), lambda: window_attention(q[:, :3], k, v, 4), lambda: window_attention(q, k, v, 4, 0, -1.0), lambda: window_attention(q.float(), k.float(), v.float(), 4)):
        with pytest.raises(DltError):
            bad()


# ---- tensors that share memory ------------------------------------------------------------------------------------------------------------
def test_written_tensors_that_overlap_are_refused():
    """Tensors that a call writes share no memory: parts of one tensor that meet are refused, parts beside each other are taken."""
    pos, tables = torch.arange(5, dtype=torch.int32, device="cuda")[None], [orc.table(8, 32).cuda()]
    for dtype in (BF, F32):
        pack = torch.randn(2, 6, 5, 64, generator=torch.Generator().manual_seed(60)).to(dtype).cuda()
        tokens = pack.transpose(1, 2).contiguous().transpose(1, 2)   # tokens outside heads
        for x in (pack, tokens):
            before = x.clone()
            for a, b in ((x[:, :4], x[:, 3:]), (x[:, 2:], x[:, :3]), (x[:1], x[:1, 1:4]), (x[:, ::2], x[:, 2:3])):
                with pytest.raises(RuntimeError, match="share memory|two tensors"):
                    rope_axes_qk_(a, b, pos, tables)
            assert torch.equal(x, before)
            want = rope_axes_qk(x, None, pos, tables)[0]
            rope_axes_qk_(x[:, :4], x[:, 4:], pos, tables)
            assert torch.equal(x, want)
            want = rope_axes_qk(x, None, pos, tables)[0]
            rope_axes_qk_(x[:, ::2], x[:, 1::2], pos, tables)
            assert torch.equal(x, want)
    both = torch.zeros(9, 2, 2, 16, 64, dtype=BF, device="cuda")
    k, seq, pages = torch.zeros(1, 2, 3, 64, dtype=BF, device="cuda"), ints(3), ints(0, 1)[None]
    flat = both.reshape(36, 16, 64)
    for a, b in ((both[:8, 0], both[1:, 0]), (both[:, 0], both[:, 0]), (flat[:16].reshape(8, 2, 16, 64), flat[2:18].reshape(8, 2, 16, 64))):
        with pytest.raises(RuntimeError, match="share memory|two tensors"):
            paged_append_(a, b, k, k, pages, seq)
    assert paged_append_(both[:, 0], both[:, 1], k, k, pages, seq) is None
    assert paged_append_(both[:4, 0], both[4:8, 0], k, k, pages, seq) is None


# ---- bounds by the number of terms -----------------------------------------------------------------------------------------------------------
TERMS = [
    # B, Hq, Hkv, Lq, Lk, dk, dv, window, sinks, dtype
    (1, 1, 1, 64, 64, 64, 64, None, 0, HF),
    (2, 4, 2, 200, 200, 64, 64, 64, 4, HF),
    (1, 6, 2, 257, 301, 80, 80, 100, 5, HF),
    (1, 1, 1, 513, 513, 128, 128, 128, 64, HF),
    (1, 2, 1, 10, 5000, 128, 128, None, 0, HF),
    (1, 1, 1, 1, 9000, 64, 64, None, 0, BF),
    (1, 4, 1, 3000, 3000, 64, 64, 33, 4, BF),
    (1, 1, 1, 4000, 4000, 64, 64, 17, 128, HF),
]


@pytest.mark.parametrize("case", TERMS, ids=name_of)
def test_against_64_bits_with_bounds_of_the_terms(case, monkeypatch):
    """The bounds of long_oracle with its flat slack replaced by what the case's own sums can be off by, relative to the sum of the terms' magnitudes.
    A sum of n products in 32 bits: n 2^-24.  A score is a sum of dk products, so that a probability is off by dk 2^-24 times the largest sum of |q k| (scaled); its exponential, logarithm
    and the softmax's own sum, of up to Lk terms, add (64 + Lk) 2^-24.  Second-order products of up to four roundings of u: 8 u^2.  o and dq sum Lk terms, dk and dv Lq times the
    heads of a group."""
    B, Hq, Hkv, Lq, Lk, dk, dv, window, n_sink, dtype = case
    gen = torch.Generator().manual_seed(61)
    mk = lambda *s: torch.randn(s, generator=gen).to(dtype).cuda()  # noqa: E731
    q, k, v, do = mk(B, Hq, Lq, dk), mk(B, Hkv, Lk, dk), mk(B, Hkv, Lk, dv), mk(B, Hq, Lq, dv)
    scale, G, u = 1.0 / math.sqrt(dk), Hq // Hkv, torch.finfo(dtype).eps / 2
    reach = float((q.double().abs() @ k.double().abs().repeat_interleave(G, 1).transpose(-1, -2)).amax()) * scale
    common = (dk * reach + 64 + Lk + dv) * 2.0 ** -24 + 8 * u * u
    for x in (q, k, v):
        x.requires_grad_(True)
    o = window_attention(q, k, v, window, n_sink, scale)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, (q, k, v), do)))
    q, k, v = (x.detach() for x in (q, k, v))
    for names, terms in ((("o", "dq"), Lk), (("dk", "dv"), Lq * G)):
        monkeypatch.setattr(orc, "SLACK", common + terms * 2.0 ** -24)
        want = orc.window(q, k, v, window, n_sink, scale, do)
        for name in names:
            orc.check(got[name], want[name], name)


# ---- captured backward passes ------------------------------------------------------------------------------------------------------------------
def test_a_captured_backward_pass_that_asks_for_other_leaves_is_taken():
    """A leaf of a live graph of the default stream is in the way only where its gradient is asked for."""
    gen = torch.Generator().manual_seed(62)
    q, k, v = (torch.randn(1, 2, 40, 64, generator=gen).to(BF).cuda().requires_grad_(True) for _ in range(3))
    side = torch.cuda.Stream()
    eager = window_attention(q, k.detach(), v.detach(), 8)   # holds q alone
    with torch.cuda.stream(side):
        want = torch.autograd.grad(window_attention(q.detach(), k, v, 8), (k, v), eager.detach())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = window_attention(q, k, v, 8)
        with pytest.raises(RuntimeError, match="graph of the default stream"):
            torch.autograd.grad(o, (q, k), eager.detach(), retain_graph=True)
        got = torch.autograd.grad(o, (k, v), eager.detach())
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.autograd.grad(eager, q, eager.detach())[0].isfinite().all()
