"""Refusals, workspaces and routes of the 8-bit cache's operators and of the pool, asked through the C ABI and the Python entry points without a GPU; the oracle's own rounding."""
import ctypes
import os

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad
from torch.utils._python_dispatch import TorchDispatchMode

from tests import paged8_oracle as orc8

BF16, FP16, FP32, E4M3, INT8 = 0, 1, 2, 0, 1
ONE = ctypes.c_void_p(256)   # never dereferenced
I64 = lambda *x: (ctypes.c_int64 * len(x))(*x)  # noqa: E731
SHAPE = dict(B=2, H=4, Hkv=2, T=1, dk=64, dv=64, page=64, n_pages=20, cols=10, window=2 ** 31 - 1, n_sink=0, sm_scale=0.125, dtype=BF16)


@pytest.fixture(scope="module")
def L():
    from dl_templates_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libdlt_hip.so not built (run __graft_entry__.build())")
    lib = _lib.load()
    lib.dlt_dry_run(1)
    yield _lib
    lib.dlt_dry_run(0)


def dense(H, N, D):
    return I64(H * N * D, N * D, D, 1)


def err(L):
    return L.load().dlt_last_error().decode()


def scales(L, format=E4M3, block=32, k=256, v=256, strides=(4, 2, 1)):
    return L.Scales8(format, block, k, v, I64(*strides), I64(*strides))


def attend(L, sc=None, ptr=None, st=None, table_stride=10, ws=ONE, ws_bytes=1 << 40, **kw):
    s = L.PagedShape(**{**SHAPE, **kw})
    ptr, st = ptr or {}, st or {}
    t = {"q": (s.H, s.T, s.dk), "k": (s.Hkv, s.page, s.dk), "v": (s.Hkv, s.page, s.dv), "o": (s.H, s.T, s.dv)}
    a = lambda n: [ptr.get(n, ONE), st.get(n, dense(*t[n]))]  # noqa: E731
    return L.load().dlt_paged8_attn(*a("q"), *a("k"), *a("v"), ptr.get("scales", sc or scales(L)), *a("o"), ptr.get("table", ONE), table_stride, ptr.get("seq", ONE), None, s, ws, ws_bytes, None)


@pytest.mark.parametrize("kw, rc, text", [
    (dict(dtype=7), 1, "dtype"), (dict(dtype=FP32), 2, "fp32"), (dict(dk=136), 2, "head dims"), (dict(dv=60), 2, "head dims"), (dict(page=24), 2, "multiple of 16"), (dict(H=3), 1, "evenly"),
    (dict(B=0), 1, "positive"), (dict(T=-1), 1, "T="), (dict(window=0), 1, "window"), (dict(sm_scale=float("nan")), 1, "sm_scale"), (dict(cols=1 << 27), 2, "tokens"),
    (dict(ptr={"table": None}), 1, "table"), (dict(ptr={"k": None}), 1, "NULL"), (dict(ptr={"v": ctypes.c_void_p(260)}), 1, "8 bytes"), (dict(ptr={"q": ctypes.c_void_p(264)}), 1, "16 bytes"),
    (dict(st={"k": I64(2048, 1024, 68, 1)}), 1, "8 bytes"), (dict(st={"v": I64(2048, -1024, 64, 1)}), 1, "negative"), (dict(st={"k": I64(2048, 1024, 1 << 40, 1)}), 2, "too large"),
    (dict(table_stride=-1), 1, "stride"), (dict(ptr={"scales": None}), 1, "scales is NULL"),
])
def test_attention_refusals(L, kw, rc, text):
    assert attend(L, **kw) == rc and text in err(L), err(L)


@pytest.mark.parametrize("kw, rc, text", [(dict(format=2), 1, "format"), (dict(block=48), 1, "whole blocks"), (dict(block=0), 1, "whole blocks"), (dict(block=8), 2, "multiple of 16"),
                                          (dict(k=None), 1, "scales is NULL"), (dict(strides=(4, -2, 1)), 1, "negative stride")])
def test_scale_refusals(L, kw, rc, text):
    assert attend(L, scales(L, **kw)) == rc and text in err(L), err(L)
    n = ctypes.c_int64()
    assert L.load().dlt_paged8_workspace(L.PagedShape(**SHAPE), scales(L, **kw), ctypes.byref(n)) == rc


def test_blocks_over_the_limit(L):
    assert attend(L, scales(L, block=256), page=256) == 2 and "up to 128" in err(L)
    assert attend(L, scales(L, block=128), page=256) == 0, err(L)


def test_workspace_and_route(L):
    lib, n = L.load(), ctypes.c_int64(-1)
    assert attend(L) == 0 and lib.dlt_last_kernel_family() == L.KERNEL_FAMILIES.index("band")
    assert attend(L, T=0, ptr={"q": None, "o": None}) == 0, err(L)
    assert lib.dlt_paged8_workspace(L.PagedShape(**SHAPE), scales(L), None) == 1 and "NULL" in err(L)

    def need(**kw):
        assert lib.dlt_paged8_workspace(L.PagedShape(**{**SHAPE, **kw}), scales(L), ctypes.byref(n)) == 0, err(L)
        return n.value
    assert need() == 0
    for kw in (dict(cols=4000), dict(cols=4000, T=7), dict(cols=4000, T=30, H=8), dict(cols=4000, T=300, H=8)):
        size = need(**kw)
        assert 0 < size <= 256 << 20
        assert attend(L, ws_bytes=size, table_stride=4000, **kw) == 0, err(L)
        assert attend(L, ws_bytes=size - 1, table_stride=4000, **kw) == 1 and "workspace" in err(L)
        assert attend(L, ws=ctypes.c_void_p(264), table_stride=4000, **kw) == 1
    # a table as wide, but few keys that a row can see
    assert need(cols=4000, window=500) == 0
    # more sequences than the lists of runs hold: whole heads
    assert need(cols=4000, B=5000) == 0


def test_append_refusals(L):
    lib = L.load()
    tab = L.RopeAxesDesc(1, 0, None, I64(0, 0, 0), (ctypes.c_void_p * 4)(256), I64(64, 0, 0, 0), (ctypes.c_int32 * 4)(32), (ctypes.c_int32 * 4)(100))

    def append(rope=None, ptr=None, st=None, sc=None, table_stride=10, **kw):
        s = L.PagedShape(**{**SHAPE, **kw})
        ptr, st = ptr or {}, st or {}
        a = lambda n, *shape: [ptr.get(n, ONE), st.get(n, dense(*shape))]  # noqa: E731
        return lib.dlt_paged8_append(*a("k", s.Hkv, s.T, s.dk), *a("v", s.Hkv, s.T, s.dv), *a("q", s.H, s.T, s.dk), ptr.get("q_out", ctypes.c_void_p(512)), dense(s.H, s.T, s.dk),
                                     *a("kc", s.Hkv, s.page, s.dk), *a("vc", s.Hkv, s.page, s.dv), ptr.get("scales", sc or scales(L)), ptr.get("table", ONE), table_stride, ptr.get("seq", ONE), None,
                                     rope, s, None)
    for kw, rc, text in ((dict(dtype=7), 1, "dtype"), (dict(B=0), 1, "B=0"), (dict(Hkv=0), 1, "Hkv=0"), (dict(T=-1), 1, "T=-1"), (dict(cols=0), 1, "cols"), (dict(cols=1 << 28), 1, "cols"),
                         (dict(dk=136), 2, "head dims"), (dict(dv=60), 2, "head dims"), (dict(ptr={"table": None}), 1, "NULL"), (dict(ptr={"seq": None}), 1, "NULL"),
                         (dict(ptr={"k": None}), 1, "NULL"), (dict(ptr={"vc": None}), 1, "NULL"), (dict(ptr={"q": None}), 1, "NULL"), (dict(ptr={"q_out": ONE}), 1, "two buffers"),
                         (dict(ptr={"scales": None}), 1, "scales is NULL"), (dict(sc=scales(L, block=48)), 1, "whole blocks"), (dict(sc=scales(L, format=-1)), 1, "format"),
                         (dict(table_stride=-1), 1, "stride"), (dict(dk=56, rope=tab), 1, "pairs"), (dict(ptr={"k": ctypes.c_void_p(264)}), 1, "16 bytes"),
                         (dict(ptr={"kc": ctypes.c_void_p(260)}), 1, "8 bytes"), (dict(st={"v": I64(128, 68, 68, 1)}), 1, "16 bytes"), (dict(st={"kc": I64(128, 64, 64, 2)}), 1, "contiguous"),
                         (dict(st={"vc": I64(8200, 4096, 68, 1)}), 1, "8 bytes"), (dict(B=1 << 20, T=1 << 12), 2, "one launch")):
        assert append(**kw) == rc and text in err(L), (kw, err(L))
    assert append(T=0, rope=tab, ptr={"k": None, "v": None, "q": None, "q_out": None}) == 0, err(L)


def test_assign_refusals(L):
    def assign(table=ONE, table_stride=10, seq=ONE, want=ONE, pool=ONE, B=4, cols=10, page=16, n_pages=100, T=3, n_new=ONE, slots=ONE):
        return L.load().dlt_page_assign(table, table_stride, seq, want, pool, B, cols, page, n_pages, T, n_new, slots, None)
    for kw, rc, text in ((dict(B=-1), 1, "B=-1"), (dict(cols=0), 1, "cols=0"), (dict(page=0), 1, "page=0"), (dict(n_pages=0), 1, "n_pages=0"), (dict(T=-2), 1, "T=-2"), (dict(B=8193), 2, "8192"),
                         (dict(cols=1 << 28), 2, "too many"), (dict(page=1 << 27), 2, "too many"), (dict(n_pages=1 << 29), 2, "too many"), (dict(T=1 << 30), 2, "too many"),
                         (dict(table=None), 1, "NULL"), (dict(seq=None), 1, "NULL"), (dict(want=None), 1, "NULL"), (dict(pool=None), 1, "NULL"), (dict(n_new=None), 1, "NULL"),
                         (dict(slots=None), 1, "NULL"), (dict(table_stride=9), 1, "overlap"), (dict(slots=ctypes.c_void_p(260)), 1, "16 bytes")):
        assert assign(**kw) == rc and text in err(L), (kw, err(L))
    assert assign(B=0, table=None, seq=None, want=None, pool=None, n_new=None, slots=None) == 0


def host():
    x = torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16)
    cache = torch.zeros(3, 2, 32, 16, dtype=torch.float8_e4m3fn)
    sc = torch.ones(3, 2, 2, dtype=torch.float8_e8m0fnu)
    return x, cache, cache.clone(), sc, sc.clone(), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)


def test_python_refusals():
    from dl_templates_amd.page_pool import page_assign_, page_pool
    from dl_templates_amd.paged_cache8 import paged8_append_, paged8_attention
    x, kc, vc, ks, vs, table, seq = host()
    append = lambda **kw: paged8_append_(*[kw.get(n, d) for n, d in dict(kc=kc, vc=vc, ks=ks, vs=vs, k=x, v=x, table=table, seq=seq, new=None, rope=None, q=None).items()])  # noqa: E731
    attention = lambda **kw: paged8_attention(*[kw.get(n, d) for n, d in dict(q=x, kc=kc, vc=vc, ks=ks, vs=vs, table=table, seq=seq, window=None, sink=0, scale=None, new=None).items()])  # noqa: E731
    for call in (append, attention):
        for kw, exc, text in ((dict(), RuntimeError, "ROCm GPU only"), (dict(kc=x), TypeError, "float8_e4m3fn or int8"), (dict(vc=vc.view(torch.int8)), TypeError, "both alike"),
                              (dict(kc=kc.view(torch.float8_e5m2), vc=vc.view(torch.float8_e5m2)), TypeError, "float8_e4m3fn or int8"), (dict(ks=ks.float()), TypeError, "e8m0fnu"),
                              (dict(ks=ks[:, :1]), AssertionError, "blocks of a page"), (dict(ks=ks[:, :, :1]), AssertionError, "blocks of a page"),
                              (dict(ks=torch.ones(3, 2, 3).to(torch.float8_e8m0fnu), vs=torch.ones(3, 2, 3).to(torch.float8_e8m0fnu)), ValueError, "one size"),
                              (dict(kc=kc[0]), AssertionError, "must have shape")):
            with pytest.raises(exc, match=text):
                call(**kw)
    with pytest.raises(ValueError, match="layout"):
        append(rope=(None, [torch.zeros(5, 8, 2)], "rows"))
    t, s, p = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), page_pool(5, "cpu")
    assert p.tolist() == [5, 0, 4, 3, 2, 1, 0]
    for args, exc, text in (((t, s, s.clone(), p, 16), RuntimeError, "ROCm GPU only"), ((t.long(), s, s, p, 16), TypeError, "page_table"), ((t, s.long(), s, p, 16), TypeError, "seq_len and want"),
                            ((t, s, s.float(), p, 16), TypeError, "seq_len and want"), ((t, s, s, p[:2], 16), TypeError, "pool"), ((t, s, s[:2], p, 16), AssertionError, "every request"),
                            ((t, s, s, p, 0), ValueError, "token"), ((t[:, :0], s, s, p, 16), ValueError, "column"), ((t, s, s, p, 16, -1), ValueError, "n_tokens"), ((t, s, s, p, 2.5), TypeError, "")):
        with pytest.raises(exc, match=text):
            page_assign_(*args)
    with pytest.raises(ValueError, match="a page"):
        page_pool(0, "cpu")


@pytest.mark.parametrize("name", ["append", "attention"])
def test_tangents_and_transforms(name):
    from dl_templates_amd.paged_cache8 import paged8_append_, paged8_attention
    x, kc, vc, ks, vs, table, seq = host()
    call = {"append": lambda y: paged8_append_(kc, vc, ks, vs, y, x, table, seq, None, None, x), "attention": lambda y: paged8_attention(y, kc, vc, ks, vs, table, seq)}[name]
    with fwd_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        call(fwd_ad.make_dual(torch.ones_like(x), torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.vmap(call)(torch.zeros(3, *x.shape, dtype=x.dtype))
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        torch.jit.trace(call, (x,), check_trace=False)

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Seen(), pytest.raises(RuntimeError, match="ROCm GPU only"):
        call(x)


def test_the_oracles_rounding():
    gen = torch.Generator().manual_seed(0)
    x = (torch.randn(200000, generator=gen) * torch.exp2(torch.randint(-12, 8, (200000,), generator=gen).float())).clamp(-448, 448)
    assert torch.equal(orc8.rounded(x.double(), torch.float8_e4m3fn), x.to(torch.float8_e4m3fn).double())
    for fmt, top in ((torch.float8_e4m3fn, 448.0), (torch.int8, 127.0)):
        for big in (top, top * (1 + 2.0 ** -20), top * 2.0 ** -9, 1.0, 1e-30, 0.0):
            e = orc8.exponent(big, fmt)
            assert big <= top * 2.0 ** e and (e == orc8.LEAST or big > top * 2.0 ** (e - 1))
    assert orc8.exponent(0.0, torch.int8) == -100
    b = torch.tensor([0, 1, 127, 254, 255], dtype=torch.uint8)
    assert torch.equal(orc8.scales(b)[:4], b[:4].view(torch.float8_e8m0fnu).double()) and torch.isnan(orc8.scales(b)[4])


def test_the_loop_that_hands_out_pages():
    table, seq, free = [[-1] * 3 for _ in range(3)], [0, 0, 0], [3, 2, 1, 0]
    # two pages and one; the third request needs three, of which one is left
    assert orc8.assign(table, seq, [17, 5, 40], free, 16, 40) == ([17, 5, 0], [list(range(17)) + [-1] * 23, list(range(32, 37)) + [-1] * 35, [-1] * 40])
    assert seq == [17, 5, 0] and free == [3] and table == [[0, 1, -1], [2, -1, -1], [-1, -1, -1]]
    # the first ends: its pages come back, the last one first, and go to the second (two more) and the third
    assert orc8.assign(table, seq, [0, 33, 1], free, 16, None) == ([0, 28, 1], [[], [], []])
    assert seq == [0, 33, 1] and free == [] and table == [[0, 1, -1], [2, 0, 1], [3, -1, -1]]


def test_more_heads_than_a_launch_holds(L):
    """Up to 32 rows of a group have a workgroup to a (batch, kv head) or a run: their number must not wrap (2^20 x 2^12 heads came out as a launch of none)."""
    for B, Hkv in ((1 << 20, 1 << 12), (1 << 24, 1), ((1 << 31) - 1, 3)):
        for G in (1, 20):
            assert attend(L, B=B, H=G * Hkv, Hkv=Hkv, dk=8, dv=8) == 2 and "workgroups" in err(L), (B, Hkv, G)
    assert attend(L, B=(1 << 24) - 1, H=1, Hkv=1, dk=8, dv=8) == 0, err(L)
