"""The long-sequence operators' refusals, workspaces and routes, asked through the C ABI and the Python entry points without a GPU."""
import ctypes
import os

import pytest
import torch

BF16, FP16, FP32 = 0, 1, 2
MAX = 2 ** 31 - 1
ONE = ctypes.c_void_p(256)   # never dereferenced
I64 = lambda *x: (ctypes.c_int64 * len(x))(*x)  # noqa: E731


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


WINDOW = dict(B=1, H=4, Hkv=2, Lq=64, Lk=64, dk=64, dv=64, window=16, n_sink=0, sm_scale=0.125, dtype=BF16)


def window(L, backward=False, ptr=None, st=None, ws=ONE, ws_bytes=1 << 40, **kw):
    s = L.WindowShape(**{**WINDOW, **kw})
    ptr, st = ptr or {}, st or {}
    t = {"q": (s.H, s.Lq, s.dk), "k": (s.Hkv, s.Lk, s.dk), "v": (s.Hkv, s.Lk, s.dv), "o": (s.H, s.Lq, s.dv), "d_o": (s.H, s.Lq, s.dv),
         "dq": (s.H, s.Lq, s.dk), "dk": (s.Hkv, s.Lk, s.dk), "dv": (s.Hkv, s.Lk, s.dv)}
    arg = lambda n: [ptr.get(n, ONE), st.get(n, dense(*t[n]))]  # noqa: E731
    lib = L.load()
    if backward:
        args = sum((arg(n) for n in ("q", "k", "v", "o")), []) + [ptr.get("low")] + arg("d_o") + [ptr.get("lse2", ONE), ptr.get("delta", ONE)] + sum((arg(n) for n in ("dq", "dk", "dv")), [])
        return lib.dlt_window_bwd(*args, s, ws, ws_bytes, None)
    return lib.dlt_window_fwd(*sum((arg(n) for n in "qkvo"), []), ptr.get("low"), ptr.get("lse2", ONE), s, ws, ws_bytes, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw, rc, text", [
    (dict(dtype=7), 1, "dtype"), (dict(dtype=FP32), 2, "fp32"), (dict(dk=136), 2, "head dims"), (dict(dv=60), 2, "head dims"), (dict(dk=0), 1, "positive"),
    (dict(B=0), 1, "positive"), (dict(Hkv=0), 1, "positive"), (dict(H=5), 1, "evenly"), (dict(window=0), 1, "window"), (dict(window=-3), 1, "window"),
    (dict(n_sink=-1), 1, "n_sink"), (dict(sm_scale=0.0), 1, "sm_scale"), (dict(sm_scale=-1.0), 1, "sm_scale"), (dict(sm_scale=float("nan")), 1, "sm_scale"),
    (dict(sm_scale=float("inf")), 1, "sm_scale"), (dict(Lq=-1), 1, "length"), (dict(Lk=1 << 30), 2, "tokens"), (dict(Lq=1 << 29), 2, "tokens"),
    (dict(ptr={"k": None}), 1, "k is NULL"), (dict(ptr={"q": ctypes.c_void_p(264)}), 1, "16 bytes"), (dict(ptr={"low": ctypes.c_void_p(264)}), 1, "o_low"),
    (dict(st={"v": I64(8192, 4096, 68, 1)}), 1, "16 bytes"), (dict(st={"q": I64(16384, 4096, 64, 2)}), 1, "contiguous"), (dict(st={"k": I64(8192, -4096, 64, 1)}), 1, "negative"),
    (dict(st={"k": I64(8192, 4096, 1 << 27, 1)}), 2, "too large"), (dict(st={"q": I64(8192, 1 << 29, 64, 1)}), 2, "too large"),
    (dict(B=MAX, Lk=4096, Lq=4096), 2, "workgroups"),
])
def test_window_refusals(L, backward, kw, rc, text):
    assert window(L, backward, **kw) == rc and text in err(L)


@pytest.mark.parametrize("kw", [{}, dict(Lq=0), dict(Lk=0), dict(window=MAX, n_sink=MAX), dict(H=2, dk=8, dv=128), dict(Lq=1, Lk=(1 << 30) - 1), dict(dtype=FP16, n_sink=64)])
def test_window_accepts(L, kw):
    lib = L.load()
    for backward in (False, True):
        assert window(L, backward, **kw) == 0, err(L)
        assert lib.dlt_last_kernel_family() == L.KERNEL_FAMILIES.index("band")
    assert window(L, ptr={"lse2": None}, **kw) == 0, err(L)   # a forward pass alone needs no sums
    assert kw.get("Lq") == 0 or (window(L, True, ptr={"lse2": None}, **kw) == 1 and "lse2" in err(L))
    if kw.get("Lq") == 0:   # a tensor without elements may be NULL
        assert window(L, ptr={"q": None, "o": None, "lse2": None}, **kw) == 0, err(L)


def test_window_workspace(L):
    lib = L.load()

    def need(backward, **kw):
        n = ctypes.c_int64(-1)
        assert lib.dlt_window_workspace(L.WindowShape(**{**WINDOW, **kw}), backward, ctypes.byref(n)) == 0, err(L)
        return n.value
    assert lib.dlt_window_workspace(L.WindowShape(**WINDOW), 0, None) == 1 and "NULL" in err(L)
    assert need(0) == 0 and need(1) == 0
    few = dict(Lq=1, Lk=20000, window=MAX)          # a decode step: one block of rows, keys shared
    assert need(0, **few) > 0
    assert need(1, Lq=20000, Lk=64, window=MAX, n_sink=4) == 0   # 64 rows see these keys: the queries before them stand at negative positions
    wide = dict(H=32, Hkv=1, Lq=1000, Lk=1000, window=MAX)   # few blocks of keys, many rows
    assert need(1, **wide) > 0
    for backward, kw in ((0, few), (1, wide)):
        n = need(backward, **kw)
        assert window(L, bool(backward), ws_bytes=n, **kw) == 0, err(L)
        assert window(L, bool(backward), ws_bytes=n - 1, **kw) == 1 and "workspace" in err(L)
        assert window(L, bool(backward), ws=None, ws_bytes=0, **kw) == 1 and "workspace" in err(L)
        assert window(L, bool(backward), ws=ctypes.c_void_p(264), ws_bytes=n, **kw) == 1 and "workspace" in err(L)
    for kw in (dict(B=300, H=32, Hkv=32, Lq=2000, Lk=2000, n_sink=2000, dk=128, dv=128), dict(Lq=1 << 20, Lk=1 << 20, n_sink=1 << 20), dict(Lq=1 << 24, Lk=(1 << 30) - 1, window=MAX),
               dict(H=MAX // 2, Hkv=1, Lq=1, Lk=1 << 20), dict(B=1 << 16, H=64, Hkv=64, Lq=1 << 14, Lk=1 << 14, n_sink=4)):
        assert need(0, **kw) <= 256 << 20 and need(1, **kw) <= 256 << 20, kw


def test_window_low_tokens(L):
    lib, n = L.load(), ctypes.c_int32(-1)

    def tokens(**kw):
        assert lib.dlt_window_low_tokens(L.WindowShape(**{**WINDOW, **kw}), ctypes.byref(n)) == 0, err(L)
        return n.value
    assert lib.dlt_window_low_tokens(L.WindowShape(**WINDOW), None) == 1 and "NULL" in err(L)
    # all rows of a window of up to 16 keys, sinks counted; else those of positions below 16, the queries before the first key among them
    assert tokens() == 64 and tokens(window=15, n_sink=1) == 64 and tokens(window=17) == 16 and tokens(window=16, n_sink=1) == 16 and tokens(window=MAX, n_sink=MAX) == 16
    assert tokens(window=100, Lk=70) == 10 and tokens(window=100, Lk=200) == 0 and tokens(window=40, Lk=54) == 26 and tokens(window=100, Lq=3) == 0 and tokens(window=100, Lq=3, Lk=5) == 3


PAGED = dict(B=2, H=4, Hkv=2, T=1, dk=64, dv=64, page=16, n_pages=100, cols=10, window=MAX, n_sink=0, sm_scale=0.125, dtype=BF16)


def attend(L, ptr=None, st=None, ws=ONE, ws_bytes=1 << 40, table_stride=10, **kw):
    s = L.PagedShape(**{**PAGED, **kw})
    ptr, st = ptr or {}, st or {}
    t = {"q": (s.H, s.T, s.dk), "k": (s.Hkv, s.page, s.dk), "v": (s.Hkv, s.page, s.dv), "o": (s.H, s.T, s.dv)}
    args = sum(([ptr.get(n, ONE), st.get(n, dense(*t[n]))] for n in "qkvo"), [])
    return L.load().dlt_paged_attn(*args, ptr.get("table", ONE), table_stride, ptr.get("seq", ONE), None, s, ws, ws_bytes, None)


@pytest.mark.parametrize("kw, rc, text", [
    (dict(dtype=7), 1, "dtype"), (dict(dtype=FP32), 2, "fp32"), (dict(dk=136), 2, "head dims"), (dict(page=24), 2, "multiple of 16"), (dict(page=0), 1, "page"),
    (dict(cols=0), 1, "cols"), (dict(n_pages=0), 1, "n_pages"), (dict(H=3), 1, "evenly"), (dict(B=0), 1, "positive"), (dict(T=-1), 1, "T="), (dict(window=0), 1, "window"),
    (dict(sm_scale=0.0), 1, "sm_scale"), (dict(cols=1 << 27), 2, "tokens"), (dict(ptr={"table": None}), 1, "table"), (dict(ptr={"seq": None}), 1, "seq_len"),
    (dict(ptr={"k": None}), 1, "NULL"), (dict(ptr={"v": ctypes.c_void_p(264)}), 1, "16 bytes"), (dict(st={"k": I64(2048, 1024, 65, 1)}), 1, "16 bytes"),
    (dict(table_stride=-1), 1, "stride"),
])
def test_paged_attention_refusals(L, kw, rc, text):
    assert attend(L, **kw) == rc and text in err(L)


def test_paged_workspace(L):
    lib, n = L.load(), ctypes.c_int64(-1)
    assert attend(L) == 0 and lib.dlt_last_kernel_family() == L.KERNEL_FAMILIES.index("band")
    assert attend(L, T=0, ptr={"q": None, "o": None}) == 0, err(L)
    assert lib.dlt_paged_workspace(L.PagedShape(**PAGED), None) == 1 and "NULL" in err(L)
    assert lib.dlt_paged_workspace(L.PagedShape(**PAGED), ctypes.byref(n)) == 0 and n.value == 0
    long = dict(cols=4000, n_pages=8000, table_stride=4000)
    assert lib.dlt_paged_workspace(L.PagedShape(**{**PAGED, "cols": 4000, "n_pages": 8000}), ctypes.byref(n)) == 0 and n.value > 0
    assert attend(L, ws_bytes=n.value, **long) == 0, err(L)
    assert attend(L, ws_bytes=n.value - 1, **long) == 1 and "workspace" in err(L)


def test_append_refusals(L):
    lib = L.load()
    tab = L.RopeAxesDesc(1, 0, None, I64(0, 0, 0), (ctypes.c_void_p * 4)(256), I64(64, 0, 0, 0), (ctypes.c_int32 * 4)(32), (ctypes.c_int32 * 4)(100))

    def append(rope=None, ptr=None, table_stride=10, **kw):
        s = L.PagedShape(**{**PAGED, **kw})
        ptr = ptr or {}
        a = lambda n, *shape: [ptr.get(n, ONE), dense(*shape)]  # noqa: E731
        return lib.dlt_paged_append(*a("k", s.Hkv, s.T, s.dk), *a("v", s.Hkv, s.T, s.dv), *a("q", s.H, s.T, s.dk), ptr.get("q_out", ctypes.c_void_p(512)), dense(s.H, s.T, s.dk),
                                    *a("kc", s.Hkv, s.page, s.dk), *a("vc", s.Hkv, s.page, s.dv), ptr.get("table", ONE), table_stride, ptr.get("seq", ONE), None, rope, s, None)
    for kw, text in ((dict(dtype=7), "dtype"), (dict(B=0), "B=0"), (dict(Hkv=0), "Hkv=0"), (dict(T=-1), "T=-1"), (dict(dv=0), "dv=0"), (dict(cols=0), "cols"), (dict(page=-1), "page"),
                     (dict(cols=1 << 28), "cols"), (dict(ptr={"table": None}), "NULL"), (dict(ptr={"seq": None}), "NULL"), (dict(ptr={"k": None}), "NULL"), (dict(ptr={"vc": None}), "NULL"),
                     (dict(ptr={"q": None}), "NULL"), (dict(ptr={"q_out": ONE}), "two buffers"), (dict(table_stride=-1), "stride"), (dict(dk=62, rope=tab), "pairs")):
        assert append(**kw) == 1 and text in err(L), kw
    assert append(T=0, rope=tab, ptr={"k": None, "v": None, "q": None, "q_out": None}) == 0, err(L)


def test_rope_axes_refusals(L):
    lib = L.load()

    def rope(n_axes=2, layout=0, pos=256, tables=(256, 256), strides=(32, 32), n_rdim=(16, 16), lens=(9, 9), q=ONE, q_out=ONE, q_out_strides=None, dtype=BF16, B=1, Hq=2, Hk=0, N=10,
             C=64, desc=True):
        pad = lambda t, x, z: (t * 4)(*(list(x) + [z] * 4)[:4])  # noqa: E731
        d = L.RopeAxesDesc(n_axes, layout, pos, I64(N, 0, 1), pad(ctypes.c_void_p, tables, None), pad(ctypes.c_int64, strides, 0), pad(ctypes.c_int32, n_rdim, 0), pad(ctypes.c_int32, lens, 0))
        return lib.dlt_rope_axes(q, dense(Hq, N, C), q_out, q_out_strides or dense(Hq, N, C), Hq, None, None, None, None, Hk, B, N, C, d if desc else None, 0, dtype, None)
    for kw, text in ((dict(n_axes=0), "axes"), (dict(n_axes=5), "axes"), (dict(layout=2), "layout"), (dict(pos=None), "pos"), (dict(tables=(256, None)), "table"), (dict(lens=(9, 0)), "empty"),
                     (dict(strides=(32, 30)), "rows of the table"), (dict(strides=(33, 32)), "rows of the table"), (dict(tables=(260, 256)), "rows of the table"), (dict(n_rdim=(16, -1)), "axis 1"),
                     (dict(n_rdim=(16, 17), strides=(32, 34)), "pairs"), (dict(dtype=3), "dtype"), (dict(q=None), "NULL"), (dict(Hk=1), "NULL"), (dict(B=-1), "shape"), (dict(C=0), "shape"),
                     (dict(desc=False), "descriptor"), (dict(q_out_strides=I64(1280, 640, 64, 2)), "in place")):
        assert rope(**kw) == 1 and text in err(L), (kw, err(L))
    assert rope(N=0, q=None, q_out=None) == 0 and rope(B=0, q=None, q_out=None) == 0


def test_python_refusals():
    """Arguments that are wrong whatever the device, and tensors that lie on the host."""
    from dl_templates_amd.paged_cache import paged_append_, paged_attention
    from dl_templates_amd.rope_axes import RotaryPositionEncodingAxes, rope_axes_qk, rope_axes_qk_
    from dl_templates_amd.window_attn import window_attention
    x = torch.zeros(1, 2, 4, 16, dtype=torch.bfloat16)
    pos, tables = torch.zeros(1, 4, dtype=torch.int32), [torch.zeros(5, 4, 2)]
    for call in (lambda: window_attention(x, x, x, 4), lambda: window_attention(x, x, x), lambda: rope_axes_qk(x, x, pos, tables), lambda: rope_axes_qk_(x, None, pos, tables)):
        with pytest.raises(RuntimeError, match="ROCm GPU only"):
            call()
    with pytest.raises(OverflowError):
        window_attention(x, x, x, 1 << 40)
    with pytest.raises(TypeError):
        window_attention(x, x, x, 2.5)
    with pytest.raises(ValueError, match="layout"):
        rope_axes_qk(x, x, pos, tables, "rows")
    with pytest.raises(RuntimeError, match="records no graph"):
        rope_axes_qk_(x.clone().requires_grad_(), None, pos, tables)
    with pytest.raises(ValueError, match="every axis"):
        RotaryPositionEncodingAxes((8, 8), (4,))
    ints = torch.zeros(1, dtype=torch.int32)
    cache = torch.zeros(3, 2, 16, 16, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        paged_attention(x, cache, cache, ints[None], ints)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        paged_append_(cache, cache.clone(), x, x, ints[None], ints)
    with pytest.raises(TypeError, match="page_table"):
        paged_attention(x, cache, cache, ints[None].long(), ints)
    with pytest.raises(TypeError, match="seq_len"):
        paged_attention(x, cache, cache, ints[None], ints.long())
    with pytest.raises(AssertionError, match="every sequence"):
        paged_attention(x, cache, cache, ints[None], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(AssertionError, match="match the cache"):
        paged_attention(x[..., :8], cache, cache, ints[None], ints)
    with pytest.raises(AssertionError, match="match their caches"):
        paged_append_(cache, cache.clone(), x[:, :1], x[:, :1], ints[None], ints)
    with pytest.raises(AssertionError, match="one dtype"):
        paged_append_(cache, cache.clone(), x.half(), x.half(), ints[None], ints)


def test_grid_positions():
    from dl_templates_amd.rope_axes import RotaryPositionEncodingAxes
    assert RotaryPositionEncodingAxes.encode_pos(2, 3).tolist() == [[0, 0, 0, 1, 1, 1], [0, 1, 2, 0, 1, 2]]
    m = RotaryPositionEncodingAxes((8, 12), (5, 7), "halves")
    assert [tuple(t.shape) for t in m.tables] == [(5, 4, 2), (7, 6, 2)]
