"""Serving with a cache held in 8 bits: the operators whose speed this package answers for, as a program that uses them calls them, and their plain forms.

Three operators, which one program uses together, step by step:

* ``assign``  pages of the cache handed to requests from their lengths, and taken back: page tables and the places of the new tokens (``page_assign_``);
* ``append``  new keys and values rotated and written into a cache of 8-bit numbers with a scale for each block of tokens and head (``paged8_append_``);
* ``attend``  attention of the newest tokens of every sequence over that cache (``paged8_attention``).

``own`` false: elementary torch operations in 32 bits, rounded once.  ``own`` true: the package's operators.

A cache is [pages, heads, page, d] of ``float8_e4m3fn`` ("e4m3") or ``int8`` numbers c, its scales [pages, heads, page / block] of ``float8_e8m0fnu``, powers of two: the
cache holds c times its block's scale.  Caches of e4m3 come back as they are, beside their scales; those of int8 as the values c times scale.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def listed():
    return [
        # one decode step of a batch: every request gets a token more, a tenth are over and give their pages back (latency of a launch)
        dict(name="assign_step", op="assign", B=64, T=1, ctx=4096, page=64, over=0.1, spare=1.0),
        # prompts of unequal length admitted at once beside running requests, small pages, more than the pool holds: those behind wait
        dict(name="assign_prompts", op="assign", B=1000, T=4000, ctx=8192, page=16, over=0.2, spare=0.6),
        # one decode step of a batch: the latency of one launch
        dict(name="append_step_bf16", op="append", dtype="bf16", fmt="e4m3", B=64, Hq=16, Hkv=4, T=1, ctx=4096, page=64, block=64, d=128, rope="halves", padded=False),
        # prompts of unequal length, padded to the longest
        dict(name="append_prompts_fp16", op="append", dtype="fp16", fmt="e4m3", B=7, Hq=16, Hkv=8, T=2047, ctx=4096, page=16, block=16, d=64, rope="blocks", padded=True),
        # pieces of two prompts, block for block
        dict(name="append_chunk_int8", op="append", dtype="bf16", fmt="int8", B=2, Hq=16, Hkv=4, T=500, ctx=700, page=64, block=32, d=128, rope="halves", padded=False),
        # one sequence, a few tokens of context: latency
        dict(name="attend_short_fp16", op="attend", dtype="fp16", fmt="e4m3", B=1, Hq=8, Hkv=8, T=1, ctx=300, page=16, block=16, W=0, S=0, d=64, uneven=0, padded=False),
        # one decode step of a batch of unequal contexts
        dict(name="attend_batch_bf16", op="attend", dtype="bf16", fmt="e4m3", B=64, Hq=32, Hkv=8, T=1, ctx=8192, page=64, block=64, W=0, S=0, d=128, uneven=0, padded=False),
        # the same under a window, heads of 64, whole numbers of 8 bits
        dict(name="attend_window_int8", op="attend", dtype="fp16", fmt="int8", B=48, Hq=16, Hkv=8, T=1, ctx=6000, page=32, block=32, W=2048, S=4, d=64, uneven=0, padded=False),
        # a few tokens each (guessed ahead) of two very long sequences, all of them visible
        dict(name="attend_long_int8", op="attend", dtype="bf16", fmt="int8", B=2, Hq=16, Hkv=4, T=3, ctx=100000, page=32, block=32, W=0, S=0, d=128, uneven=0, padded=False),
        # one long context among short ones
        dict(name="attend_uneven_bf16", op="attend", dtype="bf16", fmt="e4m3", B=16, Hq=16, Hkv=4, T=1, ctx=32768, page=64, block=16, W=0, S=0, d=128, uneven=500, padded=False),
        # a piece of a prompt over what is there of it
        dict(name="attend_prompt_bf16", op="attend", dtype="bf16", fmt="e4m3", B=1, Hq=32, Hkv=8, T=512, ctx=8192, page=64, block=64, W=0, S=0, d=128, uneven=0, padded=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["assign", "append", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if op == "assign":
        B = _log(rng, 1, 1500)
        T = rng.choice([1, rng.randint(2, 8), _log(rng, 8, 4000)])
        ctx = T + _log(rng, 1, 8192)
        while B * ctx > 6000 * 1000:
            B = B // 2 + 1
        return dict(op=op, B=B, T=T, ctx=ctx, page=page, over=rng.choice([0.0, 0.1, 0.5]), spare=rng.choice([0.3, 0.7, 1.0]))
    block = rng.choice([b for b in range(16, page + 1, 16) if page % b == 0])
    fmt, d = rng.choice(["e4m3", "e4m3", "int8"]), rng.choice([32, 64, 64, 80, 96, 128, 128])
    Hkv, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    if op == "append":
        T = rng.choice([1, rng.randint(2, 8), _log(rng, 8, 1500)])
        B = _log(rng, 1, 96 if T < 9 else 6)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), fmt=fmt, B=B, Hq=Hkv * G, Hkv=Hkv, T=T, ctx=T + _log(rng, 1, 2500), page=page, block=block, d=d,
                    rope=rng.choice(["blocks", "halves", "none"]), padded=rng.random() < 0.5)
    T = rng.choice([1, 1, rng.randint(2, 7), _log(rng, 8, 300)])
    B = _log(rng, 1, 64) if T < 8 else rng.randint(1, 2)
    most = 8192 * 64 * 8 // 3 // (B * Hkv * (1 if T < 8 else G * T // 8))
    ctx = T + _log(rng, 1, max(2, min(65536, most)))
    return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), fmt=fmt, B=B, Hq=Hkv * G, Hkv=Hkv, T=T, ctx=ctx, page=page, block=block, W=rng.choice([0, 0, _log(rng, 1, 2 * ctx)]),
                S=rng.choice([0, 4, rng.randint(1, 70)]), d=d, uneven=rng.choice([0, 0, _log(rng, 1, ctx)]), padded=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _table(length, pairs):
    """Cos and sin of positions 0 .. length - 1, fp32 [length, pairs, 2], angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    ang = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def _requests(c, seed=1):
    """Tokens that every request holds, and those that it wants to hold."""
    host = np.random.RandomState(seed)
    held = host.randint(0, c["ctx"] - c["T"] + 1, c["B"])
    want = held + (1 if c["T"] == 1 else host.randint(0, c["T"] + 1, c["B"]))
    want[host.rand(c["B"]) < c["over"]] = 0
    want[0] = held[0] + c["T"]
    return held, want


def _prepare_assign(c, seed):
    host = np.random.RandomState(seed + 1)
    held, want = _requests(c, seed)
    cols = -(-c["ctx"] // c["page"])
    pages = lambda n: -(-n // c["page"])  # noqa: E731
    used, back, asked = pages(held), np.maximum(pages(held) - pages(want), 0), np.maximum(pages(want) - pages(held), 0)
    # `spare`: of what is asked for, the part that what is free and what comes back can give
    free = max(0, int(c["spare"] * asked.sum()) - int(back.sum()))
    n = c["B"] * cols
    numbers = host.permutation(n)
    table = np.full((c["B"], cols), -1, dtype=np.int32)
    table[np.arange(cols)[None] < used[:, None]] = numbers[:used.sum()]
    pool = np.full(n + 2, -1, dtype=np.int32)
    pool[0], pool[1] = free, 0
    pool[2:2 + free] = numbers[used.sum():used.sum() + free]
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()  # noqa: E731
    return dict(case=c, table=put(table), seq=put(held), held=put(held), want=put(want), pool=put(pool))


def _lengths(c, seed=1):
    """Counts of new tokens and lengths, new ones included; the first sequence is the longest."""
    host = np.random.RandomState(seed)
    new = host.randint(0, c["T"] + 1, c["B"]) if c["padded"] else np.full(c["B"], c["T"])
    new[0] = c["T"]
    seq = np.array([host.randint(n, max(n, c.get("uneven") or c["ctx"]) + 1) for n in new])
    seq[0] = c["ctx"]
    return new, seq


def _held_cache(x, block, fmt):
    """x [pages, heads, page, d] in 8 bits, as a program that filled it earlier holds it: numbers, scales."""
    n, h, page, d = x.shape
    x = x.float().reshape(n, h, page // block, block, d)
    top = 448.0 if fmt == "e4m3" else 127.0
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((-1, -2)).clamp_min(1e-20) / top)))
    x = (x / scale[..., None, None]).clamp_(-top, top)
    x = x.to(torch.float8_e4m3fn) if fmt == "e4m3" else x.round_().to(torch.int8)
    return x.reshape(n, h, page, d), scale.to(torch.float8_e8m0fnu)


def prepare(case, seed):
    c = case
    if c["op"] == "assign":
        return _prepare_assign(c, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.RandomState(seed + 1)
    dt = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dt)

    # a pool with a tenth more pages than the sequences need (an append's: than they could need), handed out in any order
    B, T, d = c["B"], c["T"], c["d"]
    new, seq = _lengths(c, seed)
    per = -(-c["ctx"] // c["page"])
    used = -(-seq // c["page"])
    most = B * per if c["op"] == "append" else int(used.sum())
    pool = most + most // 10 + 1
    numbers, table = host.permutation(pool), np.zeros((B, per), dtype=np.int32)
    table[np.arange(per)[None] < used[:, None]] = numbers[:used.sum()]
    s = dict(case=c, scale=1.0 / math.sqrt(d), table=torch.from_numpy(table).cuda(), seq=torch.from_numpy(seq.astype(np.int32)).cuda())
    s["new"] = torch.from_numpy(new.astype(np.int32)).cuda() if c["padded"] else None
    for x in "kv":
        s[x + "c"], s[x + "s"] = _held_cache(randn(pool, c["Hkv"], c["page"], d), c["block"], c["fmt"])
    # projections leave [B, T, heads, d]; the operators see it as [B, heads, T, d]
    s["q"] = randn(B, T, c["Hq"], d).transpose(1, 2)
    if c["op"] == "append":
        s["k"], s["v"] = randn(B, T, c["Hkv"], d).transpose(1, 2), randn(B, T, c["Hkv"], d).transpose(1, 2)
        s["tables"] = [_table(c["ctx"], d // 2)]
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------------
def _assign(table, seq, want, pool, page, T):
    """Table, lengths and pool are brought up to date in place; new tokens of every request and their places."""
    B, cols = table.shape
    n = pool.numel() - 2
    pages = lambda x: (x + page - 1) // page  # noqa: E731
    held = seq.long()
    want = want.long()
    grows = (want > held) & (want <= cols * page) & ((want - held <= T) | (T == 0))
    shrinks = (want >= 0) & (want < held)
    p0, p1 = pages(held), pages(want)
    free = pool[0].long()
    col = torch.arange(cols, device=table.device)[None]
    back = shrinks[:, None] & (col >= p1[:, None]) & (col < p0[:, None])
    n_back = back.sum()
    # the stack of free pages, what comes back on top of it, the last request's last page first; one place behind it for the rest
    stack = torch.cat([pool[2:], pool[:1]])
    rank = back.reshape(-1).cumsum(0) - 1
    stack.scatter_(0, torch.where(back.reshape(-1), free + n_back - 1 - rank, n), table.reshape(-1))
    need = torch.where(grows, p1 - p0, 0)
    granted = grows & ((need.cumsum(0) <= free + n_back) | (need == 0))
    taken = granted[:, None] & (col >= p0[:, None]) & (col < p1[:, None])
    rank = (taken.reshape(-1).cumsum(0) - 1).reshape(B, cols)
    table.copy_(torch.where(taken, stack[(free + n_back - 1 - rank).clamp(0, n)], table))
    left = free + n_back - taken.sum()
    at = torch.arange(n, device=table.device)
    pool[2:] = torch.where((at >= free) & (at < left), stack[:n], pool[2:])
    pool[0] = left
    n_new = torch.where(granted, want - held, 0)
    seq.copy_(torch.where(granted | shrinks, want, held))
    t = torch.arange(T, device=table.device)[None]
    p = held[:, None] + t
    slots = torch.gather(table.long(), 1, (p // page).clamp_max(cols - 1)) * page + p % page
    return n_new.int(), torch.where(t < n_new[:, None], slots, -1).int()


def _rotate(x, cos, sin, layout):
    """Pairs of dims turned: layout "halves" i and i + C / 2; "blocks" of one axis: the same."""
    r = x.shape[-1] // 2
    x0, x1 = x[..., :r], x[..., r:]
    return torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1)


def _places(s, T):
    """Positions of the T new tokens of every sequence, -1 behind its last one: [B, T]."""
    new = s["new"] if s["new"] is not None else torch.full_like(s["seq"], T)
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    return torch.where(t < new[:, None], s["seq"][:, None] - new[:, None] + t, -1), new


def _round8(x, fmt):
    return x.to(torch.float8_e4m3fn).float() if fmt == "e4m3" else torch.round(x)


def _store(cache, scale, x, s, new, block, fmt):
    """x [B, heads, T, d] in 32 bits into the cache, block by block: the blocks that new tokens of a sequence touch are formed whole and written back."""
    B, H, T, d = x.shape
    page = cache.shape[2]
    nb = (T + block - 2) // block + 1          # blocks that T tokens can touch
    held = (s["seq"] - new).long()
    first = held // block                      # of every sequence
    pos = (first[:, None] + torch.arange(nb, device=x.device))[:, :, None] * block + torch.arange(block, device=x.device)   # [B, nb, block]
    end = s["seq"].long()[:, None, None]
    is_new, is_old = (pos >= held[:, None, None]) & (pos < end), pos < held[:, None, None]
    live = is_new.any(-1)                      # [B, nb]
    at = pos[:, :, 0].clamp_max(s["table"].shape[1] * page - block)
    pg, row = torch.gather(s["table"].long(), 1, at // page), at % page
    rows = row[:, :, None] + torch.arange(block, device=x.device)
    codes = cache[pg[:, :, None], :, rows].float()                       # [B, nb, block, H, d]
    old = scale[pg, :, row // block].float()                             # [B, nb, H]
    fresh = torch.gather(x.transpose(1, 2), 1, (pos - held[:, None, None]).clamp(0, T - 1).reshape(B, -1)[:, :, None, None].expand(-1, -1, H, d)).reshape(B, nb, block, H, d)
    fresh = torch.where(is_new[..., None, None], fresh, 0.0)
    amax = fresh.abs().amax((2, 4))                                      # [B, nb, H]
    top, most = (1.75, 8) if fmt == "e4m3" else (1.984375, 6)            # the largest number is top 2^most
    m, e = torch.frexp(amax)                                             # amax = 2 m 2^(e - 1)
    need = torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e - 1 - most + (2 * m > top), -100))
    scl = torch.where((pos[:, :, 0] >= held[:, None])[..., None], need, torch.maximum(need, old))
    by = scl[:, :, None, :, None]
    codes = torch.where(is_old[..., None, None], _round8(codes * (old[:, :, None, :, None] / by), fmt), _round8(fresh / by, fmt))
    b, j, r = torch.nonzero((is_new | is_old) & live[..., None], as_tuple=True)
    cache.view(torch.uint8)[pg[b, j], :, rows[b, j, r]] = codes[b, j, r].to(cache.dtype).view(torch.uint8)
    b, j = torch.nonzero(live, as_tuple=True)
    scale.view(torch.uint8)[pg[b, j], :, row[b, j] // block] = scl[b, j].to(scale.dtype).view(torch.uint8)


def _values(cache, scale):
    """What a cache holds, in 32 bits."""
    n, h, page, d = cache.shape
    return (cache.float().reshape(n, h, scale.shape[2], -1, d) * scale.float()[..., None, None]).reshape(cache.shape)


def _attend(q, k, v, qpos, kpos, W, S, scale):
    """q [B, Hq, Lq, d]; qpos [B, Lq], kpos [B, Lk], negative: not there.  Queries that see nothing: zeros."""
    B, Hq, Lq, d = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    qf = q.float().reshape(B, Hkv, Hq // Hkv * Lq, d)
    s = (qf @ k.transpose(-1, -2)).reshape(B, Hkv, Hq // Hkv, Lq, Lk) * scale
    p_, j = qpos[:, :, None], kpos[:, None, :]
    seen = (j >= 0) & (p_ >= 0) & (j <= p_)
    if W:
        seen = seen & ((p_ - j < W) | (j < S))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    e = torch.exp(s - m)
    p = e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    o = p.reshape(B, Hkv, Hq // Hkv * Lq, Lk) @ v
    return o.reshape(B, Hq, Lq, v.shape[-1]).to(q.dtype)


def _plain(s):
    c = s["case"]
    place, new = _places(s, c["T"])
    if c["op"] == "attend":
        B, per = s["table"].shape
        at = torch.arange(per * c["page"], device="cuda")[None]
        at = torch.where(at < s["seq"][:, None], at, -1)
        gone = (at < 0)[:, None, :, None]
        tb = s["table"].long()
        k, v = (_values(x[tb].reshape(B * per, *x.shape[1:]), y[tb].reshape(B * per, *y.shape[1:])).reshape(B, per, c["Hkv"], c["page"], c["d"]).transpose(1, 2)
                .reshape(B, c["Hkv"], per * c["page"], c["d"]).masked_fill(gone, 0) for x, y in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        return _attend(s["q"], k, v, place, at, c["W"], c["S"], s["scale"])
    q, k = s["q"], s["k"].float()
    if c["rope"] != "none":
        cs = s["tables"][0][place.long().clamp_min(0)][:, None]                       # [B, 1, T, pairs, 2]
        lost = (place < 0)[:, None, :, None]
        cos, sin = cs[..., 0].masked_fill(lost, 1.0), cs[..., 1].masked_fill(lost, 0.0)
        q, k = _rotate(q.float(), cos, sin, c["rope"]).to(q.dtype), _rotate(k, cos, sin, c["rope"])
    _store(s["kc"], s["ks"], k, s, new, c["block"], c["fmt"])
    _store(s["vc"], s["vs"], s["v"].float(), s, new, c["block"], c["fmt"])
    return q


# ---- the package's operators ----------------------------------------------------------------------------------------------------
def _own(s):
    c = s["case"]
    from dl_templates_amd.paged_cache8 import paged8_append_, paged8_attention
    if c["op"] == "attend":
        return paged8_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["seq"], c["W"] or None, c["S"], s["scale"], s["new"])
    rope = None if c["rope"] == "none" else (None, s["tables"], c["rope"])
    return paged8_append_(s["kc"], s["vc"], s["ks"], s["vs"], s["k"], s["v"], s["table"], s["seq"], s["new"], rope, s["q"])


def _own_assign(table, seq, want, pool, page, T):
    from dl_templates_amd.page_pool import page_assign_
    return page_assign_(table, seq, want, pool, page, T or None)


def run(state):
    s = state
    c = s["case"]
    with torch.no_grad():
        if c["op"] == "assign":
            # a step, and the way back: requests grow and end, then take the lengths that they had before, so that a pass leaves the state as it was
            call = _own_assign if own else _assign
            n_new, slots = call(s["table"], s["seq"], s["want"], s["pool"], c["page"], c["T"])
            again = call(s["table"], s["seq"], s["held"], s["pool"], c["page"], 0)[0]
            return n_new, slots, again, s["table"], s["seq"], s["pool"]
        o = (_own if own else _plain)(s)
        if c["op"] == "attend":
            return o
        if c["fmt"] == "int8":
            # numbers of 8 bits times powers of two: exact in bfloat16
            return _values(s["kc"], s["ks"]).bfloat16(), _values(s["vc"], s["vs"]).bfloat16(), s["ks"], s["vs"], o
        return s["kc"], s["vc"], s["ks"], s["vs"], o


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def _seen(p, W, S):
    """Keys that a query at position p sees."""
    if not W or p < W:
        return p + 1
    return W + min(S, p + 1 - W)


def work(case):
    c = case
    if c["op"] == "assign":
        held, want = _requests(c)
        pages = lambda n: -(-n // c["page"])  # noqa: E731
        moved = int(np.abs(pages(want) - pages(held)).sum())
        # both ways: lengths in and out, counts, pages from and to the pool; the places of new tokens once
        return {"bytes": 2 * (16 * c["B"] + 8 * moved) + 4 * c["B"] * c["T"], "flops": 0}
    e, d = BYTES[c["dtype"]], c["d"]
    new, seq = _lengths(c)
    if c["op"] == "append":
        n = int(new.sum())
        turned = 6 * (d // 2) * n * (c["Hq"] + c["Hkv"]) if c["rope"] != "none" else 0
        return {"bytes": d * n * (2 * e * c["Hq"] + 2 * (e + 1) * c["Hkv"]) + 8 * c["B"], "flops": turned + 4 * d * n * c["Hkv"]}
    keys = pairs = 0
    for n, m in zip(new.tolist(), seq.tolist()):
        pairs += c["Hq"] * sum(_seen(p, c["W"], c["S"]) for p in range(m - n, m))
        lo = max(0, m - n - c["W"] + 1) if c["W"] else 0
        keys += (m - lo + min(c["S"], lo)) if n else 0
    return {"bytes": 2 * c["Hkv"] * keys * d + 2 * c["Hkv"] * keys // c["block"] + 2 * e * c["Hq"] * int(new.sum()) * d + 4 * keys // c["page"], "flops": 4 * pairs * d}


# ---- the definitions, in 64 bits --------------------------------------------------------------------------------------------------
def _exact_round(x, fmt):
    """The nearest number of the format, even ones at ties; x within the format's range."""
    if fmt == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(cache, scale, x, table, lo, hi, block, fmt):
    """One sequence: x [heads, hi - lo, d] in 64 bits at positions lo .. hi - 1; cache and scale in 64 bits, written."""
    page, top = cache.shape[2], 448.0 if fmt == "e4m3" else 127.0
    for j in range(lo // block, -(-hi // block) if hi > lo else lo // block):
        a, b = max(lo, j * block), min(hi, j * block + block)
        pg, row = int(table[j * block // page]), j * block % page
        new = x[:, a - lo:b - lo]
        big = new.abs().amax((1, 2))
        e = torch.ceil(torch.log2(big / top))
        e = torch.where(big > torch.exp2(e) * top, e + 1, torch.where(big <= torch.exp2(e - 1) * top, e - 1, e))
        s = torch.where(big > 0, torch.exp2(e), 2.0 ** -100)
        old = scale[pg, :, row // block]
        if a > j * block:
            s = torch.maximum(s, old)
            held = cache[pg, :, row:row + a - j * block]
            cache[pg, :, row:row + a - j * block] = _exact_round(held * (old / s)[:, None, None], fmt)
        scale[pg, :, row // block] = s
        cache[pg, :, row + a - j * block:row + b - j * block] = _exact_round(new / s[:, None, None], fmt)


def exact(case, seed):
    c = case
    if c["op"] == "assign":
        return None
    s = prepare(c, seed)
    seq = s["seq"].tolist()
    new = s["new"].tolist() if s["new"] is not None else [c["T"]] * c["B"]
    q = s["q"].double()
    table = s["table"].tolist()
    if c["op"] == "append":
        kc, vc, ks, vs = (s[x].float().double() for x in ("kc", "vc", "ks", "vs"))
        q, r = q.clone(), c["d"] // 2
        for b in range(c["B"]):
            p = torch.arange(seq[b] - new[b], seq[b], device="cuda")
            k, v, qb = s["k"][b, :, :new[b]].double(), s["v"][b, :, :new[b]].double(), q[b, :, :new[b]]
            if c["rope"] != "none":
                z = torch.view_as_complex(s["tables"][0][p].double())
                k, qb = (torch.cat([(t := torch.complex(x[..., :r].contiguous(), x[..., r:].contiguous()) * z).real, t.imag], -1) for x in (k, qb))
            q[b, :, :new[b]] = qb
            _exact_append(kc, ks, k, table[b], seq[b] - new[b], seq[b], c["block"], c["fmt"])
            _exact_append(vc, vs, v, table[b], seq[b] - new[b], seq[b], c["block"], c["fmt"])
        if c["fmt"] == "int8":
            kc, vc = (x * y.repeat_interleave(c["block"], 2)[..., None] for x, y in ((kc, ks), (vc, vs)))
        return kc, vc, ks, vs, q
    G = c["Hq"] // c["Hkv"]
    o = torch.zeros(c["B"], c["Hq"], c["T"], c["d"], dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        if not new[b]:
            continue
        at = s["table"][b, :-(-seq[b] // c["page"])].long()
        k, v = ((x[at].to(torch.float32).double() * y[at].float().double().repeat_interleave(c["block"], 2)[..., None]).transpose(0, 1).reshape(c["Hkv"], -1, c["d"])[:, :seq[b]]
                for x, y in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        p = torch.arange(seq[b] - new[b], seq[b], device="cuda")[:, None]
        j = torch.arange(seq[b], device="cuda")[None]
        hidden = (j > p) | ((p - j >= c["W"]) & (j >= c["S"])) if c["W"] else j > p
        for h in range(c["Hkv"]):
            score = torch.einsum("gid,jd->gij", q[b, h * G:(h + 1) * G, :new[b]], k[h]) * s["scale"]
            o[b, h * G:(h + 1) * G, :new[b]] = torch.einsum("gij,jd->gid", torch.softmax(score.masked_fill_(hidden, -math.inf), -1), v[h])
    return o
