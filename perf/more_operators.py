"""Operators beside the paged cache of many sequences, as cases that can be timed
and compared: attention whose scores are capped, biased by distance, or masked by
documents and prefixes (gd_kv_attn_scored), over single tokens and prompt chunks;
and the cache's pages: forking and freeing sequences (gd_kv_fork, gd_kv_release),
pages for the next rows with copies of shared ones (gd_kv_reserve,
gd_kv_copy_pages), and compaction (gd_kv_compact).

`run` makes the library's calls where `own` is true; else it computes the same
with elementary torch operations.  `exact` restates it apart from that: attention
in 64 bits, a sequence and a head at a time, pages on the host, one entry after
the other.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

NEVER = 2 ** 31 - 1              # the document of a padding row: no position is in it

# Attention geometries: the hybrid's, its 27B variant's, the dense 1.7B's.
HEADS = [dict(H=40, HKV=8, hd=128, gated=True), dict(H=24, HKV=4, hd=256, gated=True),
         dict(H=16, HKV=8, hd=128, gated=False)]
HYBRID, WIDE, DENSE = HEADS


def _attend(name, geo, **kw):
    c = dict(kind="attend", cache="f16", x="f16", B=1, rows=1, pos=0, page=16, window=0, sinks=0, cap=0.0, bias=False,
             doc=0, prefix=0)
    return dict(c, name=name, **geo) | kw


def _pages(name, kind, geo, **kw):
    c = dict(kind=kind, cache="f16", layers=1, n_seq=1, span=64, page=16, rows=1, shared=0, fill=0.6)
    return dict(c, name=name, HKV=geo["HKV"], hd=geo["hd"]) | kw


def listed():
    return [
        # One decoded token of one conversation with capped scores: the launch counts.
        _attend("cap_token", HYBRID, cache="i8", x="f32", pos=500, cap=50.0),
        # Serving with capped scores and a window: the next tokens of 64 conversations.
        _attend("cap_batch", WIDE, B=64, pos=12000, page=64, window=4096, sinks=4, cap=30.0),
        # Serving with a bias by distance: long contexts beside short ones, read whole.
        _attend("bias_batch", HYBRID, cache="i8", B=48, pos=8191, bias=True),
        # A chunk of documents packed one after the other, padding behind them.
        _attend("doc_prompt", HYBRID, rows=4096, doc=1500, cap=50.0),
        # Prompts whose first part (an image, a task) sees itself whole, beside each other.
        _attend("prefix_prompts", WIDE, cache="i8", x="f32", B=10, rows=400, pos=900, page=48, prefix=700, cap=50.0),
        # A later chunk of a long prompt, capped and biased, of a dense model.
        _attend("bias_prompt", DENSE, x="f32", rows=1021, pos=3003, page=20, bias=True, cap=20.0),
        # A conversation branches into four answers, and one is dropped.
        _pages("branch_one", "branch", HYBRID, n_seq=8, span=40, forks=4, drops=1),
        # A server's round: hundreds of branches of long shared prompts, hundreds end.
        _pages("branch_many", "branch", HYBRID, n_seq=1024, span=2048, forks=400, drops=300, shared=200),
        # A decoding step of 64 branches, whose shared last pages are copied in 16 layers.
        _pages("grow_tokens", "grow", HYBRID, cache="i8", layers=16, n_seq=64, span=512, shared=24),
        # Pages for prompts that join, in a large pool.
        _pages("grow_prompts", "grow", WIDE, layers=2, n_seq=200, span=160, page=64, rows=700, shared=60, fill=0.85),
        # A small cache closed up after conversations ended.
        _pages("compact_few", "compact", DENSE, cache="i8", layers=4, n_seq=5, span=30, page=32, fill=0.5),
        # A server's cache closed up, eight layers of it.
        _pages("compact_many", "compact", HYBRID, layers=8, n_seq=96, span=250, shared=20, fill=0.55),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "branch", "grow", "compact"])
    geo, cache = rng.choice(HEADS), rng.choice(["i8", "f16"])
    page = rng.choice([16, 16, 48, 64, 128] if cache == "i8" else [16, 16, 20, 64, 128])
    if kind == "attend":
        c = _attend(None, geo, cache=cache, x=rng.choice(["f16", "f32"]), page=page)
        shape = rng.choice(["token", "batch", "chunk", "ragged"])
        if shape in ("batch", "ragged"):
            c["B"] = _spread(rng, 2, 64)
        if shape in ("chunk", "ragged"):
            c["rows"] = _spread(rng, 2, max(3, 2048 // c["B"]))
        most = min(32768, 400000 // c["B"], 12000000 // (c["B"] * c["rows"]))
        c["pos"] = rng.choice([0, _spread(rng, 16, most)]) if c["rows"] > 1 else _spread(rng, 16, most)
        if rng.random() < 0.3:
            c["window"], c["sinks"] = _spread(rng, 32, 4096), rng.choice([0, 4, rng.randint(1, 64)])
        c["cap"] = rng.choice([0.0, 50.0, 30.0, round(_spread(rng, 50, 1000) / 10, 1)])
        c["bias"] = rng.random() < 0.4
        c["doc"] = _spread(rng, 2, 3000) if rng.random() < 0.35 else 0
        c["prefix"] = _spread(rng, 1, 2000) if rng.random() < 0.35 else 0
    else:
        c = _pages(None, kind, geo, cache=cache, page=page, fill=round(rng.uniform(0.2, 0.98), 2))
        c["n_seq"] = _spread(rng, 2, 1024 if kind == "branch" else 256)
        c["span"] = _spread(rng, 1, 2048 if kind == "branch" else 40000 // (c["n_seq"] * max(1, page // 16)) + 1)
        c["shared"] = rng.choice([0, _spread(rng, 1, c["n_seq"])])
        if kind == "branch":
            c["forks"], c["drops"] = _spread(rng, 1, max(1, c["n_seq"] // 2)), _spread(rng, 1, c["n_seq"])
        elif kind == "grow":
            c["rows"] = rng.choice([1, _spread(rng, 2, 1500)])
            c["span"] = max(c["span"], -(-c["rows"] // page))
        if kind != "branch":
            c["layers"] = _spread(rng, 1, max(1, min(16, 1500000 // (c["n_seq"] * c["span"] * page))))
    del c["name"]
    return c


def _rng(case, what):
    return random.Random("%s %s" % (what, sorted((k, v) for k, v in case.items() if k != "name")))


# ------------------------------------------------------------------ attention: shapes and inputs


def _lengths(case):
    """(first position, rows) of each sequence: the case's largest, the others shorter."""
    r = _rng(case, "lengths")
    one = lambda top: _spread(r, 1, top)  # noqa: E731
    seqs = [(case["pos"], case["rows"])]
    seqs += [(one(case["pos"] + 1) - 1, one(case["rows"])) for _ in range(case["B"] - 1)]
    r.shuffle(seqs)
    return seqs


def _masks(case):
    """Each row's document's first position, and each sequence's prefix."""
    r = _rng(case, "masks")
    first, prefix = [], []
    for p, n in _lengths(case):
        start = p - r.randint(0, min(p, case["doc"]))
        at = p + r.randint(0, case["doc"])                 # where the next document starts
        for t in range(p, p + n):
            if t >= at:
                start, at = t, t + _spread(r, 1, max(1, case["doc"]))
            first.append(start)
        for i in range(n // 50):                           # padding
            first[-1 - i] = NEVER
        prefix.append(r.choice([0, _spread(r, 1, max(1, case["prefix"])), case["prefix"]]) if len(prefix) else case["prefix"])
    return first, prefix


def _dt(case):
    return torch.float16 if case["x"] == "f16" else torch.float32


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _planes(case, n, pages, g):
    """n planes of a cache: f16 values, or codes and the bytes of their exponents; unit normal rows."""
    HKV, P, hd = case["HKV"], case["page"], case["hd"]
    half = lambda *z: torch.randn(z, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
    if case["cache"] == "f16":
        return [half(n, pages, P, HKV, hd)]
    codes = half(n, pages, HKV, P, hd).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
    return [codes, (127 - torch.randint(4, 7, (n, pages, HKV, P // 16), generator=g, device="cuda")).to(torch.uint8)]


def _attend_inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    seqs, dt = _lengths(case), _dt(case)
    B, P, H, hd = (case[k] for k in ("B", "page", "H", "hd"))
    N = sum(r for _, r in seqs)
    need = [-(-(p + r) // P) for p, r in seqs]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.zeros(B, max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    first, prefix = _masks(case)
    # Scores of a few units: what a cap is there for.
    s = dict(case=case, q=(normal(N, H, hd) * (4 if case["cap"] else 1.5)).to(dt), gate=normal(N, H, hd).to(dt), table=table,
             pos=_ints([p for p, _ in seqs]), row_start=_ints([sum(r for _, r in seqs[:i]) for i in range(B + 1)]),
             first=_ints(first), prefix=_ints(prefix),
             slope=torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda"))
    s["planes"] = _planes(case, 2, pages, g)
    s["kc"], s["vc"] = s["planes"][0]
    s["kx"], s["vx"] = s["planes"][-1]
    s["out"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------------------ pages: shapes and inputs


def _held(case):
    """Positions that each sequence holds, which sequence it shares its pages with (-1: none), and
    the rows that it goes on by (0: idle)."""
    r = _rng(case, "held")
    n, most = case["n_seq"], case["span"] * case["page"]
    room = most - (case["rows"] if case["kind"] == "grow" else 0)
    length = [max(0, room)] + [_spread(r, 1, max(1, room)) if room > 0 else 0 for _ in range(n - 1)]
    like, rows = [-1] * n, [1] * n
    sharers = r.sample(range(1, n), min(case["shared"], n - 1))
    prompts = [j for j in range(n) if j not in sharers][:8]
    for i in sharers:                                      # branches of a few prompts
        j = r.choice(prompts)
        like[i], length[i] = j, length[j] if r.random() < 0.7 else min(length[j], _spread(r, 1, max(1, length[j])))
    for i in range(n):
        if case["rows"] > 1:
            rows[i] = case["rows"] if i == 0 else _spread(r, 1, case["rows"])
        elif i and r.random() < 0.05:
            rows[i] = 0
    if case["kind"] == "branch":                           # slots without a sequence
        for i in range(1, n):
            if r.random() < 0.4 and i not in prompts:
                length[i], like[i] = 0, -1
    return length, like, rows


def _pool(case):
    """Pages in use at the start, and pages in all."""
    P = case["page"]
    length, like, rows = _held(case)
    used = 0
    for b, n in enumerate(length):
        used += -(-n // P) if like[b] < 0 else 0
    grow = sum(-(-r // P) + 1 for r in rows) if case["kind"] == "grow" and case["fill"] < 0.9 else 0
    return used, max(used + grow, math.ceil(used / case["fill"])) + 2


def _orders(case):
    """A branch case's forks (src, dst, positions) and drops (sequence, from, to)."""
    r = _rng(case, "orders")
    length, like, _ = _held(case)
    n = case["n_seq"]
    live = [i for i in range(n) if length[i]] or [0]
    src = live[:max(1, len(live) // 4)]
    free = [i for i in range(n) if i not in src]
    r.shuffle(free)
    forks = []
    for dst in free[:case["forks"]]:
        s = r.choice(src)
        forks.append((s, dst, length[s] if r.random() < 0.7 else _spread(r, 1, max(1, length[s]))))
    drops = []
    for i in r.sample(range(n), min(n, case["drops"])):
        how = r.random()
        top = max(1, length[i])
        # Most end, some go back to an earlier position, some leave what a window has passed.
        drops.append((i, 0, 0) if how < 0.7 else (i, 0, _spread(r, 1, top)) if how < 0.85 else (i, r.randint(0, top), NEVER))
    return forks, drops


def _pages_inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    length, like, rows = _held(case)
    P, n, span = case["page"], case["n_seq"], case["span"]
    pos, rows = [p if r else -1 for p, r in zip(length, rows)], [max(1, r) for r in rows]
    _, n_pages = _pool(case)
    order = np.random.RandomState(seed % 2 ** 32).permutation(n_pages)
    width = span + (1 if case["kind"] == "grow" else 0)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for b in sorted(range(n), key=lambda b: like[b] >= 0):
        k = -(-length[b] // P)
        if like[b] < 0:
            table[b, :k] = order[at:at + k]
            at += k
        else:
            table[b, :k] = table[like[b], :k]
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    # Counts and tables side by side, so that one copy sets both back.
    s = dict(case=case, n_pages=n_pages, start=_ints(np.concatenate([refs, table.ravel()])))
    s["book"] = s["start"].clone()
    s["refs"], s["table"] = s["book"][:n_pages], s["book"][n_pages:].view(n, width)
    if case["kind"] == "branch":
        forks, drops = _orders(case)
        s["fork"] = [_ints([f[i] for f in forks]) for i in range(3)]
        s["drop"] = [_ints([d[i] for d in drops]) for i in range(3)]
        return s
    s["pairs"] = torch.full((n if case["kind"] == "grow" else n_pages, 2), -1, dtype=torch.int32, device="cuda")
    if case["kind"] == "grow":
        s["pos"] = _ints(pos)
        s["row_start"] = _ints([sum(rows[:i]) for i in range(n + 1)])
        s["n_rows"], s["pos_out"] = sum(rows), torch.zeros_like(s["pos"])
        s["count"] = _ints([0])
    else:
        s["count"] = _ints([0, 0])
    s["planes"] = _planes(case, 2 * case["layers"], n_pages, g)
    return s


_ctx = None


def prepare(case, seed):
    s = _attend_inputs(case, seed) if case["kind"] == "attend" else _pages_inputs(case, seed)
    if own:
        s["calls"] = _calls(case, s)
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        for fn, args in s["calls"]:
            if fn(*args):
                raise RuntimeError(_ctx.lib.gd_last_error(_ctx.h).decode())
        if kind == "attend":
            return {"out": s["out"]}
    elif kind == "attend":
        return {"out": _attend_plain(s["case"], s)}
    else:
        s["book"].copy_(s["start"])
        {"branch": _branch_plain, "grow": _grow_plain, "compact": _compact_plain}[kind](s["case"], s)
    res = {"table": s["table"], "refs": s["refs"]}
    if kind == "branch":
        return res
    if kind == "grow":
        res["pos"] = s["pos_out"]
    return dict(res, pairs=s["pairs"], count=s["count"], planes=s["planes"])


# ------------------------------------------------------------------ the library's calls


def _calls(case, s):
    """The calls a program makes in a pass, with their arguments in hand."""
    import ctypes as C
    import gadeon_amd as ga
    global _ctx
    if _ctx is None:
        _ctx = ga.Context(0)
    lib, p, i8 = _ctx.lib, lambda t: t.data_ptr(), case["cache"] == "i8"
    dtype = ga.I8 if i8 else ga.F16

    def cache(planes, layer):
        (k, v), (kx, vx) = planes[0][2 * layer:2 * layer + 2], planes[-1][2 * layer:2 * layer + 2]
        return ga.KV(k=p(k), v=p(v), k_exp=p(kx) if i8 else None, v_exp=p(vx) if i8 else None, n_pages=k.shape[0], dtype=dtype,
                     n_head_kv=case["HKV"], head_dim=case["hd"], page_size=case["page"])

    if case["kind"] == "attend":
        B, N, H, hd = case["B"], s["q"].shape[0], case["H"], case["hd"]
        kv = cache(s["planes"], 0)
        seqs = ga.Seqs(n_rows=N, row_start=p(s["row_start"]) if case["rows"] > 1 else None, pos=p(s["pos"]), rope_shift=None,
                       page_table=p(s["table"]), n_seq=B, max_pages=s["table"].shape[1],
                       max_len=max(q + r for q, r in _lengths(case)))
        how = ga.Scores(cap=case["cap"], window=case["window"], n_sink=case["sinks"], slope=p(s["slope"]) if case["bias"] else None,
                        first=p(s["first"]) if case["doc"] else None, prefix=p(s["prefix"]) if case["prefix"] else None)
        s["keep"] = kv, seqs, how
        return [(lib.gd_kv_attn_scored, (_ctx.h, C.byref(kv), C.byref(seqs), p(s["q"]), H * hd, p(s["gate"]) if case["gated"] else None,
                                         H * hd, p(s["out"]), ga.F16 if case["x"] == "f16" else ga.F32, H, hd ** -0.5, C.byref(how)))]
    n, width = s["table"].shape
    pages = ga.KVPages(refs=p(s["refs"]), table=p(s["table"]), n_pages=s["n_pages"], n_seq=n, max_pages=width, page_size=case["page"])
    back = (lib.gd_copy, (_ctx.h, p(s["book"]), p(s["start"]), 4 * s["book"].numel()))
    s["keep"] = pages
    if case["kind"] == "branch":
        return [back, (lib.gd_kv_fork, (_ctx.h, C.byref(pages), *map(p, s["fork"]), s["fork"][0].numel())),
                (lib.gd_kv_release, (_ctx.h, C.byref(pages), *map(p, s["drop"]), s["drop"][0].numel()))]
    layers = (ga.KV * case["layers"])(*[cache(s["planes"], i) for i in range(case["layers"])])
    copy = (lib.gd_kv_copy_pages, (_ctx.h, layers, case["layers"], p(s["pairs"]), p(s["count"]), s["pairs"].shape[0]))
    if case["kind"] == "compact":
        return [back, (lib.gd_kv_compact, (_ctx.h, C.byref(pages), p(s["pairs"]), p(s["count"]))), copy]
    seqs = ga.Seqs(n_rows=s["n_rows"], row_start=None if case["rows"] == 1 else p(s["row_start"]), pos=p(s["pos"]), rope_shift=None,
                   page_table=p(s["table"]), n_seq=n, max_pages=width, max_len=0)
    s["keep"] = pages, seqs
    return [back, (lib.gd_kv_reserve, (_ctx.h, C.byref(pages), C.byref(seqs), p(s["pairs"]), p(s["count"]), p(s["pos_out"]))), copy]


# ------------------------------------------------------------------ attention in elementary torch operations


def _cached(case, s, b, p):
    """Cached keys and values at positions p of sequences b, [..][HKV][hd] in 32 bits."""
    P = case["page"]
    page, slot = s["table"].long()[b, p // P], p % P
    if case["cache"] == "f16":
        return [s[c][page, slot].float() for c in ("kc", "vc")]
    return [s[c][page, :, slot].float() * torch.exp2(s[x][page, :, slot // 16].float() - 127)[..., None]
            for c, x in (("kc", "kx"), ("vc", "vx"))]


def _attend_plain(case, s):
    B, HKV, hd, W, N = case["B"], case["HKV"], case["hd"], case["window"], s["q"].shape[0]
    R, L = case["rows"], max(p + r for p, r in _lengths(case))
    row = torch.arange(N, device="cuda")
    b = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    i = row - s["row_start"][b]
    padded = torch.zeros(B, R, *s["q"].shape[1:], device="cuda")
    padded[b, i] = s["q"].float()
    Q = padded.view(B, R, HKV, -1, hd).transpose(1, 2).reshape(B, HKV, -1, hd)
    t = torch.arange(L, device="cuda")
    length = (s["pos"] + s["row_start"][1:] - s["row_start"][:-1])[:, None]
    K, V = _cached(case, s, torch.arange(B, device="cuda")[:, None], torch.minimum(t, length - 1))
    S = torch.matmul(Q, K.permute(0, 2, 3, 1).contiguous()).mul_(hd ** -0.5).view(B, HKV, R, -1, L)
    if case["cap"]:
        S = S.div_(case["cap"]).tanh_().mul_(case["cap"])
    at = s["pos"][:, None, None] + torch.arange(R, device="cuda")[:, None]
    if case["bias"]:
        S -= s["slope"].view(HKV, 1, -1, 1) * (at - t).abs().float()[:, None, :, None]
    seen = t <= at
    if W:
        seen &= (t > at - W) | (t < case["sinks"])
    if case["prefix"]:
        seen |= t < torch.minimum(s["prefix"][:, None], length)[:, None]
    if case["doc"]:
        first = torch.zeros(B, R, dtype=torch.int32, device="cuda")
        first[b, i] = s["first"]
        seen &= t >= first[:, :, None]
    S = S.masked_fill_(~seen[:, None, :, None], -math.inf)
    S = S.sub_(S.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    S = S.div_(S.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, HKV, -1, L)
    O = torch.matmul(S, V.transpose(1, 2).contiguous())
    out = O.view(B, HKV, R, -1, hd).transpose(1, 2).reshape(B, R, -1, hd)[b, i]
    if case["gated"]:
        out = out * (1 / (1 + torch.exp(-s["gate"].float())))
    return out.to(_dt(case))


# ------------------------------------------------------------------ pages in elementary torch operations


def _count(refs, entries, by):
    e = entries[entries >= 0].long()
    refs.index_add_(0, e, torch.full_like(e, by, dtype=torch.int32))


def _branch_plain(case, s):
    P, (src, dst, length) = case["page"], s["fork"]
    e = torch.arange(s["table"].shape[1], device="cuda")
    new = torch.where(e * P < length[:, None], s["table"][src.long()], -1)
    _count(s["refs"], s["table"][dst.long()], -1)
    _count(s["refs"], new, 1)
    s["table"][dst.long()] = new
    seq, a, z = s["drop"]
    old = s["table"][seq.long()]
    keep = ((e + 1) * P > a[:, None]) & (e * P < z[:, None])
    _count(s["refs"], torch.where(keep, -1, old), -1)
    s["table"][seq.long()] = torch.where(keep, old, -1)


def _copy_plain(s, src, dst):
    for t in s["planes"]:
        for plane in t:
            plane[dst] = plane[src]


def _grow_plain(case, s):
    table, refs, P = s["table"], s["refs"], case["page"]
    pos, rows = s["pos"], s["row_start"][1:] - s["row_start"][:-1]
    e = torch.arange(table.shape[1], device="cuda")
    # Entries of the new rows, sequence by sequence, and the pages they name.
    b, k = ((pos[:, None] >= 0) & ((e + 1) * P > pos[:, None]) & (e * P < (pos + rows)[:, None])).nonzero(as_tuple=True)
    page = table[b, k].long()
    there = page >= 0
    page0 = page.clamp(min=0)
    shared = there & (refs[page0] > 1)
    # Of the entries that share a page the last keeps it, if no other than these do.
    uses = torch.zeros_like(refs).index_add_(0, page0, shared.int())
    nth = torch.arange(len(b), device="cuda").int()
    last = torch.full_like(refs, -1).scatter_reduce_(0, page0, torch.where(shared, nth, -1), "amax")
    keeps = shared & (uses[page0] == refs[page0]) & (last[page0] == nth)
    need = ~there | (shared & ~keeps)
    free = (refs == 0).nonzero()[:, 0]
    rank = need.int().cumsum(0)
    touched = torch.zeros_like(pos).index_add_(0, b, (need | keeps).int()) > 0
    upto = torch.zeros_like(pos).index_add_(0, b, need.int()).cumsum(0)
    granted = ~touched | (upto <= len(free))
    s["pos_out"].copy_(torch.where(granted, pos, -1))
    take = need & granted[b]
    new = free[(rank[take] - 1).long()]
    copied = (shared & (k * P < pos[b]))[take]
    _count(refs, torch.where(shared, page, -1)[take], -1)
    refs[new] = 1
    table[b[take], k[take]] = new.int()
    src, dst = page[take][copied], new[copied]
    s["count"].fill_(len(src))
    s["pairs"][:len(src)] = torch.stack([src, dst], 1).int()
    _copy_plain(s, src, dst)


def _compact_plain(case, s):
    refs, table = s["refs"], s["table"]
    n = int((refs > 0).sum())
    dst = (refs[:n] == 0).nonzero()[:, 0]
    src = (refs[n:] > 0).nonzero()[:, 0].flip(0) + n
    to = torch.arange(len(refs), device="cuda").int()
    to[src] = dst.int()
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    s["count"].copy_(_ints([len(src), n]))
    s["pairs"][:len(src)] = torch.stack([src, dst], 1).int()
    _copy_plain(s, src, dst)


# ------------------------------------------------------------------ bytes and operations


def _page_bytes(case):
    """Of both planes of a page in one layer."""
    return 2 * case["page"] * case["HKV"] * (case["hd"] * 2 if case["cache"] == "f16" else case["hd"] + 1 / 16)


def work(case):
    if case["kind"] == "attend":
        return _attend_work(case)
    P, n = case["page"], case["n_seq"]
    length, like, rows = _held(case)
    used, n_pages = _pool(case)
    if case["kind"] == "branch":
        # Setting back; then rows of the table in and out, and the counts of their pages.
        forks, drops = _orders(case)
        moved = sum(-(-f[2] // P) + -(-length[f[1]] // P) for f in forks) + sum(-(-length[d[0]] // P) for d in drops)
        return {"bytes": 8 * (n_pages + n * case["span"]) + 4 * case["span"] * (3 * len(forks) + 2 * len(drops)) + 8 * moved, "flops": 0}
    back = 8 * (n_pages + n * (case["span"] + (case["kind"] == "grow")))
    if case["kind"] == "grow":
        copies = sum(1 for b in range(n) if like[b] >= 0 and rows[b] and length[b] % P)
        touched = sum(-(-(length[b] + r) // P) - length[b] // P for b, r in enumerate(rows) if r)
        return {"bytes": back + 4 * n_pages + 8 * touched + 2 * copies * case["layers"] * _page_bytes(case), "flops": 0}
    moves = round(used * (1 - used / n_pages))             # pages in use lie anywhere
    return {"bytes": back + 4 * n_pages + 4 * n * case["span"] + 8 * moves + 2 * moves * case["layers"] * _page_bytes(case), "flops": 0}


def _seen(case, p, n, i, first, prefix, t):
    """Which positions t row i sees, of a sequence's n rows from position p on."""
    at = p + i
    seen = t <= at
    if case["window"]:
        seen = seen & ((t > at - case["window"]) | (t < case["sinks"]))
    if case["prefix"]:
        seen = seen | (t < min(prefix, p + n))
    return seen & (t >= first) if case["doc"] else seen


def _attend_work(case):
    H, HKV, hd = case["H"], case["HKV"], case["hd"]
    x, c = 2 if case["x"] == "f16" else 4, 2 if case["cache"] == "f16" else 1 + 1 / (16 * hd)
    first, prefix = _masks(case)
    keys = pairs = N = 0
    for b, (p, n) in enumerate(_lengths(case)):
        t = np.arange(p + n)
        union = np.zeros(p + n, bool)
        for i in range(n):
            seen = _seen(case, p, n, i, first[N + i], prefix[b], t)
            union |= seen
            pairs += int(seen.sum())
        keys += int(union.sum())
        N += n
    return {"bytes": keys * 2 * HKV * hd * c + N * H * hd * x * (3 if case["gated"] else 2), "flops": 4 * pairs * H * hd}


# ------------------------------------------------------------------ apart from the plain forms


def _sequence(case, s, which, b, length):
    """Cached rows 0 .. length-1 of sequence b in 64 bits, [length][HKV][hd]."""
    P, pages = case["page"], s["table"][b, :-(-length // case["page"])].long()
    c = s[which + "c"][pages].double()
    if case["cache"] == "i8":
        c = c.view(len(pages), case["HKV"], P // 16, 16, case["hd"]) * 2.0 ** (s[which + "x"][pages].double() - 127)[..., None, None]
        c = c.view(len(pages), case["HKV"], P, case["hd"]).transpose(1, 2)
    return c.reshape(len(pages) * P, case["HKV"], case["hd"])[:length]


def _attend_exact(case, seed):
    s, (first, prefix) = _attend_inputs(case, seed), _masks(case)
    G, N, outs = case["H"] // case["HKV"], 0, []
    for b, (p, n) in enumerate(_lengths(case)):
        q, gate = s["q"][N:N + n].double(), s["gate"][N:N + n].double()
        K, V = (_sequence(case, s, c, b, p + n) for c in "kv")
        t, i = torch.arange(p + n, device="cuda"), torch.arange(n, device="cuda")[:, None]
        seen = _seen(case, p, n, i, _ints(first[N:N + n])[:, None], prefix[b], t)
        some = seen.any(1, keepdim=True)
        out = torch.empty_like(q)
        for h in range(case["H"]):
            S = q[:, h] @ K[:, h // G].T / math.sqrt(case["hd"])
            if case["cap"]:
                S = case["cap"] * torch.tanh(S / case["cap"])
            if case["bias"]:
                S = S - s["slope"][h].double() * (p + i - t).abs()
            w = torch.softmax(S.masked_fill(~seen & some, -math.inf), -1)
            out[:, h] = torch.where(some, w @ V[:, h // G], 0.0)
        outs.append(out * torch.sigmoid(gate) if case["gated"] else out)
        N += n
    return {"out": torch.cat(outs)}


def exact(case, seed):
    if case["kind"] == "attend":
        return _attend_exact(case, seed)
    s, P = _pages_inputs(case, seed), case["page"]
    table, refs = s["table"].cpu().numpy().copy(), s["refs"].cpu().numpy().copy()
    pairs = []
    if case["kind"] == "branch":
        before = table.copy()
        for src, dst, n in zip(*(v.tolist() for v in s["fork"])):
            table[dst] = -1
            table[dst, :-(-n // P)] = before[src, :-(-n // P)]
        for seq, a, z in zip(*(v.tolist() for v in s["drop"])):
            table[seq, :a // P] = -1
            table[seq, -(-z // P):] = -1
        refs = np.bincount(table[table >= 0], minlength=len(refs))
        return {"table": _ints(table), "refs": _ints(refs)}
    if case["kind"] == "grow":
        pos, rows = s["pos"].tolist(), np.diff(s["row_start"].cpu().numpy())
        free, pos_out, short = np.flatnonzero(refs == 0).tolist(), list(pos), False
        for b, p in enumerate(pos):
            entries = range(p // P, -(-(p + int(rows[b])) // P)) if p >= 0 and rows[b] else ()
            needs = [e for e in entries if table[b, e] < 0 or refs[table[b, e]] > 1]
            kept = any(table[b, e] >= 0 and s["refs"][table[b, e]] > 1 and refs[table[b, e]] == 1 for e in entries)
            short = short or len(needs) > len(free)
            if short and (needs or kept):
                pos_out[b] = -1
                continue
            for e in needs:
                old, new = table[b, e], free.pop(0)
                if old >= 0:
                    refs[old] -= 1
                    if e * P < p:
                        pairs.append((int(old), new))
                table[b, e], refs[new] = new, 1
        res, count = {"pos": _ints(pos_out)}, [len(pairs)]
    else:
        used = int((refs > 0).sum())
        low, high = 0, len(refs) - 1
        to = {}
        while True:
            while low < len(refs) and refs[low]:
                low += 1
            while high >= 0 and not refs[high]:
                high -= 1
            if low >= high:
                break
            refs[low], refs[high] = refs[high], 0
            to[high] = low
            pairs.append((high, low))
        table = np.array([[to.get(v, v) for v in row] for row in table.tolist()])
        res, count = {}, [len(pairs), used]
    s["pairs"][:len(pairs)] = _ints(pairs).view(-1, 2)
    for t in s["planes"]:
        for src, dst in pairs:
            t[:, dst] = t[:, src]
    planes = [t.double() if t.dtype == torch.float16 else t for t in s["planes"]]
    return {"table": _ints(table), "refs": _ints(refs), **res, "pairs": s["pairs"], "count": _ints(count), "planes": planes}
