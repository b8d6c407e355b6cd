"""The paged-cache operators for many sequences, as cases that can be timed and
compared: appending keys and values with the rotation on the way
(gd_kv_append_rope), attention over a cache of 8-bit values, and attention with a
sliding window and sinks (gd_kv_attn), each over single tokens of many
sequences and over prompt chunks.

`run` makes the library's calls where `own` is true; else it computes the same
with elementary torch operations, all sequences at once over padded keys.
`exact` restates it in 64 bits, a sequence and a kv head at a time.
"""
from __future__ import annotations

import math
import random

import torch

own = False

I8_RANGE = 65024.0               # 127 * 2^9, the largest value of the 8-bit cache

# Attention geometries: the hybrid's, its 27B variant's, the dense 1.7B's.
HEADS = [dict(H=40, HKV=8, hd=128, n_rot=64, base=1e7, gated=True),
         dict(H=24, HKV=4, hd=256, n_rot=64, base=1e7, gated=True),
         dict(H=16, HKV=8, hd=128, n_rot=128, base=1e6, gated=False)]
HYBRID, WIDE, DENSE = HEADS


def _case(name, kind, geo, **kw):
    c = dict(kind=kind, cache="i8", x="f16", B=1, rows=1, pos=0, page=16, window=0, sinks=0)
    return dict(c, name=name, **geo) | kw


def listed():
    return [
        # One decoded token of one conversation: the launch counts.
        _case("append_token", "append", HYBRID, x="f32", pos=700),
        # The prompts of a dozen conversations, joining at odd places of their blocks.
        _case("append_prompts", "append", WIDE, B=12, rows=512, pos=2000),
        # A prompt chunk into the f16 cache of the dense stack.
        _case("append_chunk", "append", DENSE, cache="f16", x="f32", rows=1000, pos=3001, page=24),
        # A short conversation's next token.
        _case("kv8_token", "attend", HYBRID, x="f32", pos=330),
        # One token at a long context.
        _case("kv8_long_token", "attend", WIDE, x="f32", pos=32767),
        # Serving: the next tokens of 64 conversations of all lengths.
        _case("kv8_batch", "attend", HYBRID, B=64, pos=8191, page=64),
        # A later chunk of a long prompt.
        _case("kv8_prompt", "attend", HYBRID, rows=512, pos=3584),
        # Prompt chunks beside each other, short ones among them.
        _case("kv8_mixed", "attend", WIDE, x="f32", B=20, rows=200, pos=5000, page=48),
        # Serving under a window: far positions, few visible keys.
        _case("window_token", "attend", DENSE, cache="f16", x="f32", B=32, pos=16000, window=1024, sinks=4),
        # A whole long prompt under a window.
        _case("window_prompt", "attend", HYBRID, cache="f16", rows=4096, window=1024, sinks=4),
        # Ragged chunks under a window that ends inside pages.
        _case("window_ragged", "attend", WIDE, cache="f16", x="f32", B=6, rows=333, pos=1500, page=20, window=400,
              sinks=17),
        # A serving step of an attention layer: append, then attend.
        _case("serve_step", "step", HYBRID, B=32, pos=3000),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "step"])
    c = dict(kind=kind, cache=rng.choice(["i8", "f16"]), x=rng.choice(["f16", "f32"]), B=1, rows=1, window=0,
             sinks=0, **rng.choice(HEADS))
    c["page"] = rng.choice([16, 16, 48, 64, 128] if c["cache"] == "i8" else [16, 16, 20, 64, 128])
    shape = rng.choice(["token", "batch", "chunk", "ragged"])
    if shape in ("batch", "ragged"):
        c["B"] = _spread(rng, 2, 64)
    if shape in ("chunk", "ragged"):
        c["rows"] = _spread(rng, 2, max(3, 2048 // c["B"]))
    most = min(32768, 250000 // c["B"], 3000000 // (c["B"] * c["rows"]))
    c["pos"] = rng.choice([0, _spread(rng, 16, most)]) if c["rows"] > 1 else _spread(rng, 16, most)
    if kind != "append" and (c["cache"] == "f16" or rng.random() < 0.3):
        c["window"], c["sinks"] = _spread(rng, 32, 4096), rng.choice([0, 1, 4, rng.randint(2, 64)])
    return c


# ------------------------------------------------------------------ shapes and inputs


def _lengths(case):
    """(first position, rows) of each sequence: the case's largest, the others shorter."""
    r = random.Random("%d %d %d" % (case["B"], case["rows"], case["pos"]))
    one = lambda top: _spread(r, 1, top)  # noqa: E731
    seqs = [(case["pos"], case["rows"])]
    seqs += [(one(case["pos"] + 1) - 1, one(case["rows"])) for _ in range(case["B"] - 1)]
    r.shuffle(seqs)
    return seqs


def _dt(case):
    return torch.float16 if case["x"] == "f16" else torch.float32


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    seqs, dt = _lengths(case), _dt(case)
    B, P, H, HKV, hd = (case[k] for k in ("B", "page", "H", "HKV", "hd"))
    N = sum(r for _, r in seqs)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    sums = lambda v: ints([sum(v[:i]) for i in range(len(v) + 1)])  # noqa: E731
    normal = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)  # noqa: E731
    need = [-(-(p + r) // P) for p, r in seqs]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.zeros(B, max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(q=normal(N, H, hd), k=normal(N, HKV, hd), v=normal(N, HKV, hd), gate=normal(N, H, hd), table=table,
             pos=ints([p for p, _ in seqs]), row_start=sums([r for _, r in seqs]))
    # What is read back of an append: the blocks of 16 positions that it touched.
    back = [(p // 16 * 16, p % 16 + r) for p, r in seqs]
    s["back_pos"], s["back_start"] = ints([p for p, _ in back]), sums([r for _, r in back])
    s["back"] = [torch.zeros(sum(r for _, r in back), HKV, hd, dtype=torch.float16, device="cuda") for _ in "kv"]
    half = lambda *z: torch.randn(z, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
    if case["cache"] == "f16":
        s["kc"], s["vc"] = half(pages, P, HKV, hd), half(pages, P, HKV, hd)
    else:
        # Unit normal rows: codes of up to 127 at steps of 2^-6 .. 2^-4.
        for c in "kv":
            s[c + "c"] = half(pages, HKV, P, hd).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
            s[c + "x"] = (127 - torch.randint(4, 7, (pages, HKV, P // 16), generator=g, device="cuda")).to(torch.uint8)
    s["out"], s["q_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["q"])
    return s


_ctx = None


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["calls"] = _calls(case, s)
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------ the library's calls


def _calls(case, s):
    """The calls a program makes in a pass, with their arguments in hand."""
    import ctypes as C
    import gadeon_amd as ga
    global _ctx
    if _ctx is None:
        _ctx = ga.Context(0)
    B, N, H, HKV, hd = case["B"], s["q"].shape[0], case["H"], case["HKV"], case["hd"]
    i8 = case["cache"] == "i8"
    x = ga.F16 if case["x"] == "f16" else ga.F32
    kv = ga.KV(k=s["kc"].data_ptr(), v=s["vc"].data_ptr(), k_exp=s["kx"].data_ptr() if i8 else None,
               v_exp=s["vx"].data_ptr() if i8 else None, n_pages=s["kc"].shape[0], dtype=ga.I8 if i8 else ga.F16,
               n_head_kv=HKV, head_dim=hd, page_size=case["page"])
    most = max(p + r for p, r in _lengths(case))

    def seqs(start, pos, rows):
        return ga.Seqs(n_rows=rows, row_start=start.data_ptr() if rows != B else None, pos=pos.data_ptr(),
                       rope_shift=None, page_table=s["table"].data_ptr(), n_seq=B, max_pages=s["table"].shape[1],
                       max_len=most)

    new = seqs(s["row_start"], s["pos"], N)
    back = seqs(s["back_start"], s["back_pos"], s["back"][0].shape[0])
    p = lambda t: t.data_ptr()  # noqa: E731
    q = s["q_out"] if case["kind"] == "step" else s["q"]
    append = (_ctx.lib.gd_kv_append_rope, (_ctx.h, C.byref(kv), C.byref(new), p(s["q"]), H * hd, p(s["q_out"]), H,
                                           p(s["k"]), HKV * hd, p(s["v"]), HKV * hd, x, case["n_rot"], case["base"]))
    read = (_ctx.lib.gd_kv_read, (_ctx.h, C.byref(kv), C.byref(back), p(s["back"][0]), p(s["back"][1]), ga.F16))
    attend = (_ctx.lib.gd_kv_attn, (_ctx.h, C.byref(kv), C.byref(new), p(q), H * hd,
                                    p(s["gate"]) if case["gated"] else None, H * hd, p(s["out"]), x, H, hd ** -0.5,
                                    case["window"], case["sinks"]))
    return {"append": [append, read], "attend": [attend], "step": [append, attend, read]}[case["kind"]]


def _run_own(s):
    for fn, args in s["calls"]:
        if fn(*args):
            raise RuntimeError(_ctx.lib.gd_last_error(_ctx.h).decode())
    kind = s["case"]["kind"]
    res = {} if kind == "attend" else {"q": s["q_out"], "k": s["back"][0], "v": s["back"][1]}
    return res if kind == "append" else dict(res, out=s["out"])


# ------------------------------------------------------------------ in elementary torch operations


def _rows(start, pos, n):
    """Sequence, index in it and position of each of n rows."""
    r = torch.arange(n, device="cuda")
    b = torch.searchsorted(start[1:].long(), r, right=True)
    i = r - start[b]
    return b, i, pos[b] + i


def _rotate(x, p, case):
    """x [N][heads][hd] turned to positions p, in 64 bits (angles of far positions, codes next to a border)."""
    h = case["n_rot"] // 2
    ang = p.double()[:, None] * case["base"] ** (-torch.arange(h, device="cuda").double() / h)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b, rest = x[..., :h].double(), x[..., h:2 * h].double(), x[..., 2 * h:].double()
    return torch.cat([a * c - b * s, a * s + b * c, rest], -1)


def _append_i8(case, s, x, codes, exps, b, p):
    """x [N][HKV][hd] in 64 bits -> codes [pages][HKV][P][hd] and exponents [pages][HKV][P/16]."""
    B, P, N = case["B"], case["page"], x.shape[0]
    start, pos = s["row_start"].long(), s["pos"].long()
    first = pos // 16                                      # each sequence's first block, and blocks
    count = (pos + start[1:] - start[:-1] + 15) // 16 - first
    ends = count.cumsum(0)
    blocks = N // 16 + 2 * B                               # at least as many as there are
    blk = (ends - count)[b] + p // 16 - first[b]           # block of each row
    u = torch.arange(blocks, device="cuda")
    ub = torch.searchsorted(ends, u, right=True).clamp(max=B - 1)
    there = u < ends[-1]
    ul = first[ub] + u - (ends - count)[ub]                # its place in the sequence
    page = s["table"].long()[ub, (ul * 16 // P).clamp(max=s["table"].shape[1] - 1)]
    slot = ul * 16 % P
    old_rows = torch.where(u == (ends - count)[ub], pos[ub] % 16, 0)    # rows of it that were there
    new = torch.zeros(blocks, 16, *x.shape[1:], dtype=x.dtype, device="cuda")
    new[blk, p % 16] = x
    new.clamp_(-I8_RANGE, I8_RANGE)
    m, e = torch.frexp(new.abs().amax((1, 3)))             # m in [0.5, 1): 127 2^e holds m 2^x
    e = torch.where(m <= 127 / 128, e - 7, e - 6).clamp(-24, 9)
    e = torch.where(m == 0, -24, e)
    e_old = exps[page, :, slot // 16].int() - 127
    had = (old_rows > 0)[:, None]
    e_new = torch.where(had, torch.maximum(e, e_old), e)
    at = slot[:, None] + torch.arange(16, device="cuda")
    old = codes[page[:, None], :, at].double()             # [blocks][16][HKV][hd]
    old = old * torch.where(had, torch.exp2((e_old - e_new).double()), 0)[:, None, :, None]
    is_old = (torch.arange(16, device="cuda") < old_rows[:, None])[:, :, None, None]
    c = torch.where(is_old, old, new * torch.exp2(-e_new.double())[:, None, :, None]).round()
    is_new = torch.zeros(blocks, 16, dtype=torch.bool, device="cuda")
    is_new[blk, p % 16] = True
    keep = (is_new | is_old[:, :, 0, 0]) & there[:, None]
    ku, ki = keep.nonzero(as_tuple=True)
    codes[page[ku], :, at[ku, ki]] = c[ku, ki].to(torch.int8)
    exps[page[there], :, (slot // 16)[there]] = (e_new + 127)[there].to(torch.uint8)


def _append_plain(case, s):
    N, P = s["q"].shape[0], case["page"]
    b, _, p = _rows(s["row_start"], s["pos"], N)
    q, k = _rotate(s["q"], p, case), _rotate(s["k"], p, case)
    if case["cache"] == "i8":
        _append_i8(case, s, k, s["kc"], s["kx"], b, p)
        _append_i8(case, s, s["v"].double(), s["vc"], s["vx"], b, p)
    else:
        page = s["table"].long()[b, p // P]
        s["kc"][page, p % P] = k.float().clamp(-65504, 65504).half()
        s["vc"][page, p % P] = s["v"].float().clamp(-65504, 65504).half()
    return q.to(_dt(case))


def _cached(case, s, b, p):
    """Cached keys and values at positions p of sequences b, [..][HKV][hd] in 32 bits."""
    P = case["page"]
    page, slot = s["table"].long()[b, p // P], p % P
    if case["cache"] == "f16":
        return [s[c][page, slot].float() for c in ("kc", "vc")]
    return [s[c][page, :, slot].float() * torch.exp2(s[x][page, :, slot // 16].float() - 127)[..., None]
            for c, x in (("kc", "kx"), ("vc", "vx"))]


def _attend_plain(case, s, q):
    B, HKV, hd, W = case["B"], case["HKV"], case["hd"], case["window"]
    R, L, N = case["rows"], max(p + r for p, r in _lengths(case)), q.shape[0]
    b, i, p = _rows(s["row_start"], s["pos"], N)
    padded = torch.zeros(B, R, *q.shape[1:], device="cuda")
    padded[b, i] = q.float()
    Q = padded.view(B, R, HKV, -1, hd).transpose(1, 2).reshape(B, HKV, -1, hd)
    t = torch.arange(L, device="cuda")
    length = s["pos"] + s["row_start"][1:] - s["row_start"][:-1]
    K, V = _cached(case, s, torch.arange(B, device="cuda")[:, None], torch.minimum(t, length[:, None] - 1))
    S = torch.matmul(Q, K.permute(0, 2, 3, 1).contiguous()).mul_(hd ** -0.5)
    at = s["pos"][:, None, None] + torch.arange(R, device="cuda")[:, None]
    seen = t <= at
    if W:
        seen &= (t > at - W) | (t < case["sinks"])
    S = S.view(B, HKV, R, -1, L).masked_fill_(~seen[:, None, :, None], -math.inf)
    S = S.sub_(S.amax(-1, keepdim=True)).exp_()
    S = S.div_(S.sum(-1, keepdim=True)).view(B, HKV, -1, L)
    O = torch.matmul(S, V.transpose(1, 2).contiguous())
    out = O.view(B, HKV, R, -1, hd).transpose(1, 2).reshape(B, R, -1, hd)[b, i]
    if case["gated"]:
        out = out * (1 / (1 + torch.exp(-s["gate"].float())))
    return out.to(_dt(case))


def _run_plain(s):
    case, res, q = s["case"], {}, s["q"]
    if case["kind"] != "attend":
        q = _append_plain(case, s)
        b, _, p = _rows(s["back_start"], s["back_pos"], s["back"][0].shape[0])
        k, v = _cached(case, s, b, p)
        res = {"q": q, "k": k.half(), "v": v.half()}
    return res if case["kind"] == "append" else dict(res, out=_attend_plain(case, s, q))


# ------------------------------------------------------------------ bytes and operations


def work(case):
    seqs, H, HKV, hd, W = _lengths(case), case["H"], case["HKV"], case["hd"], case["window"]
    x, c = 2 if case["x"] == "f16" else 4, 2 if case["cache"] == "f16" else 1 + 1 / (16 * hd)
    N, row = sum(r for _, r in seqs), HKV * hd * 2          # elements of a position's key and value
    nbytes = flops = 0
    if case["kind"] != "attend":
        # Rows in, queries in and out, cache rows out; then the touched blocks read back as f16.
        back = sum(p % 16 + r for p, r in seqs)
        nbytes += N * (row * (x + c) + 2 * H * hd * x) + back * row * (c + 2)
        flops += 3 * N * (H + HKV) * case["n_rot"]
    if case["kind"] != "append":
        keys = pairs = 0
        for p, r in seqs:
            low = max(0, p - W + 1) if W else 0              # first key of the first row's window
            sinks = min(case["sinks"], low)
            keys += p + r - low + sinks
            for n in (range(p + 1, p + r + 1) if W else ()):
                pairs += min(n, W + min(case["sinks"], max(0, n - W)))
            pairs += 0 if W else r * p + r * (r + 1) // 2
        nbytes += keys * row * c + N * H * hd * x * (3 if case["gated"] else 2)
        flops += 4 * pairs * H * hd
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ in 64 bits


def _turned(x, first, case):
    """Rows of one sequence from position `first`, as complex turns of the rotated pairs."""
    h = case["n_rot"] // 2
    p = torch.arange(first, first + x.shape[0], device="cuda", dtype=torch.float64)
    w = torch.tensor([case["base"] ** (-2.0 * j / case["n_rot"]) for j in range(h)], dtype=torch.float64, device="cuda")
    z = torch.complex(x[..., :h].contiguous(), x[..., h:2 * h].contiguous()) * torch.polar(torch.ones_like(w), p[:, None] * w)[:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * h:]], -1)


def _quantized(new, old, e_old):
    """One block's rows of one kv head: old codes and exponent, new values -> values of all."""
    top = min(float(new.abs().max()), I8_RANGE)
    e = next(e for e in range(-24, 10) if top <= 127 * 2.0 ** e)
    if old.shape[0]:
        e = max(e, e_old)
    rows = [(old * 2.0 ** (e_old - e)), new.clamp(-I8_RANGE, I8_RANGE) * 2.0 ** -e]
    return torch.cat(rows).round() * 2.0 ** e


def _sequence(case, s, which, b, length):
    """Cached rows 0 .. length-1 of sequence b in 64 bits, [length][HKV][hd]."""
    P, pages = case["page"], s["table"][b, :-(-length // case["page"])].long()
    c = s[which + "c"][pages].double()
    if case["cache"] == "i8":
        c = c.view(len(pages), case["HKV"], P // 16, 16, case["hd"]) * 2.0 ** (s[which + "x"][pages].double() - 127)[..., None, None]
        c = c.view(len(pages), case["HKV"], P, case["hd"]).transpose(1, 2)
    return c.reshape(len(pages) * P, case["HKV"], case["hd"])[:length]


def _after(case, s, which, b, p, x):
    """Rows of sequence b from its first touched block on, after x was appended at p."""
    p0, old = p // 16 * 16, _sequence(case, s, which, b, p)
    if case["cache"] == "f16":
        return torch.cat([old[p0:], x.clamp(-65504, 65504).half().double()])
    out = torch.empty(p - p0 + x.shape[0], *x.shape[1:], dtype=torch.float64, device="cuda")
    page, slot = int(s["table"][b, p0 // case["page"]]), p0 % case["page"]
    head = 16 - p % 16
    for h in range(case["HKV"]):
        e_old = int(s[which + "x"][page, h, slot // 16]) - 127
        codes = s[which + "c"][page, h, slot:slot + p - p0].double()
        out[:p - p0 + head, h] = _quantized(x[:head, h], codes, e_old)
    rest = x[head:]                                        # whole blocks, then what is left
    n = rest.shape[0] // 16 * 16
    full = rest[:n].reshape(n // 16, 16, *x.shape[1:])
    top = full.abs().amax((1, 3), keepdim=True).clamp(max=I8_RANGE)
    e = torch.full_like(top, 9)
    for k in range(8, -25, -1):
        e = torch.where(top <= 127 * 2.0 ** k, torch.full_like(e, k), e)
    out[p - p0 + head:p - p0 + head + n] = ((full.clamp(-I8_RANGE, I8_RANGE) * 2.0 ** -e).round() * 2.0 ** e).flatten(0, 1)
    for h in range(case["HKV"] if n < rest.shape[0] else 0):
        out[p - p0 + head + n:, h] = _quantized(rest[n:, h], rest[:0, h], 0)
    return out


def exact(case, seed):
    s, seqs = _inputs(case, seed), _lengths(case)
    res = {"q": [], "k": [], "v": [], "out": []}
    n, G = 0, case["H"] // case["HKV"]
    for b, (p, r) in enumerate(seqs):
        q, k, v, gate = (s[c][n:n + r].double() for c in ("q", "k", "v", "gate"))
        n += r
        if case["kind"] != "attend":
            q, k = _turned(q, p, case), _turned(k, p, case)
            q = q.to(_dt(case)).double() if case["kind"] == "step" else q
            tails = [_after(case, s, c, b, p, x) for c, x in (("k", k), ("v", v))]
            res["q"].append(q)
            res["k"].append(tails[0])
            res["v"].append(tails[1])
        if case["kind"] == "append":
            continue
        K, V = (_sequence(case, s, c, b, p + r) for c in "kv")
        if case["kind"] == "step":
            K, V = (torch.cat([c[:p // 16 * 16], t]) for c, t in zip((K, V), tails))
        t, at = torch.arange(p + r, device="cuda"), torch.arange(p, p + r, device="cuda")[:, None]
        seen = (t <= at) & ((t > at - case["window"]) | (t < case["sinks"]) if case["window"] else (t <= at))
        out = torch.empty_like(q)
        for h in range(case["H"]):
            S = (q[:, h] @ K[:, h // G].T * case["hd"] ** -0.5).masked_fill(~seen, -math.inf)
            out[:, h] = torch.softmax(S, -1) @ V[:, h // G]
        res["out"].append(out * torch.sigmoid(gate) if case["gated"] else out)
    return {k: torch.cat(v) for k, v in res.items() if v}
