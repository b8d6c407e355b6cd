"""gd_kv_attn_scored against a restatement in 64 bits: capped scores, a bias by distance,
documents (rows that see nothing among them) and prefixes, each and together, over single
tokens and ragged chunks, f16 and 8-bit caches, with windows and sinks; NaN and infinities
where nobody looks; in place, split keys, replays with changed masks.

Tolerances are test_gpu_kv_cache.py's with what the scores add.  A cap's slope is 1 at
most, so errors before it pass at most whole; its tanh loses eight roundings of 32 bits
(f16 rows, whose weights are rounded to 2^-11: 2^-21 of the cap), and scaling, bias and
their sum three each of the score and of the bias.  Of biases only those count whose keys
have weight: a row sees its own key, whose score is -A' at least (A' the largest score,
capped), so a key biased by 2 A' + 30 weighs under e^-30."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga
from test_gpu_kv_cache import ATTN, Batch, bound, raw, rows_of

pytestmark = pytest.mark.gpu
NEVER = 2**31 - 1


def attend(q, K, V, p0, scale, window, sinks, gate, cap=0.0, slope=None, first=None, prefix=0):
    n, H, hd = q.shape
    T, G = K.shape[0], H // K.shape[1]
    t, at = np.arange(T), p0 + np.arange(n)[:, None]
    seen = (t <= at) & ((t > at - window) | (t < sinks) if window else t <= at)
    seen |= t < prefix                                     # (T: the sequence's end)
    if first is not None:
        seen &= t >= first[:, None]
    out = np.zeros((n, H, hd))
    for h in range(H):
        s = q[:, h].astype(np.float64) @ np.where(np.isnan(K[:, h // G]), 0, K[:, h // G]).T * scale
        s = cap * np.tanh(s / cap) if cap else s
        if slope is not None:
            s = s - np.float64(slope[h]) * np.abs(at - t)
        s = np.where(seen, s, -np.inf)
        m = s.max(1, keepdims=True, initial=-np.inf)
        w = np.exp(s - np.where(np.isfinite(m), m, 0))
        out[:, h] = w @ np.where(np.isnan(V[:, h // G]), 0, V[:, h // G]) / np.maximum(w.sum(1, keepdims=True), 1e-300)
    return out if gate is None else out / (1 + np.exp(-gate.astype(np.float64)))


def most_off(q, K, V, p0, scale, f16, cap, slope):
    """test_gpu_kv_cache.bound, and what cap and bias add to a score's error."""
    G = q.shape[1] // K.shape[1]
    k = np.abs(np.nan_to_num(K))
    A = max((np.abs(q[:, h].astype(np.float64)) @ k[:, h // G].T).max(initial=0) for h in range(q.shape[1])) * abs(scale)
    top = min(A, cap) if cap else A
    bias = 0.0 if slope is None else min(float(np.abs(slope).max()) * (p0 + q.shape[0]), 2 * top + 30)
    more = 2.0 ** -24 * (3 * A + 8 * top + 6 * bias) + (2.0 ** -21 * cap if cap and f16 else 0)
    return bound(q, K, V, scale, f16) + 2 * np.abs(np.nan_to_num(V)).max(initial=0) * more


def masks(rng, seqs, doc, prefix):
    """Documents that start anywhere, rows that see nothing among them; prefixes of all lengths."""
    first, pre = [], []
    for p, r in seqs:
        at = np.sort(rng.integers(0, max(p + r, 1), r)) if rng.random() < 0.5 else np.full(r, max(0, p - 40))
        at = np.minimum(at, np.arange(p, p + r))
        if doc == "odd":
            at = np.where(rng.random(r) < 0.3, rng.choice([NEVER, -7, 0, max(p, 0) + r, max(p, 0) + 1], r), at)
        first.append(at)
        top = max(p + r, 1)
        pre.append(int(rng.choice([0, 1, top // 2, top - 1, top, top + 9, NEVER, -3])))
    return np.concatenate(first).astype(np.int32) if doc else None, np.array(pre, np.int32) if prefix else None


def run(ctx, bt, q, gate, how, window=0, sinks=0, scale=0.1, out=None):
    x, (n, H, hd) = ga.F16 if q.dtype == np.float16 else ga.F32, q.shape
    ptr = {k: None if v is None else bt.put(v) for k, v in how.items() if k != "cap"}
    sc = ga.Scores(cap=how.get("cap", 0.0), window=window, n_sink=sinks, **ptr)
    do = bt.put(np.full(q.shape, -77, q.dtype).view(raw(q).dtype)) if out is None else out
    args = (*bt.ref, bt.put(raw(q)), H * hd, None if gate is None else bt.put(raw(gate)), H * hd, do, x, H, scale, C.byref(sc))
    ctx.gd_kv_attn_scored(*args)
    return ctx.get(do, q.shape, q.dtype), lambda: (ctx.gd_kv_attn_scored(*args), ctx.get(do, q.shape, q.dtype))[1]


def check(ctx, seqs, dtype, x16, hd, H, hkv, page, what, window=0, sinks=0, gated=True, seed=0, row_start=True, max_len=0,
          scale=None, cap=20.0):
    with Batch(ctx, seqs, dtype, hkv, hd, page, seed=seed, row_start=row_start, lead=2 if row_start else 0,
               trail=3 if row_start else 0) as bt:
        KV, rng, scale = bt.fill(), bt.rng, hd ** -0.5 if scale is None else scale
        bt.desc.max_len = max_len
        q, gate = rows_of(rng, (bt.n, H, hd), x16), rows_of(rng, (bt.n, H, hd), x16)
        q = (q * 5).astype(q.dtype)                        # scores that a cap bends
        doc = "odd" if "odd" in what else "doc" in what
        first, prefix = masks(rng, seqs, doc, "prefix" in what)
        how = dict(cap=cap if "cap" in what else 0.0, slope=None, first=None, prefix=prefix)
        if "bias" in what:
            how["slope"] = (2.0 ** rng.uniform(-8, 0, H)).astype(np.float32)
        if first is not None:
            how["first"] = np.concatenate([np.zeros(bt.start[0], np.int32), first, np.zeros(bt.n - bt.start[-1], np.int32)])
        got, again = run(ctx, bt, q, gate if gated else None, how, window, sinks, scale)
        done = np.zeros(bt.n, bool)
        for b, (p, r) in enumerate(seqs):
            if p < 0 or r == 0:
                continue
            rows = slice(bt.start[b], bt.start[b] + r)
            done[rows] = True
            want = attend(q[rows], *KV[b], p, np.float32(scale), window, sinks, gate[rows] if gated else None, how["cap"],
                          how["slope"], None if first is None else how["first"][rows], 0 if prefix is None else prefix[b])
            err = np.abs(got[rows] - want)
            most = most_off(q[rows], *KV[b], p, scale, x16, how["cap"], how["slope"])
            assert err.max() <= most, (b, p, r, err.max(), most, np.argwhere(err > most)[:4])
        assert (got[~done] == -77).all()
        assert np.array_equal(again(), got)                # no order of arrival in it


WHAT = ["cap", "bias", "doc", "prefix", "odd doc", "cap bias odd doc prefix"]


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd,H,hkv,page", [(128, 40, 8, 16), (256, 24, 4, 48), (128, 3, 3, 32), (256, 18, 1, 16)])
@pytest.mark.parametrize("which", list(ATTN))
@pytest.mark.parametrize("what", WHAT)
def test_scores(ctx, dtype, x16, hd, H, hkv, page, which, what):
    check(ctx, ATTN[which], dtype, x16, hd, H, hkv, page if dtype == ga.I8 or H == 40 else page - 3, what, gated=H != 3,
          seed=hd + H, row_start=not which.startswith("tok"))


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("which", list(ATTN))
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (100, 5), (64, 130), (1000, 1), (1 << 30, 3)])
def test_windows(ctx, dtype, which, window, sinks):
    """Windows and sinks with documents and prefixes, which end before, in and behind them."""
    for x16, hd, H, hkv, what in ((False, 128, 10, 2, "doc prefix"), (True, 256, 6, 1, "cap prefix"), (True, 128, 5, 1, "odd doc"),
                                  (False, 256, 4, 2, "bias prefix")):
        check(ctx, ATTN[which], dtype, x16, hd, H, hkv, 16 if dtype == ga.I8 else 10, what, window, sinks, gated=x16,
              seed=window, row_start=not which.startswith("tok"))


@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("cap", [1e-3, 0.5, 5.0, 1e4, 1e30])
def test_caps(ctx, x16, cap):
    """From caps that leave signs to caps that leave the scores."""
    for which, hd in (("tokens", 128), ("ragged", 128), ("tokens", 256), ("later", 256)):
        check(ctx, ATTN[which], ga.F16, x16, hd, 8, 2, 16, "cap", row_start=which != "tokens", cap=min(cap, 1e9) if x16 else cap)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scales(ctx, scale):
    for which in ("tokens", "later"):
        for x16 in (False, True):
            check(ctx, ATTN[which], ga.I8, x16, 128, 4, 2, 16, "cap bias", row_start=which == "later", scale=scale)


@pytest.mark.parametrize("cap,scale", [(1e-30, 1e30), (1e-30, -1e30), (64.0, 1e30), (1e-30, 1e-30), (1e30, 1e30)])
def test_caps_and_scales_far_apart(ctx, cap, scale):
    """Rows of zeros have scores of 0 whatever they are scaled by; a cap of next to nothing leaves
    next to nothing of the others' scores: all keys weigh the same."""
    for seqs, start in (([(700, 1), (31, 1)], False), ([(700, 90), (31, 3)], True)):
        for x16 in (False, True):
            with Batch(ctx, seqs, ga.F16, 2, 128, 16, row_start=start) as bt:
                KV = bt.fill()
                q = rows_of(bt.rng, (bt.n, 4, 128), x16)
                if cap > 1:
                    q[:] = 0
                q[::2] = 0
                got, _ = run(ctx, bt, q, None, dict(cap=cap), scale=scale)
                for b, (p, r) in enumerate(seqs):
                    rows = slice(bt.start[b], bt.start[b] + r)
                    want = attend(q[rows] * 0, *KV[b], p, 1.0, 0, 0, None)
                    assert np.abs(got[rows] - want).max() <= bound(q[rows] * 0, *KV[b], 1.0, x16) + 2.0 ** -24, (b, x16)


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("what", ["cap bias", "doc prefix", "odd doc"])
def test_split_keys(ctx, dtype, what):
    """Long sequences beside short and idle ones, over and under 64 of them; splits of which a
    document leaves some without keys."""
    rng = np.random.default_rng(5)
    for n in (3, 40, 90):
        tokens = [(int(p), 1) for p in rng.integers(-5, 60, n)]
        chunks = [(int(rng.integers(-5, 60)), int(rng.integers(0, 3))) for _ in range(n)]
        for b, (p, r) in zip((0, n // 2, n - 1), [(9000, 1), (1800, 40), (2500, 7)]):
            tokens[b], chunks[b] = (p, 1), (p, r)
        for seqs, start in ((tokens, False), (tokens, True), (chunks, True)):
            check(ctx, seqs, dtype, n == 40, 256 if n == 3 else 128, 6, 2, 16, what, gated=n == 3, row_start=start, seed=n)


@pytest.mark.parametrize("H,hkv,rows", [(40, 8, 1700), (24, 1, 2800)])
def test_documents_of_many_units(ctx, H, hkv, rows):
    """More workgroups than the chip holds, which go by their documents' lengths; over 512 units of a
    sequence, where they do not."""
    seqs = [(0, rows), (50, 130), (700, 1)]
    with Batch(ctx, seqs, ga.F16, hkv, 128, 16) as bt:
        KV, rng = bt.fill(), bt.rng
        q = (rows_of(rng, (bt.n, H, 128), True) * 3).astype(np.float16)
        first, _ = masks(rng, seqs, "odd", False)
        first[:rows] = np.minimum(np.sort(rng.choice(rows, 9))[rng.integers(0, 9, rows // 100 + 1)].repeat(100)[:rows], np.arange(rows))
        got, again = run(ctx, bt, q, q, dict(first=first, cap=20.0))
        for b, (p, r) in enumerate(seqs):
            at = slice(bt.start[b], bt.start[b] + r)
            pick = [0, H // 2, H - 1]                       # (heads of the first and the last kv head)
            for h in pick:
                one = lambda x: x[at][:, h:h + 1]           # noqa: E731
                K, V = (c[:, h // (H // hkv)][:, None] for c in KV[b])
                want = attend(one(q), K, V, p, np.float32(0.1), 0, 0, one(q), 20.0, None, first[at])
                err, most = np.abs(one(got) - want).max(), most_off(one(q), K, V, p, 0.1, True, 20.0, None)
                assert err <= most, (b, h, err, most)
        assert np.array_equal(again(), got)


@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
def test_plain_scores_are_the_other_entrys(ctx, x16):
    """No cap and no arrays: gd_kv_attn's results; arrays that change nothing: within its bound."""
    for which in ("tokens", "ragged"):
        with Batch(ctx, ATTN[which], ga.I8, 2, 128, 16, row_start=which == "ragged") as bt:
            KV = bt.fill()
            q = rows_of(bt.rng, (bt.n, 4, 128), x16)
            got, _ = run(ctx, bt, q, None, {}, 100, 3)
            do = bt.put(raw(np.full_like(q, -77)))
            ctx.gd_kv_attn(*bt.ref, bt.put(raw(q)), 512, None, 0, do, ga.F16 if x16 else ga.F32, 4, 0.1, 100, 3)
            assert np.array_equal(got, ctx.get(do, q.shape, q.dtype))
            how = dict(slope=np.zeros(4, np.float32), first=np.zeros(bt.n, np.int32), prefix=np.zeros(len(ATTN[which]), np.int32))
            same, _ = run(ctx, bt, q, None, how, 100, 3)
            for b, (p, r) in enumerate(ATTN[which]):
                rows = slice(bt.start[b], bt.start[b] + r)
                if p >= 0 and r:
                    assert np.abs(same[rows] - got[rows]).max() <= 2 * most_off(q[rows], *KV[b], p, 0.1, x16, 0, None)


def test_rows_that_see_nothing_are_zeros(ctx):
    """All rows of a call, f16 and f32, tokens and chunks, whole and split, gated or not."""
    for seqs, start in (([(40, 1), (9000, 1)], False), ([(40, 70), (9000, 3)], True)):
        for hd in (128, 256):
            for x16 in (False, True):
                with Batch(ctx, seqs, ga.I8, 1, hd, 16, row_start=start) as bt:
                    bt.fill()
                    q = rows_of(bt.rng, (bt.n, 5, hd), x16)
                    for how in (dict(first=np.full(bt.n, NEVER, np.int32)), dict(first=np.full(bt.n, 9003, np.int32), cap=9.0)):
                        got, again = run(ctx, bt, q, q if x16 else None, how)
                        assert not got.any() and not again().any()


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_non_finite_values_where_nobody_looks(ctx, dtype, x16, hd, value):
    """A value that is no number reaches the rows of its own document and no other, capped or not."""
    H, hkv, page, seqs, bad = 4, 2, 16, [(0, 200), (130, 1), (60, 40)], 90
    with Batch(ctx, seqs, dtype, hkv, hd, page) as bt:
        KV, planes = bt.fill(), bt.planes()
        q = rows_of(bt.rng, (bt.n, H, hd), x16)
        first = np.concatenate([np.where(np.arange(200) < 112, 0, 112), [112], np.where(np.arange(60, 100) < 96, 48, 96)])
        for which in (0, 1):
            p = [a.copy() for a in planes]
            for b in range(3):
                pg = bt.table[b, bad // page]
                if dtype == ga.F16:
                    p[which][pg, bad % page, 1, 7] = value
                else:
                    p[2 + which][pg, 1, 0] = 255
            for d, a in zip((bt.kv.k, bt.kv.v, bt.kv.k_exp, bt.kv.v_exp), p):
                ctx.set(d, a)
            for cap in (0.0, 30.0):
                got, _ = run(ctx, bt, q, None, dict(first=first.astype(np.int32), cap=cap), scale=hd ** -0.5)
                for b, (p0, r) in enumerate(seqs):
                    rows = slice(bt.start[b], bt.start[b] + r)
                    want = attend(q[rows], *KV[b], p0, np.float32(hd ** -0.5), 0, 0, None, cap, None, first[rows])
                    at = p0 + np.arange(r)
                    sees = (at >= bad // 16 * 16) & (first[rows] <= bad)
                    fine = np.repeat(~sees[:, None], H, 1)
                    fine[:, :H // 2] = True
                    err = np.abs(got[rows] - want)[fine]
                    most = most_off(q[rows], *KV[b], p0, hd ** -0.5, x16, cap, None)
                    assert np.isfinite(err).all() and err.max(initial=0) <= most, (which, b)


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("tokens", [True, False], ids=["tokens", "chunks"])
def test_a_nan_is_not_capped(ctx, dtype, x16, hd, tokens):
    """A key that is no number makes the heads that see it NaN, one of q its own head, under any cap."""
    H, hkv, page, bad = 4, 2, 16, 90
    with Batch(ctx, [(130, 1), (120, 1), (60, 1)] if tokens else [(130, 5), (60, 40), (0, 20)], dtype, hkv, hd, page, row_start=not tokens) as bt:
        bt.fill()
        planes = bt.planes()
        for b in range(3):
            pg = bt.table[b, bad // page]
            if pg < 0:
                continue
            if dtype == ga.F16:
                planes[0][pg, bad % page, 1, 7] = np.nan
            else:
                planes[2][pg, 1, 0] = 255
        for d, a in zip((bt.kv.k, bt.kv.v, bt.kv.k_exp, bt.kv.v_exp), planes):
            ctx.set(d, a)
        q = rows_of(bt.rng, (bt.n, H, hd), x16)
        for cap in (0.0, 30.0, 500.0, 5000.0):
            for slope in (None, np.full(H, 0.01, np.float32)):
                q[:] = rows_of(bt.rng, (bt.n, H, hd), x16)
                q[-1, 0, 3] = np.nan
                got, _ = run(ctx, bt, q, None, dict(cap=cap, slope=slope), scale=hd ** -0.5)
                want = np.zeros((bt.n, H), bool)
                for b, (p0, r) in enumerate(bt.seqs):
                    at = p0 + np.arange(r)
                    want[bt.start[b]:bt.start[b] + r, H // 2:] = (at >= (bad if dtype == ga.F16 else bad // 16 * 16))[:, None]
                want[-1, 0] = True
                assert np.array_equal(np.isnan(got).all(2), want) and np.array_equal(np.isnan(got).any(2), want), (cap, slope is None)


def test_masked_pages_that_are_not_there(ctx):
    """Pages before every document, and before the window, may be dropped."""
    for dtype in (ga.I8, ga.F16):
        for seqs, start in (([(300, 1), (170, 1)], False), ([(300, 20), (170, 90)], True)):
            with Batch(ctx, seqs, dtype, 2, 128, 16, row_start=start) as bt:
                bt.fill()
                q = rows_of(bt.rng, (bt.n, 4, 128), False)
                how = dict(first=np.full(bt.n, 100, np.int32), cap=9.0, slope=np.full(4, 0.01, np.float32))
                got, again = run(ctx, bt, q, None, how)
                table = bt.table.copy()
                table[:, :6] = [[-1, bt.pages, 2**31 - 1, -2**31, -1, bt.pages + 1]]
                ctx.set(bt.desc.page_table, table)
                assert got.any() and np.array_equal(again(), got)


def test_far_positions(ctx):
    """Distances past 2^24 positions: pages of 2^20 positions, of which the last are there."""
    page, hd, p = 1 << 20, 128, (1 << 25) + 77
    with Batch(ctx, [(0, 200)], ga.F16, 1, hd, page, spare=40) as bt:
        ((K, V),) = bt.fill()
        table = np.full(bt.table.shape, -1, np.int32)
        table[0, p // page] = table[0, 0] = bt.table[0, 0]  # the same 200 keys, far apart
        ctx.set(bt.desc.page_table, table)
        rows = 3
        bt.desc.n_rows, bt.desc.row_start, bt.desc.pos = rows, bt.put(np.array([0, rows], np.int32)), bt.put(np.array([p], np.int32))
        q, slope = rows_of(bt.rng, (rows, 4, hd), False), np.array([1e-8, 1e-7, 3e-9, 0.01], np.float32)
        bt.desc.max_len = 0
        got, _ = run(ctx, bt, q, None, dict(slope=slope), 77, 200)
        T = p % page + rows
        keys = np.concatenate([np.arange(200), p // page * page + np.arange(T)])
        for i in range(rows):
            see = (keys <= p + i) & ((keys > p + i - 77) | (keys < 200))
            for h in range(4):
                t, k = keys[see], np.concatenate([np.arange(200), np.arange(T)])[see]
                s = K[k, 0] @ q[i, h].astype(np.float64) * np.float32(0.1) - np.float64(slope[h]) * np.abs(p + i - t)
                w = np.exp(s - s.max())
                want = w @ V[k, 0] / w.sum()
                assert np.abs(got[i, h] - want).max() <= most_off(q, K, V, p, 0.1, False, 0, slope[:3]), (i, h)


def test_in_place(ctx):
    hd, H = 128, 8
    for seqs, start in (([(3000, 1), (70, 1)], False), ([(2100, 130), (5, 3)], True)):
        with Batch(ctx, seqs, ga.I8, 2, hd, 16, row_start=start) as bt:
            bt.fill()
            q, g = (rows_of(bt.rng, (bt.n, H, hd), True) for _ in "qg")
            how = dict(cap=10.0, slope=np.full(H, 0.1, np.float32))
            want, _ = run(ctx, bt, q, g, how)
            sc = ga.Scores(cap=10.0, slope=bt.put(how["slope"]))
            for over in (0, 1):
                d = [bt.put(raw(q)), bt.put(raw(g))]
                ctx.gd_kv_attn_scored(*bt.ref, d[0], H * hd, d[1], H * hd, d[over], ga.F16, H, 0.1, C.byref(sc))
                assert np.array_equal(ctx.get(d[over], q.shape, q.dtype), want)


@pytest.mark.parametrize("tokens", [True, False], ids=["tokens", "chunks"])
def test_replays_with_changed_masks(ctx, tokens):
    """A recorded call replayed with other slopes, documents, prefixes, positions and tables."""
    seqs = [(2100, 1), (40, 1), (-1, 1)] if tokens else [(2100, 30), (40, 90), (7, 3)]
    with Batch(ctx, seqs, ga.F16, 2, 128, 16, row_start=not tokens) as bt:
        bt.fill()
        H, rng = 6, bt.rng
        q = rows_of(rng, (bt.n, H, 128), True)
        dq, do = bt.put(raw(q)), bt.put(raw(np.zeros_like(q)))
        d = dict(slope=bt.put(np.zeros(H, np.float32)), first=bt.put(np.zeros(bt.n, np.int32)), prefix=bt.put(np.zeros(3, np.int32)))
        sc = ga.Scores(cap=12.0, window=300, n_sink=2, **d)
        call = lambda: ctx.gd_kv_attn_scored(*bt.ref, dq, H * 128, None, 0, do, ga.F16, H, 0.1, C.byref(sc))  # noqa: E731
        call()
        g = C.c_void_p()
        ctx.gd_graph_begin()
        call()
        ctx.gd_graph_end(C.byref(g))
        seen = []
        for i in range(4):
            ctx.set(d["slope"], rng.random(H).astype(np.float32) / 8)
            ctx.set(d["first"], rng.integers(0, 60, bt.n).astype(np.int32))
            ctx.set(d["prefix"], rng.integers(0, 2000, 3).astype(np.int32))
            ctx.set(bt.desc.pos, np.array([2100 - 50 * i, 40 - i, -1 if i % 2 else 7], np.int32))
            ctx.set(do, raw(np.zeros_like(q)))
            ctx.gd_graph_launch(g)
            one = ctx.get(do, q.shape, q.dtype)
            ctx.set(do, raw(np.zeros_like(q)))
            call()
            assert one.any() and np.array_equal(ctx.get(do, q.shape, q.dtype), one)
            seen.append(one)
        assert all(not np.array_equal(a, b) for a, b in zip(seen, seen[1:]))
        ctx.lib.gd_graph_destroy(g)
