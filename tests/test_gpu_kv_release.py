"""gd_kv_release of what a window has passed where attention still sees the start of the
sequence: with gd_kv_pages.keep the pages of sinks and prefixes stay, against a model
on the host, entry by entry, and against the attention of a cache that lets go of nothing, bit for bit."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga
from test_gpu_kv_cache import Batch, raw, rows_of
from test_gpu_kv_pages import SIZES, Device, filled

pytestmark = pytest.mark.gpu
I32 = np.int32


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("seed", [0, 1])
def test_kept_starts(ctx, size, seed):
    rng = np.random.default_rng(seed)
    n_seq, width, P, _ = size
    with Device(ctx, *size) as d:
        filled(d, rng)
        keep = rng.choice([-5, 0, 1, P, P + 1, width * P, 2**31 - 1, int(rng.integers(width * P))], n_seq)
        d.pages.keep = d.put(keep.astype(I32))
        for k in (1, n_seq, n_seq + 3):
            seq, frm = rng.integers(-1, n_seq + 1, k), rng.integers(0, width * P, k)
            to = rng.choice([0, P, width * P, 2**31 - 1], k)
            for b, f, t in zip(seq, frm, to):
                if 0 <= b < n_seq:
                    p = np.arange(width) * P
                    for e in np.flatnonzero((d.m.table[b] >= 0) & ~(((p + P > f) | (p < keep[b])) & (p < t))):
                        d.m.count(d.m.table[b, e], -1)
                        d.m.table[b, e] = -1
            ctx.gd_kv_release(d.ref, d.put(seq.astype(I32)), d.put(frm.astype(I32)), d.put(to.astype(I32)), k)
            d.same()


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("tokens", [True, False], ids=["tokens", "chunks"])
@pytest.mark.parametrize("sinks,prefix", [(5, 0), (0, 70), (40, 20)])
def test_windows_that_let_go(ctx, dtype, tokens, sinks, prefix):
    """What is let go of goes to others (here: becomes NaN); sinks and prefixes are seen as before."""
    window, P, H, hkv, hd = 100, 16, 4, 2, 128
    seqs = [(700, 1), (90, 1), (3000, 1)] if tokens else [(700, 30), (90, 5), (3000, 3)]
    with Batch(ctx, seqs, dtype, hkv, hd, P, row_start=not tokens) as bt:
        bt.fill()
        B = len(seqs)
        q, pre = rows_of(bt.rng, (bt.n, H, hd), False), np.array([prefix, 0, max(0, prefix - 11)], I32)
        sc = ga.Scores(cap=9.0, window=window, n_sink=sinks, prefix=bt.put(pre) if prefix else None)
        dq, do = bt.put(raw(q)), bt.put(raw(np.full_like(q, -77)))

        def attend():
            ctx.gd_kv_attn_scored(*bt.ref, dq, H * hd, None, 0, do, ga.F32, H, 0.1, C.byref(sc))
            return ctx.get(do, q.shape, np.float32)

        want = attend()
        refs = np.bincount(bt.table[bt.table >= 0], minlength=bt.pages).astype(I32)
        pages = ga.KVPages(refs=bt.put(refs), table=bt.desc.page_table, n_pages=bt.pages, n_seq=B, max_pages=bt.table.shape[1],
                           page_size=P, keep=bt.put(np.maximum(pre, sinks).astype(I32)))
        pos = np.array([p for p, _ in seqs], I32)
        ctx.gd_kv_release(C.byref(pages), bt.put(np.arange(B, dtype=I32)), bt.put(pos - window), bt.put(np.full(B, 2**31 - 1, I32)), B)
        table, left = ctx.get(bt.desc.page_table, bt.table.shape, I32), ctx.get(pages.refs, bt.pages, I32)
        assert np.array_equal(left, np.bincount(table[table >= 0], minlength=bt.pages))
        free = np.flatnonzero((refs > 0) & (left == 0))
        assert len(free) >= (700 - 100) // P + (3000 - 100) // P - 2 * (max(prefix, sinks) // P + 2)
        planes = bt.planes()
        for a in planes[:2] if dtype == ga.F16 else planes[2:]:
            a[free] = np.nan if dtype == ga.F16 else 255
        for p, a in zip((bt.kv.k, bt.kv.v, bt.kv.k_exp, bt.kv.v_exp), planes):
            ctx.set(p, a)
        assert np.array_equal(attend(), want)
        ctx.gd_kv_release(C.byref(pages), bt.put(np.arange(B, dtype=I32)), None, bt.put(np.zeros(B, I32)), B)
        assert not ctx.get(pages.refs, bt.pages, I32).any()    # ended: the starts too


def test_ranges_of_nothing(ctx):
    """Where from is not before to: one page stays, if it holds both from and to - 1, and else none."""
    for frm, to, left in ((5, 5, [0]), (5, 1, [0]), (16, 16, []), (17, 16, []), (40, 36, [2]), (40, 20, []), (0, 0, []), (9, -4, [])):
        with Device(ctx, 1, 4, 16, 4) as d:
            d.m.table[0], d.m.refs[:] = [3, 1, 2, 0], 1
            d.set()
            ctx.gd_kv_release(d.ref, *(d.put(np.array([x], I32)) for x in (0, frm, to)), 1)
            d.m.release([0], [frm], [to])
            d.same()
            assert list(np.flatnonzero(d.m.table[0] >= 0)) == left
