"""gd_kv_fork and gd_kv_release of thousands of orders, up to the most that a call takes: all of one
sequence, of a few, of all, over rows of one part and of several, against what they come to
on the host; and that orders of one sequence cost what others do."""
import ctypes as C
import time

import numpy as np
import pytest

import gadeon_amd as ga

pytestmark = pytest.mark.gpu
I32, P = np.int32, 16


class Book:
    def __init__(self, ctx, n_seq, width, rng):
        self.ctx, self.bufs = ctx, []
        n = n_seq * width
        self.table = np.where(rng.random((n_seq, width)) < 0.8, rng.integers(0, n, (n_seq, width)), -1).astype(I32)
        self.refs = np.bincount(self.table[self.table >= 0], minlength=n).astype(I32)
        self.pages = ga.KVPages(refs=self.put(self.refs), table=self.put(self.table), n_pages=n, n_seq=n_seq, max_pages=width, page_size=P)

    def put(self, a):
        self.bufs.append(self.ctx.put(np.asarray(a, I32)))
        return self.bufs[-1]

    def same(self, table):
        assert np.array_equal(self.ctx.get(self.pages.table, table.shape, I32), table)
        assert np.array_equal(self.ctx.get(self.pages.refs, self.refs.shape, I32), np.bincount(table[table >= 0], minlength=len(self.refs)))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for p in self.bufs:
            self.ctx.free(p)


# Orders, sequences that they name, sequences, entries of a row (1024 are a part).
SIZES = [(300, 1, 3, 2500), (5000, 1, 2, 40), (5000, 7, 9, 3000), (20000, 3000, 3001, 1100), (65536, 1, 1, 5000), (65536, 40000, 40000, 9)]


@pytest.mark.parametrize("n,named,n_seq,width", SIZES)
def test_release(ctx, n, named, n_seq, width):
    rng = np.random.default_rng(n)
    with Book(ctx, n_seq, width, rng) as b:
        # Each order leaves most of the row; together they leave what lies in all their ranges.
        seq, top = rng.integers(0, named, n), width * P
        frm, to = rng.integers(0, top // 3 + 1, n), rng.integers(2 * top // 3, top + 2, n)
        lo, hi = np.zeros(n_seq, int), np.full(n_seq, top + 1)
        np.maximum.at(lo, seq, frm)
        np.minimum.at(hi, seq, to)
        p = np.arange(width) * P
        want = np.where((p + P > lo[:, None]) & (p < hi[:, None]), b.table, -1)
        assert (want != b.table).any()
        args = C.byref(b.pages), b.put(seq), b.put(frm), b.put(to), n
        ctx.get(args[1], 1, I32)
        start = time.perf_counter()
        ctx.gd_kv_release(*args)
        ctx.get(args[1], 1, I32)
        # (Some microseconds; of orders that each walk those before them, 65536 over five parts take seconds.)
        assert time.perf_counter() - start < 0.5
        b.same(want.astype(I32))


@pytest.mark.parametrize("n,named,n_seq,width", SIZES[1:])
def test_fork(ctx, n, named, n_seq, width):
    rng = np.random.default_rng(n)
    with Book(ctx, n_seq, width, rng) as b:
        # Sources are the first tenth of the sequences; some orders go over one of them.
        few = max(1, n_seq // 10)
        src, dst = rng.integers(0, few, n), rng.integers(0, n_seq, n)
        length = rng.integers(0, width * P + 2, n)
        last = np.full(n_seq, -1)
        last[dst] = np.arange(n)                               # (the last one stays)
        last[src] = -1
        want = b.table.copy()
        for d in np.flatnonzero(last >= 0):
            i = last[d]
            want[d] = np.where(np.arange(width) * P < length[i], b.table[src[i]], -1)
        ctx.gd_kv_fork(C.byref(b.pages), b.put(src), b.put(dst), b.put(length), n)
        b.same(want)
