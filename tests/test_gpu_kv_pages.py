"""The cache's pages (gd_kv_fork, gd_kv_release, gd_kv_reserve, gd_kv_compact,
gd_kv_copy_pages) against a model on the host that goes entry by entry, bit for bit; and a
serving loop of them with appends and attention, eager and recorded, against the
conversations' own histories."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga
import test_gpu_kv_cache as kc
from test_gpu_kv_cache import raw, rows_of

pytestmark = pytest.mark.gpu
I32 = np.int32


# ------------------------------------------------------------------ the model


class Model:
    def __init__(self, n_seq, max_pages, page, n_pages):
        self.refs, self.table, self.P = np.zeros(n_pages, I32), np.full((n_seq, max_pages), -1, I32), page

    def there(self, page):
        return 0 <= page < len(self.refs)

    def count(self, page, by):
        if self.there(page):
            self.refs[page] += by

    def fork(self, src, dst, length):
        n, before = len(self.table), self.table.copy()
        for i, (s, d, m) in enumerate(zip(src, dst, length)):
            if not (0 <= s < n and 0 <= d < n) or d in src or d in dst[i + 1:]:
                continue
            for e in range(self.table.shape[1]):
                new = before[s, e] if e * self.P < m and self.there(before[s, e]) else -1
                self.count(self.table[d, e], -1)
                self.count(new, 1)
                if self.there(self.table[d, e]) or self.table[d, e] != new:
                    self.table[d, e] = new

    def release(self, seq, frm, to):
        for i, b in enumerate(seq):
            if not 0 <= b < len(self.table):
                continue
            for e in range(self.table.shape[1]):
                p = e * self.P
                if (p + self.P > (frm[i] if frm is not None else 0) and p < to[i]) or not self.there(self.table[b, e]):
                    continue
                self.count(self.table[b, e], -1)
                self.table[b, e] = -1

    def reserve(self, pos, rows):
        free, out, copies, short = list(np.flatnonzero(self.refs <= 0)), list(pos), [], False
        start, total = self.refs.copy(), 0
        for b, (p, r) in enumerate(zip(pos, rows)):
            if p < 0 or r <= 0:
                continue
            entries = [e for e in range(p // self.P, (p + r - 1) // self.P + 1) if e < self.table.shape[1]]
            needs = [e for e in entries if not self.there(self.table[b, e]) or self.refs[self.table[b, e]] > 1]
            kept = any(self.there(self.table[b, e]) and start[self.table[b, e]] > 1 for e in entries)
            short = short or len(needs) > len(free)
            if short and (needs or kept):
                out[b] = -1
                continue
            for e in needs:
                old, new = self.table[b, e], free.pop(0)
                self.count(old, -1)
                if self.there(old) and e * self.P < p:
                    copies.append((old, new))
                self.table[b, e], self.refs[new] = new, 1
        return np.array(out, I32), copies

    def compact(self):
        moves = []
        while True:
            free, used = np.flatnonzero(self.refs <= 0), np.flatnonzero(self.refs > 0)
            if not len(free) or not len(used) or free[0] > used[-1]:
                return moves, len(used)
            moves.append((used[-1], free[0]))
            self.refs[free[0]], self.refs[used[-1]] = self.refs[used[-1]], 0
            self.table[self.table == used[-1]] = free[0]


class Device:
    """The same on the device, beside a model of it."""

    def __init__(self, ctx, n_seq, max_pages, page, n_pages):
        self.ctx, self.m, self.bufs = ctx, Model(n_seq, max_pages, page, n_pages), []
        self.refs, self.table = self.put(self.m.refs), self.put(self.m.table)
        self.copies, self.pos_out = self.put(np.zeros((n_seq, 2), I32)), self.put(np.zeros(n_seq, I32))
        self.moves, self.n = self.put(np.zeros((n_pages, 2), I32)), self.put(np.zeros(2, I32))
        self.pages = ga.KVPages(refs=self.refs, table=self.table, n_pages=n_pages, n_seq=n_seq, max_pages=max_pages, page_size=page)
        self.ref = C.byref(self.pages)

    def put(self, a):
        self.bufs.append(self.ctx.put(np.asarray(a)))
        return self.bufs[-1]

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for p in self.bufs:
            self.ctx.free(p)

    def set(self):
        self.ctx.set(self.refs, self.m.refs)
        self.ctx.set(self.table, self.m.table)

    def same(self):
        assert np.array_equal(self.ctx.get(self.table, self.m.table.shape, I32), self.m.table)
        assert np.array_equal(self.ctx.get(self.refs, self.m.refs.shape, I32), self.m.refs)

    def fork(self, src, dst, length):
        self.m.fork(list(src), list(dst), list(length))
        self.ctx.gd_kv_fork(self.ref, *(self.put(np.array(a, I32)) for a in (src, dst, length)), len(src))
        self.same()

    def release(self, seq, frm, to):
        self.m.release(seq, frm, to)
        self.ctx.gd_kv_release(self.ref, self.put(np.array(seq, I32)), None if frm is None else self.put(np.array(frm, I32)),
                               self.put(np.array(to, I32)), len(seq))
        self.same()

    def seqs(self, pos, rows, tokens):
        start = np.cumsum([0, *rows]).astype(I32)
        return ga.Seqs(n_rows=int(start[-1]), row_start=None if tokens else self.put(start), pos=self.put(np.array(pos, I32)), rope_shift=None,
                       page_table=self.table, n_seq=len(pos), max_pages=self.pages.max_pages, max_len=0)

    def reserve(self, pos, rows, tokens=False, in_place=False):
        want, copies = self.m.reserve(pos, rows)
        s, mark = self.seqs(pos, rows, tokens), np.full((len(pos), 2), -9, I32)
        self.ctx.set(self.copies, mark)
        out = s.pos if in_place else self.pos_out
        self.ctx.gd_kv_reserve(self.ref, C.byref(s), self.copies, self.n, out)
        assert np.array_equal(self.ctx.get(out, len(pos), I32), want)
        mark[:len(copies)] = np.array(copies, I32).reshape(-1, 2)
        assert self.ctx.get(self.n, 1, I32)[0] == len(copies) and np.array_equal(self.ctx.get(self.copies, mark.shape, I32), mark)
        self.same()
        return want, copies

    def compact(self):
        moves, used = self.m.compact()
        mark = np.full((len(self.m.refs), 2), -9, I32)
        self.ctx.set(self.moves, mark)
        self.ctx.gd_kv_compact(self.ref, self.moves, self.n)
        mark[:len(moves)] = np.array(moves, I32).reshape(-1, 2)
        assert list(self.ctx.get(self.n, 2, I32)) == [len(moves), used]
        assert np.array_equal(self.ctx.get(self.moves, mark.shape, I32), mark)
        self.same()


def filled(d, rng, share=True):
    """Sequences of all lengths, some branches of others, pages anywhere."""
    m, n = d.m, len(d.m.table)
    order, at = rng.permutation(len(m.refs)), 0
    for b in range(n):
        if share and b and rng.random() < 0.4:
            s, k = int(rng.integers(b)), int(rng.integers(m.table.shape[1] + 1))
            m.table[b, :k] = m.table[s, :k]
        elif rng.random() < 0.8:
            k = min(int(rng.integers(m.table.shape[1] + 1)), len(order) - at)
            m.table[b, :k] = order[at:at + k]
            at += k
    m.refs[:] = np.bincount(m.table[m.table >= 0], minlength=len(m.refs))
    d.set()


SIZES = [(1, 1, 1, 1), (3, 5, 16, 12), (8, 40, 20, 100), (70, 17, 48, 900), (130, 9, 16, 4097), (5, 1500, 1, 9000), (300, 30, 64, 5000)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("seed", [0, 1])
def test_fork_and_release(ctx, size, seed):
    rng = np.random.default_rng(seed)
    n_seq, width, P, _ = size
    with Device(ctx, *size) as d:
        filled(d, rng)
        for k in (1, max(1, n_seq // 3), n_seq + 3):
            src, dst = rng.integers(-1, n_seq + 1, k), rng.integers(-1, n_seq + 1, k)
            if k > 1:
                src = rng.choice(src[:max(1, k // 4)], k)       # a few prompts, branches named twice
            d.fork(src, dst, rng.choice([-5, 0, 1, P, P + 1, width * P - 1, width * P, 2**31 - 1, int(rng.integers(width * P))], k))
            d.release(rng.integers(-1, n_seq + 1, k), None if k == 1 else rng.integers(-3, width * P, k),
                      rng.choice([-4, 0, 1, P, width * P // 2, 2**31 - 1], k))
        d.release(range(n_seq), None, [0] * n_seq)
        assert not d.m.refs.any() and (d.m.table == -1).all()


def test_fork_leaves_out(ctx):
    """Orders of themselves, over a source, over each other (the last one counts), out of range."""
    with Device(ctx, 6, 4, 16, 20) as d:
        d.m.table[0], d.m.table[1, :2], d.m.table[2, :3] = [3, 9, 1, 7], [5, 6], [2, 4, 8]
        d.m.refs[[3, 9, 1, 7, 5, 6, 2, 4, 8]] = 1
        d.set()
        d.fork([0, 1, 0, 0, 2, -1, 6, 1], [0, 2, 3, 3, 3, 4, 4, 7], [64] * 8)
        assert list(d.m.table[3]) == [2, 4, 8, -1] and d.m.refs[8] == 2 and d.m.refs[3] == 1
        d.fork([0, 0, 0], [4, 5, 1], [33, 16, 17])
        assert list(d.m.table[4]) == [3, 9, 1, -1] and list(d.m.table[1]) == [3, 9, -1, -1] and d.m.refs[3] == 4 and not d.m.refs[5]


def test_entries_that_name_no_page(ctx):
    """Of tables that hold other values than pages: taken for none, counted nowhere."""
    with Device(ctx, 4, 6, 16, 9) as d:
        d.m.table[0], d.m.table[1] = [4, -7, 9, 2**31 - 1, -2**31, 8], [0, 1, 2, -1, 100, 3]
        d.m.refs[[4, 8, 0, 1, 2, 3]] = 1
        d.set()
        d.fork([0], [2], [96])
        d.release([1], None, [32])
        d.reserve([0, 40, -1, 0], [96, 3, 5, 1])
        d.compact()


# (The last ones pass 4096 sequences or entries of their rows.)
@pytest.mark.parametrize("size", SIZES + [(512, 5, 16, 3000), (513, 2, 16, 1500), (2049, 2, 16, 6000), (4000, 2, 16, 9000), (4500, 3, 16, 15000),
                                         (3, 6000, 1, 20000)], ids=str)
@pytest.mark.parametrize("tokens", [True, False], ids=["tokens", "chunks"])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_reserve(ctx, size, tokens, seed):
    """Steps that need pages, copies and nothing, beside idle sequences, until the cache is full
    and past that."""
    rng = np.random.default_rng(seed)
    n_seq, width, P, n_pages = size
    with Device(ctx, *size) as d:
        filled(d, rng, seed != 1)
        for step in range(6):
            pos = rng.integers(-2, width * P + 3, n_seq)
            if step % 2:                                        # go on where their pages end, or in the last
                held = (d.m.table >= 0).sum(1) * P
                pos = np.maximum(held - rng.integers(0, P + 1, n_seq), 0)
            rows = np.ones(n_seq, int) if tokens else rng.choice([0, 1, 2, P, 3 * P + 1], n_seq)
            if not tokens and step == 4:
                rows[-1] = width * P + 5                        # past the table
            d.reserve(pos.tolist(), rows.tolist(), tokens, in_place=step == 3)


@pytest.mark.parametrize("n", [5, 300, 1500, 4200])
@pytest.mark.parametrize("n_pages", [16383, 16384, 20479, 20481, 37000, 70001])
def test_reserve_behind_pages_in_use(ctx, n, n_pages):
    """Free pages behind many in use: at the end, one here and there, one too few."""
    for free in ([*range(n_pages - n, n_pages)], [1, 4095, 4096, 16383] + [*range(n_pages - n + 1, n_pages)],
                 [*range(n_pages - n + 1, n_pages)], [*range(0, n_pages, max(1, n_pages // n))]):
        with Device(ctx, n, 1, 16, n_pages) as d:
            d.m.refs[:] = 1
            d.m.refs[[f for f in free if f < n_pages]] = 0
            d.set()
            d.reserve([0] * n, [1] * n, True)


@pytest.mark.parametrize("n", [500, 1000, 4096, 4097, 9000])
@pytest.mark.parametrize("groups", [1, 7, 499])
def test_reserve_many_that_share(ctx, n, groups):
    """All sequences go on in a page that they share in groups: of each the last keeps it."""
    with Device(ctx, n, 2, 16, n + 3 * groups) as d:
        d.m.table[:, 0] = (np.arange(n) % groups) * 3
        d.m.refs[:] = np.bincount(d.m.table[:, 0], minlength=len(d.m.refs))
        d.set()
        out, copies = d.reserve((np.arange(n) % 15 + 1).tolist(), [1] * n, True)
        assert (out >= 0).all() and len(copies) == n - groups


def test_reserve_shares_out(ctx):
    """Four branches that go on in their shared page: three copies, the last keeps it; beside a
    holder outside the call all four copy; too few pages: the first ones get theirs, the others
    keep what they had."""
    for outside, n_pages, served in ((0, 20, 4), (1, 20, 4), (0, 4, 2), (0, 5, 4), (1, 5, 3), (0, 2, 0)):
        with Device(ctx, 5, 3, 16, n_pages) as d:
            d.m.table[:4, :2] = [[0, 1]] * 4
            d.m.refs[:2] = 4 + outside
            d.set()
            out, copies = d.reserve([20, 31, 17, 20, -1], [1] * 5, True)
            assert (out[:4] >= 0).sum() == served and len(copies) == min(served, 3 + outside), (outside, n_pages)
            assert all(src == 1 for src, _ in copies)


def test_reserve_when_full_keeps_on(ctx):
    """Who needs nothing goes on though others do not, but not on a page that an idle one shares."""
    with Device(ctx, 5, 3, 16, 4) as d:
        d.m.table[:, 0] = [0, 1, 2, 3, 3]
        d.m.refs[:] = [1, 1, 1, 2]
        d.set()
        out, copies = d.reserve([5, 16, 7, 3, 3], [1] * 5, True)
        assert list(out) == [5, -1, 7, -1, -1] and not copies
        out, copies = d.reserve([5, 15, 7, -1, -1], [1, 1, 2, 1, 1])
        assert list(out) == [5, 15, 7, -1, -1] and not copies


def test_rows_that_overlap_stay_in_bounds(ctx):
    """Row starts that do not ascend (which they must): something is reserved, nothing else touched."""
    for n, width in ((1500, 40), (1200, 3), (5000, 40)):
        overlap(ctx, n, width)


def overlap(ctx, n, width):
    with Device(ctx, n, width, 1, 70000) as d:
        s = d.seqs([0] * n, [1] * n, False)
        start = np.zeros(n + 1, I32)
        start[1::2] = n                                         # every other one has all rows
        d.ctx.set(s.row_start, start)
        ctx.gd_kv_reserve(d.ref, C.byref(s), d.copies, d.n, d.pos_out)
        table, refs = ctx.get(d.table, d.m.table.shape, I32), ctx.get(d.refs, 70000, I32)
        assert np.array_equal(refs, np.bincount(table[table >= 0], minlength=70000)) and refs.max() == 1


# (Around 1024, 4096 and 16384 pages, 2048 and 6144 entries of the table, where other kernels take over.)
EDGES = [((40, 600, 16, 30000), 0), ((2, 3, 16, 300001), 1), ((200, 400, 16, 16000), 0), ((100, 300, 16, 16384), 1),
         ((100, 100, 16, 16385), 0), ((1, 65537, 16, 900), 1), ((20, 300, 16, 4096), 0), ((20, 308, 16, 4096), 1),
         ((20, 300, 16, 4097), 0), ((20, 102, 16, 1024), 0), ((20, 103, 16, 1024), 1), ((9, 50, 16, 1025), 0)]


@pytest.mark.parametrize("size,seed", [(s, i) for s in SIZES for i in range(3)] + EDGES, ids=str)
def test_compact(ctx, size, seed):
    rng = np.random.default_rng(seed)
    with Device(ctx, *size) as d:
        if seed < 2:
            filled(d, rng)
            d.m.refs[rng.integers(0, size[3], 3)] += 1          # held by the program
            d.set()
        elif size[0] * size[1] >= size[3] or size[3] == 1:      # full
            d.m.refs[:] = 1
            d.set()
        d.compact()
        d.compact()
        assert not len(d.m.compact()[0])


@pytest.mark.parametrize("n,n_pages", [(40, 900), (5000, 20000)])
def test_recordings(ctx, n, n_pages):
    """Reserving, releasing and closing up as recorded graphs, replayed in turn with calls between that
    grow the workspace and use it, every time as the model has it."""
    rng = np.random.default_rng(n)
    with Device(ctx, n, 3, 16, n_pages) as d:
        s = d.seqs([0] * n, [1] * n, True)
        gone, to = d.put(np.zeros(n // 3, I32)), d.put(np.zeros(n // 3, I32))
        calls = [lambda: ctx.gd_kv_reserve(d.ref, C.byref(s), d.copies, d.n, d.pos_out),
                 lambda: ctx.gd_kv_release(d.ref, gone, None, to, n // 3), lambda: ctx.gd_kv_compact(d.ref, d.moves, d.n)]
        graphs = []
        for call in calls:
            call()
            graphs.append(C.c_void_p())
            ctx.gd_graph_begin()
            call()
            ctx.gd_graph_end(C.byref(graphs[-1]))
        d.set()                                                 # (as it was)
        big = Device(ctx, 4, 4, 16, 200000)
        for i in range(4):
            pos = rng.integers(-1, 40, n)
            ctx.set(s.pos, pos.astype(I32))
            out, copies = d.m.reserve(pos.tolist(), [1] * n)
            ctx.gd_graph_launch(graphs[0])
            assert np.array_equal(ctx.get(d.pos_out, n, I32), out) and ctx.get(d.n, 1, I32)[0] == len(copies)
            d.same()
            filled(big, rng)
            big.compact()
            which = rng.integers(0, n, n // 3)
            ctx.set(gone, which.astype(I32))
            d.m.release(which, None, [0] * len(which))
            ctx.gd_graph_launch(graphs[1])
            d.same()
            big.reserve([0, 5, -1, 63], [1] * 4, True)
            moves, used = d.m.compact()
            ctx.gd_graph_launch(graphs[2])
            assert list(ctx.get(d.n, 2, I32)) == [len(moves), used]
            d.same()
        big.__exit__()
        for g in graphs:
            ctx.lib.gd_graph_destroy(g)


# ------------------------------------------------------------------ copies


@pytest.mark.parametrize("caches", [[(ga.F16, 8, 128, 16)], [(ga.I8, 3, 256, 48)] * 3, [(ga.F16, 1, 128, 7)] * 70,
                                    [(ga.I8, 8, 128, 16), (ga.F16, 2, 256, 16), (ga.I8, 1, 128, 16)],
                                    [(ga.F16, 8, 256, 500)], [(ga.I8, 1, 128, 2000)]], ids=["f16", "i8", "many", "mixed", "wide", "long"])
@pytest.mark.parametrize("count", ["null", "fewer", "more", "none", "negative"])
def test_copy_pages(ctx, caches, count):
    rng, n_pages, kvs, planes = np.random.default_rng(len(caches)), 23, (ga.KV * len(caches))(), []
    for kv, (dtype, hkv, hd, page) in zip(kvs, caches):
        ctx.gd_kv_alloc(dtype, hkv, hd, page, n_pages, C.byref(kv))
        size = page * hkv * hd * (2 if dtype == ga.F16 else 1)
        for p, n in ((kv.k, size), (kv.v, size), (kv.k_exp, page // 16 * hkv), (kv.v_exp, page // 16 * hkv)):
            if p:
                a = rng.integers(0, 256, (n_pages, n), dtype=np.uint8)
                ctx.set(p, a)
                planes.append((p, a))
    order = rng.permutation(n_pages)
    pairs = np.array([(order[0], order[1]), (order[0], order[2]), (-1, order[3]), (order[4], n_pages), (order[5], order[6]),
                      (order[7], -2**31), (order[8], order[9]), (order[0], order[10])], I32)
    n = {"null": 8, "fewer": 6, "more": 8, "none": 0, "negative": 0}[count]
    value = {"fewer": 6, "more": 2**31 - 1, "none": 0, "negative": -4}.get(count)
    dp, dn = ctx.put(pairs), None if value is None else ctx.put(np.array([value], I32))
    ctx.gd_kv_copy_pages(kvs, len(caches), dp, dn, 8)
    for p, a in planes:
        for src, dst in pairs[:n]:
            if 0 <= src < n_pages and 0 <= dst < n_pages:
                a[dst] = a[src]
        assert np.array_equal(ctx.get(p, a.shape, np.uint8), a)
    ctx.free(dp)
    if dn:
        ctx.free(dn)
    for kv in kvs:
        ctx.gd_kv_free(C.byref(kv))


def test_copy_pages_past_4_gib(ctx):
    """Pages whose places in a plane pass 2^32 bytes."""
    kv, page, hkv, hd = ga.KV(), 4096, 4, 128                   # 4 MiB a page and plane
    ctx.gd_kv_alloc(ga.F16, hkv, hd, page, 1100, C.byref(kv))
    rng, a = np.random.default_rng(3), []
    for p in (kv.k, kv.v):
        a.append(rng.integers(0, 256, page * hkv * hd * 2, dtype=np.uint8))
        ctx.set(p + 1097 * a[-1].size, a[-1])
    dp = ctx.put(np.array([[1097, 1], [1097, 1098]], I32))
    ctx.gd_kv_copy_pages(C.byref(kv), 1, dp, None, 2)
    for p, x in zip((kv.k, kv.v), a):
        for at in (1, 1097, 1098):
            assert np.array_equal(ctx.get(p + at * x.size, x.size, np.uint8), x)
        for at in (0, 2, 1096, 1099):
            assert not ctx.get(p + at * x.size, x.size, np.uint8).any()
    ctx.free(dp)
    ctx.gd_kv_free(C.byref(kv))


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("recorded", [False, True], ids=["eager", "recorded"])
def test_a_servers_rounds(ctx, dtype, recorded):
    """Two layers' caches under one table: prompts, branches, steps (reserve, copy, append,
    attend with capped scores; the recorded one replayed), ends, windows that pass, compaction. Every
    step's attention is held, bit for bit, to that of a cache of its own for each conversation, appended to
    in the same steps."""
    hd, H, hkv, P, n_seq, width, n_pages, layers = 128, 4, 2, 16, 6, 12, 60, 2
    rng, scale = np.random.default_rng(11), 0.1
    kvs, own = (ga.KV * layers)(), (ga.KV * layers)()
    for kv, pages in [(k, n_pages) for k in kvs] + [(k, n_seq * width) for k in own]:
        ctx.gd_kv_alloc(dtype, hkv, hd, P, pages, C.byref(kv))
    sc = ga.Scores(cap=8.0)
    with Device(ctx, n_seq, width, P, n_pages) as d:
        # The conversations' own caches: a page table that never changes, positions that do.
        fixed = d.put(np.arange(n_seq * width, dtype=I32).reshape(n_seq, width))
        pos, length = d.put(np.zeros(n_seq, I32)), np.full(n_seq, -1)
        x = [[d.put(np.zeros((200, h, hd), np.float32)) for h in (H, hkv, hkv)] for _ in range(layers)]
        outs = [d.put(np.zeros((200, H, hd), np.float32)) for _ in range(2 * layers)]
        start = d.put(np.zeros(n_seq + 1, I32))

        def describe(n_rows, tokens, table, at):
            return ga.Seqs(n_rows=n_rows, row_start=None if tokens else start, pos=at, rope_shift=None, page_table=table, n_seq=n_seq,
                           max_pages=width, max_len=width * P)

        def attend(cache, s, out):
            for i in range(layers):
                q, k, v = x[i]
                ctx.gd_kv_append_rope(C.byref(cache[i]), C.byref(s), None, 0, None, 0, k, hkv * hd, v, hkv * hd, ga.F32, 64, 1e6)
                ctx.gd_kv_attn_scored(C.byref(cache[i]), C.byref(s), q, H * hd, None, 0, out[i], ga.F32, H, scale, C.byref(sc))

        def step(n_rows, tokens):
            s = describe(n_rows, tokens, d.table, pos)
            ctx.gd_kv_reserve(d.ref, C.byref(s), d.copies, d.n, d.pos_out)
            ctx.gd_kv_copy_pages(kvs, layers, d.copies, d.n, n_seq)
            attend(kvs, describe(n_rows, tokens, d.table, d.pos_out), outs[:layers])

        def rows_in(rows, tokens):
            n = int(sum(rows))
            ctx.set(start, np.cumsum([0, *rows]).astype(I32))
            ctx.set(pos, length.astype(I32))
            for one in x:
                for p, h in zip(one, (H, hkv, hkv)):
                    ctx.set(p, rows_of(rng, (n, h, hd), False))
            for o in outs:
                ctx.set(o, np.full((n, H, hd), -7, np.float32))
            return n

        def check(n, rows, tokens):
            want, copies = d.m.reserve(length.tolist(), rows)
            assert np.array_equal(ctx.get(d.pos_out, n_seq, I32), want) and ctx.get(d.n, 1, I32)[0] == len(copies)
            d.same()
            attend(own, describe(n, tokens, fixed, pos), outs[layers:])
            assert np.array_equal(want, length)                 # (pages enough here)
            for i in range(layers):
                a, b = (ctx.get(o, (n, H, hd), np.float32) for o in (outs[i], outs[layers + i]))
                assert np.array_equal(a, b) and (a != -7).any()
            length[length >= 0] += np.array(rows)[length >= 0]

        def branch(src, dst):
            d.fork([src] * len(dst), dst, [int(length[src])] * len(dst))
            for b in dst:
                length[b] = length[src]
                for kv in own:                                  # the same history, copied whole
                    pairs = d.put(np.stack([src * width + np.arange(width), b * width + np.arange(width)], 1).astype(I32))
                    ctx.gd_kv_copy_pages(C.byref(kv), 1, pairs, None, width)

        def rounds(n, graph=None):
            for _ in range(n):
                k = rows_in([1] * n_seq, True)
                if graph:
                    ctx.gd_graph_launch(graph)
                else:
                    step(k, True)
                check(k, [1] * n_seq, True)

        length[:2] = 0                                          # two prompts, one in two chunks
        for rows in ([37, 20, 0, 0, 0, 0], [5, 0, 0, 0, 0, 0]):
            n = rows_in(rows, False)
            step(n, False)
            check(n, rows, False)
        rounds(2)
        graph = C.c_void_p()
        if recorded:
            ctx.gd_graph_begin()
            step(n_seq, True)
            ctx.gd_graph_end(C.byref(graph))
        g = graph if recorded else None
        branch(0, [2, 3, 4])
        rounds(7, g)
        branch(1, [5])
        d.release([3], None, [0])
        length[3] = -1
        rounds(20, g)
        d.release([0, 4], None, [0, 0])
        length[[0, 4]] = -1
        d.compact()
        ctx.gd_kv_copy_pages(kvs, layers, d.moves, d.n, n_pages)
        rounds(3, g)
        branch(5, [0, 4])
        d.release([2], None, [int(length[2]) - 9])              # back to an earlier position, and on
        length[2] -= 9
        rounds(6, g)
        d.compact()
        ctx.gd_kv_copy_pages(kvs, layers, d.moves, d.n, n_pages)
        rounds(2, g)
        if recorded:
            ctx.lib.gd_graph_destroy(graph)
    for kv in (*kvs, *own):
        ctx.gd_kv_free(C.byref(kv))
