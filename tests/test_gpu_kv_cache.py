"""The paged cache of many sequences (gd_kv_append_rope, gd_kv_read, gd_kv_attn)
against restatements in 64 bits: a cache of f16 values or 8-bit codes, ragged
batches with idle and empty sequences, windows and sinks, pages that are not there,
stale and non-finite values where nobody looks, strides, replays.

Codes are the definition's, but where a value lies within 1e-6 of a step of the
border between two (a phase in f64 off by 1e-13 of a turn moves it by less):
there the neighbour passes.  Attention is held to what its arithmetic can lose:
scores to 2^-22 of sum |q k| scale (f16 hi + lo rows) and to hd / 16 + 8 roundings of
32-bit sums, each weight to that and 2^-21 for its exponential, numerator and
denominator alike, sums over L keys to L / 16 + 4 roundings; f16 rows to a rounding
of each weight and of the result too, 2^-11 each."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga

pytestmark = pytest.mark.gpu
NAN16 = 0x7e00


# ------------------------------------------------------------------ in 64 bits


def rotate(x, p, n_rot, base):
    """x [rows][heads][hd] at positions p [rows]."""
    h, y = n_rot // 2, x.astype(np.float64)
    ang = np.asarray(p, np.float64)[:, None, None] * np.float64(base) ** (-2.0 * np.arange(h) / max(n_rot, 1))
    a, b, c, s = y[..., :h].copy(), y[..., h:n_rot].copy(), np.cos(ang), np.sin(ang)
    y[..., :h], y[..., h:n_rot] = a * c - b * s, a * s + b * c
    return y


def exponent(x):
    top = min(np.abs(x).max(initial=0.0), 127 * 512.0)
    return next(e for e in range(-24, 10) if top <= 127 * 2.0 ** e)


def steps(x, e):
    """Values in steps of 2^e, before rounding."""
    return np.clip(np.asarray(x, np.float64) * 2.0 ** -e, -127, 127)


def attend(q, K, V, first, scale, window, sinks, gate):
    """q [n][H][hd] at positions first .., K and V [T][HKV][hd] (NaN rows: not there)."""
    n, H, hd = q.shape
    T, G = K.shape[0], H // K.shape[1]
    t, at = np.arange(T), first + np.arange(n)[:, None]
    seen = (t <= at) & ((t > at - window) | (t < sinks) if window else t <= at)
    seen &= ~np.isnan(K[:, 0, 0])
    out = np.zeros((n, H, hd))
    for h in range(H):
        k, v = np.nan_to_num(K[:, h // G]), np.nan_to_num(V[:, h // G])
        s = np.where(seen, q[:, h].astype(np.float64) @ k.T * scale, -np.inf)
        m = s.max(1, keepdims=True, initial=-np.inf)
        p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
        out[:, h] = p @ v / np.maximum(p.sum(1, keepdims=True), 1e-300)
    return out if gate is None else out / (1 + np.exp(-gate.astype(np.float64)))


def bound(q, K, V, scale, f16):
    """The most an output may be off, from the largest sum |q k| scale and value."""
    hd = q.shape[-1]
    k, v = np.abs(np.nan_to_num(K)), np.abs(np.nan_to_num(V)).max(initial=0)
    G = q.shape[1] // K.shape[1]
    A = max((np.abs(q[:, h].astype(np.float64)) @ k[:, h // G].T).max(initial=0) for h in range(q.shape[1])) * abs(scale)
    score = A * (2.0 ** -22 + (hd / 16 + 8) * 2.0 ** -24)
    return v * (2 * (score + 2.0 ** -21) + (K.shape[0] / 16 + 4) * 2.0 ** -24 + (2 * 2.0 ** -11 if f16 else 0))


# ------------------------------------------------------------------ on the device


class Batch:
    """Sequences [(pos, rows)] with a shuffled page table over a cache."""

    def __init__(self, ctx, seqs, dtype, hkv, hd, page, seed=0, spare=0, row_start=True, lead=0, trail=0):
        self.ctx, self.seqs, self.rng = ctx, seqs, np.random.default_rng(seed)
        self.dtype, self.hkv, self.hd, self.page = dtype, hkv, hd, page
        need = [-(-max(p + r, 0) // page) for p, r in seqs]
        self.pages, width = sum(need) + 2, max(need + [1]) + spare
        order = self.rng.permutation(self.pages).astype(np.int32)
        self.table, at = np.full((len(seqs), width), -1, np.int32), 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        rows = [r for _, r in seqs]
        self.start = (lead + np.cumsum([0] + rows)).astype(np.int32)
        self.n = int(self.start[-1]) + trail
        self.kv, self.bufs = ga.KV(), []
        ctx.gd_kv_alloc(dtype, hkv, hd, page, self.pages, C.byref(self.kv))
        self.desc = ga.Seqs(n_rows=self.n, row_start=self.put(self.start) if row_start else None,
                            pos=self.put(np.array([p for p, _ in seqs], np.int32)), rope_shift=None,
                            page_table=self.put(self.table), n_seq=len(seqs), max_pages=width, max_len=0)
        self.ref = (C.byref(self.kv), C.byref(self.desc))

    def put(self, a):
        self.bufs.append(self.ctx.put(a))
        return self.bufs[-1]

    def close(self):
        for p in self.bufs:
            self.ctx.free(p)
        self.ctx.gd_kv_free(C.byref(self.kv))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    # -- planes as arrays, and back
    def planes(self):
        if self.dtype == ga.F16:
            shape = (self.pages, self.page, self.hkv, self.hd)
            return [self.ctx.get(p, shape, np.float16) for p in (self.kv.k, self.kv.v)]
        shape = (self.pages, self.hkv, self.page, self.hd)
        return [self.ctx.get(p, shape, np.int8) for p in (self.kv.k, self.kv.v)] + [
            self.ctx.get(p, (self.pages, self.hkv, self.page // 16), np.uint8) for p in (self.kv.k_exp, self.kv.v_exp)]

    def fill(self, scale=1.0):
        """Unit normal cache values at all positions, NaN (an unread block's mark) elsewhere;
        -> K, V [T][HKV][hd] of each sequence in 64 bits."""
        rng, res = self.rng, []
        if self.dtype == ga.F16:
            planes = [np.full((self.pages, self.page, self.hkv, self.hd), np.nan, np.float16) for _ in "kv"]
        else:
            planes = [rng.integers(-128, 128, (self.pages, self.hkv, self.page, self.hd)).astype(np.int8) for _ in "kv"]
            planes += [np.full((self.pages, self.hkv, self.page // 16), 255, np.uint8) for _ in "kv"]
        for b, (p, r) in enumerate(self.seqs):
            T = max(p + r, 0)
            t = np.arange(T)
            page, slot = self.table[b, t // self.page], t % self.page
            one = []
            for c in range(2):
                x = rng.standard_normal((T, self.hkv, self.hd)) * scale
                if self.dtype == ga.F16:
                    planes[c][page, slot] = x.astype(np.float16)
                    one.append(x.astype(np.float16).astype(np.float64))
                    continue
                e = rng.integers(-7, -3, (-(-T // 16), self.hkv))
                code = np.rint(np.clip(x * 32, -127, 127)).astype(np.int8)
                planes[c][page, :, slot] = code
                planes[2 + c][page, :, slot // 16] = (e[t // 16] + 127).astype(np.uint8)
                one.append(code * 2.0 ** e[t // 16][..., None])
            res.append(one)
        for p, a in zip((self.kv.k, self.kv.v, self.kv.k_exp, self.kv.v_exp), planes):
            self.ctx.set(p, a)
        return res


def rows_of(rng, shape, f16):
    x = rng.standard_normal(shape)
    return x.astype(np.float16) if f16 else x.astype(np.float32)


def raw(x):
    return x.view(np.uint16) if x.dtype == np.float16 else x


# ------------------------------------------------------------------ append

SEQS = {
    "token": [(0, 1)],
    "tokens": [(17, 1), (0, 1), (15, 1), (1600, 1), (-1, 1), (31, 1)],
    "chunk": [(5, 100)],
    "aligned": [(32, 64)],
    "ragged": [(0, 33), (40, 0), (15, 2), (-7, 3), (100, 17), (16, 16), (2003, 5)],
}


def many(n):
    rng = np.random.default_rng(n)
    return [(int(rng.integers(0, 90)), int(rng.integers(0, 6))) for _ in range(n)]


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd,H,hkv,n_rot,page", [(128, 40, 8, 64, 16), (256, 6, 1, 256, 48), (128, 3, 3, 2, 32),
                                                  (256, 4, 2, 64, 16)])
@pytest.mark.parametrize("which", [*SEQS, "many"])
def test_append(ctx, dtype, x16, hd, H, hkv, n_rot, page, which):
    """Rows into a cache that already holds the positions before them: codes and
    exponents (or halves) by the definition, everything else as it was; then read back."""
    seqs = many(150) if which == "many" else SEQS[which]
    page = page if dtype == ga.I8 else page - 5             # pages that end inside a block
    base = 1e7 if hd == 128 else 1e6
    with Batch(ctx, seqs, dtype, hkv, hd, page, seed=hd + n_rot, row_start=which not in ("token", "tokens"),
               trail=0 if which.startswith("tok") else 3) as bt:
        bt.fill()
        before = bt.planes()
        rng = bt.rng
        q, k, v = (rows_of(rng, (bt.n, h, hd), x16) for h in (H, hkv, hkv))
        grow = rng.choice([0.01, 1.0, 30.0], (bt.n, hkv, 1))   # rows that raise their block's exponent, or not
        k, v = (k * grow).astype(k.dtype), (v * grow[::-1]).astype(v.dtype)
        dq, dk, dv = (bt.put(raw(a)) for a in (q, k, v))
        dqo = bt.put(np.full(q.shape, -77, q.dtype).view(raw(q).dtype))
        ctx.gd_kv_append_rope(*bt.ref, dq, H * hd, dqo, H, dk, hkv * hd, dv, hkv * hd, ga.F16 if x16 else ga.F32,
                              n_rot, base)
        qo = ctx.get(dqo, q.shape, q.dtype)
        after, want, slack = bt.planes(), [a.copy() for a in before], [np.zeros(a.shape, bool) for a in before[:2]]
        done = np.zeros(bt.n, bool)
        values = [np.zeros((bt.n, hkv, hd)) for _ in "kv"]
        for b, (p, r) in enumerate(seqs):
            if p < 0 or r == 0:
                continue
            rows = slice(bt.start[b], bt.start[b] + r)
            done[rows] = True
            kr, qr = rotate(k[rows], p + np.arange(r), n_rot, base), rotate(q[rows], p + np.arange(r), n_rot, base)
            # cos, sin, two products and a sum in 32 bits of rows of two such terms; then x's type
            size = np.abs(q[rows]).max() * 2
            assert np.abs(qo[rows] - qr).max() <= size * (4 * 2.0 ** -24 + (2.0 ** -11 if x16 else 0)), b
            for c, x in enumerate((kr, v[rows].astype(np.float64))):
                for i in range(r if dtype == ga.F16 else 0):
                    want[c][bt.table[b, (p + i) // page], (p + i) % page] = np.clip(x[i], -65504, 65504).astype(np.float16)
                t = p
                while dtype == ga.I8 and t < p + r:
                    end, pg = min(t // 16 * 16 + 16, p + r), bt.table[b, t // page]
                    for h in range(hkv):
                        new, s0 = x[t - p:end - p, h], t // 16 * 16 % page
                        e, off = exponent(new), t % 16
                        if off:
                            e0 = int(before[2 + c][pg, h, s0 // 16]) - 127
                            e = max(e, e0)
                            old = before[c][pg, h, s0:s0 + off].astype(np.float64)
                            want[c][pg, h, s0:s0 + off] = np.rint(old * 2.0 ** (e0 - e))
                        st = steps(new, e)
                        want[c][pg, h, s0 + off:s0 + off + end - t] = np.rint(st)
                        slack[c][pg, h, s0 + off:s0 + off + end - t] = np.abs(st - np.floor(st) - 0.5) < 1e-6
                        want[2 + c][pg, h, s0 // 16] = e + 127
                        values[c][rows][t - p:end - p, h] = np.rint(st) * 2.0 ** e
                    t = end
        assert (qo[~done] == -77).all()
        if dtype == ga.I8:
            for c in range(2):
                assert np.array_equal(after[2 + c], want[2 + c])
                off = np.abs(after[c].astype(int) - want[c])
                # -128 stands in blocks never written, whose codes may be anything
                assert off.max() <= 1 and not (off[~slack[c]] != 0).any(), c
        else:
            for c in range(2):
                # keys: f32 rotation (as q's), then half a step
                same = np.isnan(want[c]) == np.isnan(after[c])
                assert same.all()
                a, w = np.nan_to_num(after[c]).astype(np.float64), np.nan_to_num(want[c]).astype(np.float64)
                assert (np.abs(a - w) <= (np.abs(w) * 2.0 ** -10 + np.abs(k).max() * 2.0 ** -21 if c == 0 else 0)).all()
        # the appended rows as values, in both types
        for np_t, code in ((np.float32, ga.F32), (np.float16, ga.F16)):
            ko, vo = (bt.put(np.full((bt.n, hkv, hd), -9, np_t).view(raw(np.zeros(1, np_t)).dtype)) for _ in "kv")
            ctx.gd_kv_read(*bt.ref, ko, vo, code)
            for c, d in enumerate((ko, vo)):
                got = ctx.get(d, (bt.n, hkv, hd), np_t)
                assert (got[~done] == -9).all()
                for b, (p, r) in enumerate(seqs):
                    for i in range(r if p >= 0 else 0):
                        pg, sl = bt.table[b, (p + i) // page], (p + i) % page
                        if dtype == ga.I8:
                            x = after[c][pg, :, sl] * 2.0 ** (after[2 + c][pg, :, sl // 16].astype(np.float64)[:, None] - 127)
                        else:
                            x = after[c][pg, sl]
                        assert np.array_equal(got[bt.start[b] + i], x.astype(np_t))


def test_append_strides_in_place_and_shift(ctx):
    """Rows of a fused projection by their strides, q turned in place, a rotation shift."""
    hd, H, hkv, n_rot, base = 128, 4, 2, 64, 1e6
    with Batch(ctx, [(9, 20), (3, 1)], ga.I8, hkv, hd, 16) as bt:
        width = (H + 2 * hkv) * hd + 24
        x = bt.rng.standard_normal((bt.n, width)).astype(np.float32)
        d = bt.put(x)
        bt.desc.rope_shift = bt.put(np.array([-13, 10**6], np.int32))
        at = [0, H * hd, (H + hkv) * hd]
        dq = bt.put(np.ascontiguousarray(x[:, :H * hd]))
        rows, outs = [d + 4 * a for a in at], []
        for src, stride, out in ((rows[0], width, bt.put(np.zeros((bt.n, H * hd), np.float32))), (dq, H * hd, dq)):
            ctx.gd_kv_append_rope(*bt.ref, src, stride, out, H, rows[1], width, rows[2], width, ga.F32, n_rot, base)
            outs.append(ctx.get(out, (bt.n, H, hd), np.float32))
        assert np.array_equal(*outs)
        p = np.concatenate([9 + np.arange(20) - 13, [10**6 + 3]])
        want = rotate(x[:, :H * hd].reshape(bt.n, H, hd), p, n_rot, base)
        assert np.abs(outs[0] - want).max() <= np.abs(x).max() * 2 * 4 * 2.0 ** -24
        ko, vo = (bt.put(np.zeros((bt.n, hkv, hd), np.float32)) for _ in "kv")
        ctx.gd_kv_read(*bt.ref, ko, vo, ga.F32)
        k = rotate(x[:, at[1]:at[2]].reshape(bt.n, hkv, hd), p, n_rot, base)
        step = 2.0 ** exponent(k)
        assert np.abs(ctx.get(ko, k.shape, np.float32) - k).max() <= step * 0.5001


@pytest.mark.parametrize("order", [(1.0, 50.0), (50.0, 1.0)], ids=["grows", "stays"])
def test_append_token_by_token(ctx, order):
    """32 single appends: each value within half a step, plus half the sum of the earlier
    steps' where the exponent grew (at most a step in all, as those halve); a rewind."""
    hd, hkv = 128, 2
    with Batch(ctx, [(0, 32)], ga.I8, hkv, hd, 32) as bt:
        x = bt.rng.standard_normal((32, hkv, hd)).astype(np.float32) * np.geomspace(*order, 32)[:, None, None].astype(np.float32)
        d, one = bt.put(x), bt.put(np.zeros(1, np.int32))
        s = ga.Seqs(n_rows=1, row_start=None, pos=one, rope_shift=None, page_table=bt.desc.page_table, n_seq=1,
                    max_pages=1, max_len=32)
        for t in list(range(32)) + [20, 21]:
            ctx.set(one, np.array([t], np.int32))
            ctx.gd_kv_append_rope(C.byref(bt.kv), C.byref(s), None, 0, None, 0, d + t * hkv * hd * 4, hkv * hd,
                                  d + t * hkv * hd * 4, hkv * hd, ga.F32, 0, 0.0)
        ko, vo = (bt.put(np.zeros((32, hkv, hd), np.float32)) for _ in "kv")
        ctx.gd_kv_read(*bt.ref, ko, vo, ga.F32)
        k, v = (ctx.get(p, x.shape, np.float32) for p in (ko, vo))
        assert np.array_equal(k, v)
        for b in range(2):
            for h in range(hkv):
                blk = x[16 * b:16 * b + 16, h]
                assert np.abs(k[16 * b:16 * b + 16, h] - blk).max() <= 2.0 ** exponent(blk)


def test_append_extremes(ctx):
    """Values past the range, of the least step and below, zeros, NaN and infinities."""
    hd, hkv = 128, 1
    rows = np.zeros((6 * 16, hkv, hd), np.float32)
    rows[0, 0, :3] = [1e30, -np.inf, 65024.0]
    rows[16, 0, :4] = [2.0 ** -24, 2.0 ** -25, 1.5 * 2.0 ** -24, -2.0 ** -30]
    rows[48, 0, :2] = [127.0, -126.5]
    rows[64, 0, 5], rows[65, 0, 6] = np.nan, 3.0
    rows[80, 0, 0] = 127.00001
    for dtype in (ga.I8, ga.F16):
        with Batch(ctx, [(0, 96)], dtype, hkv, hd, 32) as bt:
            d = bt.put(rows)
            ctx.gd_kv_append_rope(*bt.ref, None, 0, None, 0, d, hd, d, hd, ga.F32, 0, 0.0)
            ko, vo = (bt.put(np.zeros(rows.shape, np.float32)) for _ in "kv")
            ctx.gd_kv_read(*bt.ref, ko, vo, ga.F32)
            k, v = (ctx.get(p, rows.shape, np.float32) for p in (ko, vo))
            assert np.array_equal(k, v, equal_nan=True)
            if dtype == ga.F16:
                want = np.clip(rows, -65504, 65504).astype(np.float16).astype(np.float32)
                assert np.array_equal(k, want, equal_nan=True)
                continue
            assert list(k[0, 0, :3]) == [65024.0, -65024.0, 65024.0]
            assert list(k[16, 0, :4]) == [2.0 ** -24, 0.0, 2.0 ** -23, 0.0]
            assert not k[32:48].any()
            assert list(k[48, 0, :2]) == [127.0, -126.0]
            assert np.isnan(k[64:80]).all()
            assert k[80, 0, 0] == 128.0 and not k[81:].any()
            # a block that took a NaN stays so for its later rows, and starts anew with its first
            one = bt.put(np.array([66], np.int32))
            s = ga.Seqs(n_rows=1, row_start=None, pos=one, rope_shift=None, page_table=bt.desc.page_table, n_seq=1,
                        max_pages=bt.desc.max_pages, max_len=0)
            for at, nan in ((66, True), (64, False)):
                ctx.set(one, np.array([at], np.int32))
                ctx.gd_kv_append_rope(C.byref(bt.kv), C.byref(s), None, 0, None, 0, d, hd, d, hd, ga.F32, 0, 0.0)
                ctx.gd_kv_read(C.byref(bt.kv), C.byref(s), ko, vo, ga.F32)
                assert np.isnan(ctx.get(ko, (1, hd), np.float32)).all() == nan


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
def test_pages_that_are_not_there(ctx, dtype):
    """Rows for absent pages and past the table are dropped; read as zeros, not attended to."""
    hd, H, hkv, page = 128, 4, 2, 16
    with Batch(ctx, [(0, 70), (0, 10)], dtype, hkv, hd, page, trail=0) as bt:
        KV = bt.fill()
        table = bt.table.copy()
        table[0, 1], table[0, 3], table[1, 0] = -5, bt.pages, 2**31 - 1
        ctx.set(bt.desc.page_table, table)
        bt.desc.max_pages, before = 5, bt.planes()
        assert table.shape[1] == 5                          # 70 positions: five pages of 16, no more
        ctx.set(bt.desc.pos, np.array([12, 0], np.int32))  # rows 12 .. 81: two past the table
        q, x = (rows_of(bt.rng, (bt.n, h, hd), False) for h in (H, hkv))
        dq, dx, do = bt.put(q), bt.put(x), bt.put(np.full(q.shape, 5, np.float32))
        ctx.gd_kv_append_rope(*bt.ref, None, 0, None, 0, dx, hkv * hd, dx, hkv * hd, ga.F32, 0, 0.0)
        after = bt.planes()
        mine = [table[0, i] for i in (0, 2, 4)]
        others = [i for i in range(bt.pages) if i not in mine]
        for a, w in zip(after, before):
            assert np.array_equal(a[others].view(np.uint8), w[others].view(np.uint8))
        ko, vo = (bt.put(np.full((bt.n, hkv, hd), 5, np.float32)) for _ in "kv")
        ctx.gd_kv_read(*bt.ref, ko, vo, ga.F32)
        k = ctx.get(ko, x.shape, np.float32)
        gone = np.array([(12 + i) // 16 in (1, 3) or 12 + i >= 80 for i in range(70)] + [True] * 10)
        assert not k[gone].any() and k[~gone].any(axis=(1, 2)).all()
        scale = hd ** -0.5
        ctx.gd_kv_attn(*bt.ref, dq, H * hd, None, 0, do, ga.F32, H, scale, 0, 0)
        got = ctx.get(do, q.shape, np.float32)
        assert not got[70:].any()                          # its only page is not there
        K, V = (np.full((82, hkv, hd), np.nan) for _ in "kv")
        K[:12], V[:12] = (c[:12] for c in KV[0])
        if dtype == ga.I8:                                 # the block's old rows may have changed their step
            d2 = ga.Seqs(n_rows=12, row_start=bt.put(np.array([0, 12], np.int32)), pos=bt.put(np.zeros(1, np.int32)),
                         rope_shift=None, page_table=bt.desc.page_table, n_seq=1, max_pages=5, max_len=0)
            ctx.gd_kv_read(C.byref(bt.kv), C.byref(d2), ko, vo, ga.F32)
            K[:12], V[:12] = (ctx.get(p, (12, hkv, hd), np.float32) for p in (ko, vo))
            ctx.gd_kv_read(*bt.ref, ko, vo, ga.F32)
        K[12:][~gone[:70]] = k[:70][~gone[:70]]
        V[12:][~gone[:70]] = ctx.get(vo, x.shape, np.float32)[:70][~gone[:70]]
        want = attend(q[:70], K, V, 12, scale, 0, 0, None)
        assert np.abs(got[:70] - want).max() <= bound(q[:70], K, V, scale, False)


# ------------------------------------------------------------------ attention

ATTN = {
    "token": [(0, 1)],
    "tokens": [(17, 1), (0, 1), (700, 1), (-1, 1), (31, 1), (32, 1), (2500, 1)],
    "chunk": [(0, 150)],
    "later": [(611, 70)],
    "ragged": [(0, 33), (40, 0), (1015, 2), (-7, 3), (300, 67), (16, 16), (4000, 5)],
}
MASKS = [(0, 0), (1, 0), (40, 0), (100, 5), (64, 130), (1000, 1), (1 << 30, 3)]


def check_attention(ctx, seqs, dtype, x16, hd, H, hkv, page, window, sinks, gated, seed=0, row_start=True, max_len=0,
                    scale=None):
    with Batch(ctx, seqs, dtype, hkv, hd, page, seed=seed, row_start=row_start, lead=2 if row_start else 0,
               trail=3 if row_start else 0) as bt:
        KV = bt.fill()
        bt.desc.max_len = max_len
        q, gate = (rows_of(bt.rng, (bt.n, H, hd), x16) for _ in "qg")
        dq, dg = bt.put(raw(q)), bt.put(raw(gate))
        do = bt.put(np.full(q.shape, -77, q.dtype).view(raw(q).dtype))
        scale = hd ** -0.5 if scale is None else scale
        call = lambda: ctx.gd_kv_attn(*bt.ref, dq, H * hd, dg if gated else None, H * hd, do,  # noqa: E731
                                      ga.F16 if x16 else ga.F32, H, scale, window, sinks)
        call()
        got = ctx.get(do, q.shape, q.dtype)
        done = np.zeros(bt.n, bool)
        for b, (p, r) in enumerate(seqs):
            if p < 0 or r == 0:
                continue
            rows = slice(bt.start[b], bt.start[b] + r)
            done[rows] = True
            want = attend(q[rows], *KV[b], p, np.float32(scale), window, sinks, gate[rows] if gated else None)
            err, most = np.abs(got[rows] - want).max(), bound(q[rows], *KV[b], scale, x16)
            assert err <= most, (b, p, r, err, most)
        assert (got[~done] == -77).all()
        call()
        assert np.array_equal(ctx.get(do, q.shape, q.dtype), got)     # no order of arrival in it


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd,H,hkv,page", [(128, 40, 8, 16), (256, 24, 4, 48), (128, 3, 3, 32), (256, 18, 1, 16)])
@pytest.mark.parametrize("which", list(ATTN))
def test_attention(ctx, dtype, x16, hd, H, hkv, page, which):
    check_attention(ctx, ATTN[which], dtype, x16, hd, H, hkv, page if dtype == ga.I8 else page - 3, 0, 0,
                    gated=H != 3, seed=hd + H, row_start=not which.startswith("tok"))


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("which", list(ATTN))
@pytest.mark.parametrize("window,sinks", MASKS[1:])
def test_windows_and_sinks(ctx, dtype, which, window, sinks):
    for x16, hd, H, hkv in ((False, 128, 10, 2), (True, 256, 6, 1)):
        check_attention(ctx, ATTN[which], dtype, x16, hd, H, hkv, 16 if dtype == ga.I8 else 10, window, sinks,
                        gated=x16, seed=window, row_start=not which.startswith("tok"))


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("max_len", [1, 3000, 1 << 30])
def test_max_len_is_a_hint(ctx, dtype, max_len):
    for which in ("tokens", "ragged"):
        check_attention(ctx, ATTN[which], dtype, False, 128, 40, 8, 16, 0, 0, True, row_start=which == "ragged",
                        max_len=max_len)


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
def test_many_sequences(ctx, dtype):
    rng = np.random.default_rng(4)
    tokens = [(int(p), 1) for p in rng.integers(0, 400, 130)]
    chunks = [(int(rng.integers(0, 60)), int(rng.integers(0, 5))) for _ in range(130)]
    for seqs, start in ((tokens, False), (tokens, True), (chunks, True)):
        check_attention(ctx, seqs, dtype, True, 128, 10, 2, 16, 0, 0, False, row_start=start)


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("n", [130, 70])
def test_many_sequences_of_split_keys(ctx, dtype, n):
    """More sequences than a wave has lanes, a few of them long, idle ones among them."""
    rng = np.random.default_rng(n)
    long = [(3000, 1), (1800, 40), (2500, 7)]
    tokens = [(int(p), 1) for p in rng.integers(-5, 60, n)]
    chunks = [(int(rng.integers(-5, 60)), int(rng.integers(0, 3))) for _ in range(n)]
    for b, (p, r) in zip((0, n // 2, n - 1), long):
        tokens[b], chunks[b] = (p, 1), (p, r)
    for seqs, start in ((tokens, False), (tokens, True), (chunks, True)):
        check_attention(ctx, seqs, dtype, False, 128, 6, 2, 16, 0, 0, False, row_start=start)


@pytest.mark.parametrize("which", ["tokens", "ragged"])
def test_the_largest_window_is_none(ctx, which):
    outs = []
    for window, sinks in ((0, 0), (2**31 - 1, 0), (2**31 - 1, 2**31 - 1), (1, 2**31 - 1)):
        with Batch(ctx, ATTN[which], ga.I8, 2, 128, 16, row_start=which == "ragged") as bt:
            KV, start = bt.fill(), bt.start
            bt.desc.max_len = 4005
            q = rows_of(bt.rng, (bt.n, 4, 128), False)
            dq, do = bt.put(q), bt.put(np.zeros_like(q))
            ctx.gd_kv_attn(*bt.ref, dq, 512, None, 0, do, ga.F32, 4, 0.1, window, sinks)
            outs.append(ctx.get(do, q.shape, np.float32))
    assert outs[0].any() and all(np.array_equal(outs[0], o) for o in outs[1:3])
    for b, (p, r) in enumerate(ATTN[which]):                 # (maybe split elsewhere)
        rows = slice(start[b], start[b] + r) if which == "ragged" else slice(b, b + 1)
        if p >= 0 and r:
            assert np.abs(outs[3][rows] - outs[0][rows]).max() <= 2 * bound(q[rows], *KV[b], 0.1, False)


def test_row_starts_out_of_bounds(ctx):
    """Row starts before the first row and past the last one are taken for those; rows that no
    sequence has stay."""
    with Batch(ctx, [(0, 9), (40, 5), (7, 20)], ga.F16, 2, 128, 16) as bt:
        KV = bt.fill()
        q = rows_of(bt.rng, (bt.n, 4, 128), False)
        dq, do = bt.put(q), bt.put(np.full_like(q, -77))
        ctx.set(bt.desc.row_start, np.array([-2**31, 9, 14, 2**31 - 1], np.int32))
        ctx.gd_kv_attn(*bt.ref, dq, 512, None, 0, do, ga.F32, 4, 0.1, 0, 0)
        got = ctx.get(do, q.shape, np.float32)
        for b, rows in enumerate((slice(0, 9), slice(9, 14), slice(14, 34))):
            want = attend(q[rows], *KV[b], (0, 40, 7)[b], np.float32(0.1), 0, 0, None)
            assert np.abs(got[rows] - want).max() <= bound(q[rows], *KV[b], 0.1, False)
        ctx.set(bt.desc.row_start, np.array([9, 3, 14, 5], np.int32))        # no rows, 3 .. 13, no rows
        ctx.set(do, np.full_like(q, -77))
        ctx.gd_kv_attn(*bt.ref, dq, 512, None, 0, do, ga.F32, 4, 0.1, 0, 0)
        got = ctx.get(do, q.shape, np.float32)
        assert (got[:3] == -77).all() and (got[14:] == -77).all() and (got[3:14] != -77).all()


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0])
def test_scales(ctx, dtype, scale):
    for which in ("tokens", "later"):
        check_attention(ctx, ATTN[which], dtype, False, 128, 4, 2, 16, 0, 0, False, row_start=which == "later", scale=scale)


@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("which", ["tokens", "ragged"])
@pytest.mark.parametrize("ks,vs", [((-24, -20), (5, 10)), ((8, 10), (-24, -19)), ((-24, 10), (-24, 10))])
def test_steps_of_the_whole_range(ctx, x16, which, ks, vs):
    """8-bit blocks of all steps, every code among them, beside each other."""
    hd, H, hkv, seqs = 128, 4, 2, ATTN[which]
    with Batch(ctx, seqs, ga.I8, hkv, hd, 16, row_start=which == "ragged") as bt:
        rng, KV = bt.rng, [[], []]
        planes = [rng.integers(-127, 128, (bt.pages, hkv, 16, hd)).astype(np.int8) for _ in "kv"]
        planes += [(127 + rng.integers(*e, (bt.pages, hkv, 1))).astype(np.uint8) for e in (ks, vs)]
        for p, a in zip((bt.kv.k, bt.kv.v, bt.kv.k_exp, bt.kv.v_exp), planes):
            ctx.set(p, a)
        q = rows_of(rng, (bt.n, H, hd), x16)
        dq, do = bt.put(raw(q)), bt.put(raw(np.zeros_like(q)))
        # Scores of up to some tens, whatever the keys' steps.
        scale = float(np.float32(2.0 ** (-ks[1] - 6)))
        ctx.gd_kv_attn(*bt.ref, dq, H * hd, None, 0, do, ga.F16 if x16 else ga.F32, H, scale, 0, 0)
        got = ctx.get(do, q.shape, q.dtype)
        for b, (p, r) in enumerate(seqs):
            t = np.arange(max(p + r, 0))
            K, V = (planes[c][bt.table[b, t // 16], :, t % 16] * 2.0 ** (
                planes[2 + c][bt.table[b, t // 16], :, 0].astype(np.float64)[..., None] - 127) for c in range(2))
            rows = slice(bt.start[b], bt.start[b] + (r if p >= 0 else 0))
            want = attend(q[rows], K, V, p, scale, 0, 0, None)
            err = np.abs(got[rows] - want).max(initial=0)
            # f16 rows: results under 2^-14 are rounded to steps of 2^-24
            assert err <= bound(q[rows], K, V, scale, x16) + (2.0 ** -25 if x16 else 0), (b, err)


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd", [128, 256])
def test_non_finite_values_where_nobody_looks(ctx, dtype, x16, hd):
    """A NaN or infinite key and value reach the rows that see them, and no other: rows
    before them, rows whose window has left them, other heads, other sequences."""
    H, hkv, page, window, sinks = 4, 2, 16, 50, 3
    seqs, bad = [(0, 200), (130, 1), (60, 40)], 90
    with Batch(ctx, seqs, dtype, hkv, hd, page) as bt:
        KV = bt.fill()
        q = rows_of(bt.rng, (bt.n, H, hd), x16)
        dq, do, scale = bt.put(raw(q)), bt.put(raw(np.zeros_like(q))), hd ** -0.5
        planes = bt.planes()
        for which in (0, 1):
            for value in (np.nan, np.inf, -np.inf):
                p = [a.copy() for a in planes]
                first = bad
                for b in range(2):
                    pg = bt.table[b, bad // page]
                    if dtype == ga.F16:
                        p[which][pg, bad % page, 1, 7] = value
                    else:                                  # the mark of the block's 16 positions
                        p[2 + which][pg, 1, 0] = 255
                        first = bad // 16 * 16
                for d, a in zip((bt.kv.k, bt.kv.v, bt.kv.k_exp, bt.kv.v_exp), p):
                    ctx.set(d, a)
                ctx.gd_kv_attn(*bt.ref, dq, H * hd, None, 0, do, ga.F16 if x16 else ga.F32, H, scale, window, sinks)
                got = ctx.get(do, q.shape, q.dtype)
                last = first if dtype == ga.F16 else first + 15
                for b, (p0, r) in enumerate(seqs):
                    rows = slice(bt.start[b], bt.start[b] + r)
                    want = attend(q[rows], *KV[b], p0, np.float32(scale), window, sinks, None)
                    at = p0 + np.arange(r)
                    sees = (at >= first) & (at < last + window) if b < 2 else np.zeros(r, bool)
                    fine = np.repeat(~sees[:, None], H, 1)
                    fine[:, :H // 2] = True                # head 0's kv head is untouched
                    err = np.abs(got[rows] - want)[fine]
                    assert np.isfinite(err).all() and err.max(initial=0) <= bound(q[rows], *KV[b], scale, x16), (which, value, b)
                    if which == 1 or dtype == ga.I8:
                        assert not np.isfinite(got[rows][~fine]).all(-1).any()


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
def test_in_place_and_strides(ctx, dtype):
    """out over q and over gate, and rows of a fused projection by their strides."""
    hd, H, hkv, seqs = 128, 4, 2, [(0, 90), (300, 3)]
    with Batch(ctx, seqs, dtype, hkv, hd, 16) as bt:
        bt.fill()
        x = bt.rng.standard_normal((bt.n, 2 * H * hd + 8)).astype(np.float32)
        d, row = bt.put(x), H * hd
        q, g = bt.put(np.ascontiguousarray(x[:, :row])), bt.put(np.ascontiguousarray(x[:, row:2 * row]))
        outs = []
        for qp, qs, gp, gs, out in ((d, 2 * row + 8, d + row * 4, 2 * row + 8, bt.put(np.zeros((bt.n, row), np.float32))),
                                    (d, 2 * row + 8, g, row, g), (q, row, d + row * 4, 2 * row + 8, q)):
            ctx.gd_kv_attn(*bt.ref, qp, qs, gp, gs, out, ga.F32, H, hd ** -0.5, 0, 0)
            outs.append(ctx.get(out, (bt.n, row), np.float32))
        assert outs[0].any() and np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
def test_a_conversation_and_its_replays(ctx, dtype):
    """Prompts of three sequences, then tokens: append and attend in a recorded graph,
    replayed with positions and rows changed in place, eager calls and syncs between;
    every step against 64 bits on what the cache holds, and against the eager calls bit for bit."""
    hd, H, hkv, n_rot, base, page, steps = 128, 10, 2, 64, 1e6, 16, 12
    prompts = [37, 5, 80]
    seqs = [(0, n + steps) for n in prompts]
    scale = hd ** -0.5

    def program(graph):
        rng, outs = np.random.default_rng(8), []
        with Batch(ctx, seqs, dtype, hkv, hd, page, seed=1) as bt:
            start = np.cumsum([0] + prompts).astype(np.int32)
            N = int(start[-1])
            first = ga.Seqs(n_rows=N, row_start=bt.put(start), pos=bt.put(np.zeros(3, np.int32)), rope_shift=None,
                            page_table=bt.desc.page_table, n_seq=3, max_pages=bt.desc.max_pages, max_len=80)
            one = ga.Seqs(n_rows=3, row_start=None, pos=bt.put(np.zeros(3, np.int32)), rope_shift=None,
                          page_table=bt.desc.page_table, n_seq=3, max_pages=bt.desc.max_pages, max_len=92)
            q, k, v = (rows_of(rng, (N, h, hd), False) for h in (H, hkv, hkv))
            dq, dk, dv = (bt.put(a) for a in (q, k, v))
            do = bt.put(np.zeros_like(q))

            def step(s):
                ctx.gd_kv_append_rope(C.byref(bt.kv), C.byref(s), dq, H * hd, dq, H, dk, hkv * hd, dv, hkv * hd, ga.F32,
                                      n_rot, base)
                ctx.gd_kv_attn(C.byref(bt.kv), C.byref(s), dq, H * hd, None, 0, do, ga.F32, H, scale, 30, 2)

            def held():
                ko, vo = (bt.put(np.zeros((bt.n, hkv, hd), np.float32)) for _ in "kv")
                ctx.gd_kv_read(*bt.ref, ko, vo, ga.F32)
                return [ctx.get(p, (bt.n, hkv, hd), np.float32) for p in (ko, vo)]

            def check(s, rows, lengths, at):
                got, cached = ctx.get(do, (rows, H, hd), np.float32), held()
                qr = ctx.get(dq, (rows, H, hd), np.float32)
                outs.append(got)
                for b in range(3):
                    K, V = (c[bt.start[b]:bt.start[b] + lengths[b]] for c in cached)
                    r = slice(start[b], start[b + 1]) if s is first else slice(b, b + 1)
                    want = attend(qr[r], K, V, at[b], np.float32(scale), 30, 2, None)
                    assert np.abs(got[r] - want).max() <= bound(qr[r], K, V, scale, False), (at, b)

            step(first)
            check(first, N, prompts, [0, 0, 0])
            g = C.c_void_p()
            if graph:
                ctx.set(one.pos, np.array(prompts, np.int32))
                ctx.gd_graph_begin()
                step(one)
                ctx.gd_graph_end(C.byref(g))
            for t in range(steps):
                at = [n + t for n in prompts]
                ctx.set(one.pos, np.array(at, np.int32))
                for d, h in ((dq, H), (dk, hkv), (dv, hkv)):
                    ctx.set(d, rows_of(rng, (3, h, hd), False))
                if graph:
                    ctx.gd_graph_launch(g)
                else:
                    step(one)
                check(one, 3, [a + 1 for a in at], at)
            if graph:
                ctx.lib.gd_graph_destroy(g)
        return outs

    for a, b in zip(program(False), program(True)):
        assert np.array_equal(a, b)


def test_recordings_that_share_a_workspace(ctx):
    """Partials past the attention scratch: two recordings replayed in turn with eager calls
    between them, the workspace grown by one after they were made."""
    def batch(seqs, H, seed):
        bt = Batch(ctx, seqs, ga.I8, 2, 128, 16, seed=seed)
        bt.fill()
        q = rows_of(bt.rng, (bt.n, H, 128), False)
        dq, do = bt.put(q), bt.put(np.zeros_like(q))

        def run(graph=None):
            ctx.set(do, np.zeros_like(q))
            if graph:
                ctx.gd_graph_launch(graph)
            else:
                call()
            return ctx.get(do, q.shape, np.float32)

        def call():
            ctx.gd_kv_attn(*bt.ref, dq, H * 128, None, 0, do, ga.F32, H, 0.1, 0, 0)
        return bt, call, run

    small, large = [batch([(3000, 60), (10, 4), (900, 90)], 8, 1), batch([(1500, 130)], 16, 2)], batch([(2000, 700)], 16, 3)
    try:
        want, graphs = [], []
        for _, call, run in small:
            want.append(run())
            g = C.c_void_p()
            ctx.gd_graph_begin()
            call()
            ctx.gd_graph_end(C.byref(g))
            graphs.append(g)
        big = large[2]()
        for _ in range(3):
            for (_, _, run), w, g in zip(small, want, graphs):
                assert w.any() and np.array_equal(run(g), w)
                assert np.array_equal(large[2](), big) and np.array_equal(run(), w)
        for g in graphs:
            ctx.lib.gd_graph_destroy(g)
    finally:
        for bt, _, _ in (*small, large):
            bt.close()


def test_f16_cache_is_the_other_entries_cache(ctx):
    """gd_kv_append's pool attended by gd_kv_attn, and the other way round gd_attn_paged's."""
    hd, H, hkv, page, T = 128, 8, 2, 16, 300
    with Batch(ctx, [(0, T)], ga.F16, hkv, hd, page) as bt:
        k, v = (rows_of(bt.rng, (T, hkv, hd), False) for _ in "kv")
        q = rows_of(bt.rng, (H, hd), False)
        dk, dv, dq, do = bt.put(k), bt.put(v), bt.put(q), bt.put(np.zeros_like(q))
        table = bt.desc.page_table
        s = ga.Seqs(n_rows=1, row_start=None, pos=bt.put(np.array([T - 1], np.int32)), rope_shift=None, page_table=table,
                    n_seq=1, max_pages=bt.desc.max_pages, max_len=T)
        part, scale = bt.put(np.zeros(H * 16 * (hd + 2), np.float32)), hd ** -0.5
        K, V = (a.astype(np.float16).astype(np.float64) for a in (k, v))
        want = attend(q[None], K, V, T - 1, scale, 0, 0, None)[0]
        for own in (False, True):
            if own:
                ctx.gd_fill_u32(bt.kv.k, 0, bt.pages * page * hkv * hd // 2)
                ctx.gd_kv_append_rope(*bt.ref, None, 0, None, 0, dk, hkv * hd, dv, hkv * hd, ga.F32, 0, 0.0)
            else:
                ctx.gd_kv_append(dk, dv, bt.kv.k, bt.kv.v, table, hkv * hd, 0, page, T)
            ctx.gd_kv_attn(C.byref(bt.kv), C.byref(s), dq, H * hd, None, 0, do, ga.F32, H, scale, 0, 0)
            assert np.abs(ctx.get(do, q.shape, np.float32) - want).max() <= bound(q[None], K, V, scale, False)
            ctx.gd_attn_paged(dq, bt.kv.k, bt.kv.v, table, None, do, part, hd, H, hkv, T, hkv * hd, page,
                              C.c_float(scale), 0, 0)
            assert np.abs(ctx.get(do, q.shape, np.float32) - want).max() <= bound(q[None], K, V, scale, False)
