"""gd_kv_attn where keys are split and merged, against the statement in 64 bits of
test_gpu_kv_cache.py: results in the place of q or of the gate, bit for bit those of a
buffer of their own, for each merge (few rows and many, tokens and chunks, head
counts that fill its groups of heads and ones that do not); up to the most splits and
past them; and a cache of halves in pages of whole tiles, at every length."""
import numpy as np
import pytest

import gadeon_amd as ga
from test_gpu_kv_cache import ATTN, Batch, attend, bound, check_attention, raw, rows_of

pytestmark = pytest.mark.gpu

# (sequences, whether they are tokens): 1 to 4 rows, then over 1024 rows and heads.
FEW = {"token": [(3000, 1)], "tokens": [(2000, 1), (-1, 1), (3100, 1), (70, 1)], "chunk": [(2900, 3)]}


def many(which, H):
    rows = 1024 // H + 9
    if which == "tokens":
        return [(1400 + i if i % 8 == 5 else i, 1) for i in range(rows)]
    return [(2100, rows - 40), (5, 3), (-1, 2), (1700, 35)]


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd,H,hkv", [(128, 10, 2), (128, 8, 2), (128, 3, 3), (256, 6, 1), (256, 18, 2)])
@pytest.mark.parametrize("which", [*FEW, "many tokens", "many rows"])
def test_in_place_of_split_keys(ctx, dtype, x16, hd, H, hkv, which):
    seqs = FEW[which] if which in FEW else many(which.split()[1], H)
    with Batch(ctx, seqs, dtype, hkv, hd, 16, row_start="tok" not in which) as bt:
        KV, x = bt.fill(), ga.F16 if x16 else ga.F32
        q, g = (rows_of(bt.rng, (bt.n, H, hd), x16) for _ in "qg")
        dq, dg, do = (bt.put(raw(a)) for a in (q, g, np.zeros_like(q)))
        row, scale = H * hd, hd ** -0.5
        ctx.gd_kv_attn(*bt.ref, dq, row, dg, row, do, x, H, scale, 0, 0)
        out = ctx.get(do, q.shape, q.dtype)
        done = np.repeat([p >= 0 for p, _ in seqs], [r for _, r in seqs])
        for b, (p, r) in enumerate(seqs):                   # (some rows of each: the rest bit for bit below)
            at = slice(bt.start[b] + max(0, r - 3), bt.start[b] + r)
            want = attend(q[at], *KV[b], p + max(0, r - 3), np.float32(scale), 0, 0, g[at]) if p >= 0 else out[at]
            assert np.abs(out[at] - want).max() <= bound(q[at], *KV[b], scale, x16), (b, p, r)
        for again in range(3):                              # out over the gate, then over q
            ctx.set(dg, raw(g))
            ctx.gd_kv_attn(*bt.ref, dq, row, dg, row, dg, x, H, scale, 0, 0)
            got = ctx.get(dg, q.shape, q.dtype)
            assert np.array_equal(got[done], out[done]) and np.array_equal(got[~done], g[~done])
        ctx.set(dg, raw(g))
        ctx.gd_kv_attn(*bt.ref, dq, row, dg, row, dq, x, H, scale, 0, 0)
        got = ctx.get(dq, q.shape, q.dtype)
        assert np.array_equal(got[done], out[done]) and np.array_equal(got[~done], q[~done])


# Blocks of 32 keys (chunks of head dim 128: 64) of a long sequence, at least 8 (4 of head dim 256,
# 4 of chunks) a split, 64 splits at most: 24 to 47 splits at 6000 positions, 32 to 64 at 10000,
# 64 of more blocks each at 20000.
@pytest.mark.parametrize("cache,page", [(ga.I8, 16), (ga.F16, 16), (ga.F16, 20)], ids=["i8", "f16", "f16odd"])
@pytest.mark.parametrize("hd,H,hkv", [(128, 5, 1), (128, 8, 2), (256, 6, 1), (256, 12, 2)])
@pytest.mark.parametrize("T", [6000, 10000, 20000])
@pytest.mark.parametrize("rows", [0, 3], ids=["token", "chunk"])
def test_most_splits(ctx, cache, page, hd, H, hkv, T, rows):
    check_attention(ctx, [(T, max(rows, 1))], cache, hd == 256, hd, H, hkv, page, 0, 0, True, seed=T, row_start=rows > 0)


@pytest.mark.parametrize("cache", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16,hd,H", [(False, 128, 8), (True, 256, 6)])
def test_most_splits_of_many_rows(ctx, cache, x16, hd, H):
    """Over 1024 rows and heads in 50 splits or more of a long sequence, a short one beside it."""
    check_attention(ctx, [(17000, 1024 // H + 1), (3, 40)], cache, x16, hd, H, 1, 16, 0, 0, True)


@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd,H,hkv", [(128, 40, 8), (128, 3, 3), (256, 24, 4), (256, 18, 1)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("which", list(ATTN))
def test_pages_of_whole_tiles_of_halves(ctx, x16, hd, H, hkv, page, which):
    check_attention(ctx, ATTN[which], ga.F16, x16, hd, H, hkv, page, 0, 0, H != 3, seed=hd + H,
                    row_start=not which.startswith("tok"))


@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("which", list(ATTN))
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (100, 5), (64, 130), (1000, 1), (1 << 30, 3)])
def test_windows_over_pages_of_whole_tiles_of_halves(ctx, x16, which, window, sinks):
    for hd, H, hkv in ((128, 10, 2), (256, 6, 1)):
        check_attention(ctx, ATTN[which], ga.F16, x16, hd, H, hkv, 32, window, sinks, x16, seed=window,
                        row_start=not which.startswith("tok"))
