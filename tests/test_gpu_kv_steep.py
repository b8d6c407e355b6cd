"""gd_kv_attn_scored under slopes as steep as 32 bits hold and infinite ones: a row sees the nearest key
alone (its own), or, where they fall, the farthest; a slope that is no number makes its head so."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga
from test_gpu_kv_cache import Batch, raw, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("tokens", [True, False], ids=["tokens", "chunks"])
def test_steep_slopes(ctx, dtype, x16, hd, tokens):
    seqs = [(0, 1), (31, 1), (700, 1), (9000, 1)] if tokens else [(0, 70), (31, 3), (700, 20), (9000, 2)]
    slope = np.array([1e25, 1e37, 1e38, 3.4e38, np.inf, -1e25, -1e37, -3.4e38, -np.inf, np.nan], np.float32)
    H = len(slope)
    with Batch(ctx, seqs, dtype, 2, hd, 16, row_start=not tokens) as bt:
        KV = bt.fill()
        q = rows_of(bt.rng, (bt.n, H, hd), x16)
        do = bt.put(raw(q))
        for cap in (0.0, 5.0, 2000.0):
            sc = ga.Scores(cap=cap, slope=bt.put(slope))
            ctx.gd_kv_attn_scored(*bt.ref, bt.put(raw(q)), H * hd, None, 0, do, ga.F16 if x16 else ga.F32, H, 0.1, C.byref(sc))
            got = ctx.get(do, q.shape, q.dtype)
            assert np.isnan(got[:, -1]).all()
            for b, (p, r) in enumerate(seqs):
                V = np.repeat(KV[b][1], H // 2, 1)
                for i in range(r):
                    # (One weight of 1: the value, which halves hold; its quotient by the sum, and its product, a rounding each.)
                    want = np.where((slope > 0)[:-1, None], V[p + i, :-1], V[0, :-1])
                    assert (np.abs(got[bt.start[b] + i, :-1] - want) <= 2.0 ** -22 * np.abs(want)).all(), (cap, b, i)
