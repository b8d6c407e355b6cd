"""Rows at positions past their page table, whose own keys are not there: of a window that starts
behind the table's last position too they see the sinks, and the prefix, up to that one."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga
from test_gpu_kv_cache import Batch, bound, raw, rows_of
from test_gpu_kv_scores import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,page,held", [(ga.F16, 10, 170), (ga.F16, 16, 176), (ga.I8, 16, 176), (ga.I8, 48, 192)])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("tokens", [True, False], ids=["tokens", "chunks"])
def test_sinks_and_prefixes(ctx, dtype, page, held, hd, x16, tokens):
    H, hkv, rows, scale = 4, 2, 1 if tokens else 3, hd ** -0.5
    with Batch(ctx, [(held - rows, rows)], dtype, hkv, hd, page, row_start=not tokens) as bt:
        ((K, V),) = bt.fill()
        assert bt.desc.max_pages * page == held
        q = rows_of(bt.rng, (rows, H, hd), x16)
        dq, do = bt.put(raw(q)), bt.put(raw(q))
        x = ga.F16 if x16 else ga.F32
        # (Windows that start in the block of keys that the table ends in, in the next and far behind.)
        for p, window in ((held + 2, 1), (held + 15, 10), (held + 200, 100), (5000, 40)):
            ctx.set(bt.desc.pos, np.array([p], np.int32))
            for seen in (held - 9, held, held + 3, 4000):
                # (All keys that are there, up to `seen` of them: nothing of the window is.)
                n = min(seen, held)
                want = attend(q, K[:n], V[:n], 10000, np.float32(scale), 0, 0, None)
                most = bound(q, K, V, scale, x16)
                ctx.gd_kv_attn(*bt.ref, dq, H * hd, None, 0, do, x, H, scale, window, seen)
                got = [ctx.get(do, q.shape, q.dtype)]
                for sinks, prefix in ((seen, None), (0, seen)):
                    sc = ga.Scores(window=window, n_sink=sinks, prefix=bt.put(np.array([prefix or 0], np.int32)))
                    ctx.gd_kv_attn_scored(*bt.ref, dq, H * hd, None, 0, do, x, H, scale, C.byref(sc))
                    got.append(ctx.get(do, q.shape, q.dtype))
                for g, what in zip(got, ("plain", "sinks", "prefix")):
                    assert np.abs(g - want).max() <= most, (p, window, seen, what)
