"""The paged cache where numbers are large: pages whose rows lie past 2^32 bytes of their plane,
positions up to 2^31, and many query heads to a kv head."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga
from test_gpu_kv_cache import attend, bound, check_attention, exponent, rotate

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("hd,page", [(128, 64), (256, 48)])
@pytest.mark.parametrize("which", ["tokens", "chunks"])
def test_pages_past_32_bits(ctx, dtype, hd, page, which):
    """Sequences in the last pages of planes of over 4 GiB: appended, read back, attended to."""
    hkv, H, size = 8, 16, 1 if dtype == ga.I8 else 2
    pages = (1 << 32) // (page * hkv * hd * size) + 40
    kv, bufs = ga.KV(), []
    put = lambda a: bufs.append(ctx.put(a)) or bufs[-1]  # noqa: E731
    ctx.gd_kv_alloc(dtype, hkv, hd, page, pages, C.byref(kv))
    try:
        rng = np.random.default_rng(hd)
        lens = [150, 37, 90]
        table = np.array([pages - 1 - 3 * np.arange(4), 7 - np.arange(4), pages - 3 - 3 * np.arange(4)], np.int32)
        first = [0, 0, 0]
        start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        N = int(start[-1])
        q, k, v = (rng.standard_normal((N, h, hd)).astype(np.float32) for h in (H, hkv, hkv))
        dt = put(table)
        s = ga.Seqs(n_rows=N, row_start=put(start), pos=put(np.array(first, np.int32)), rope_shift=None, page_table=dt,
                    n_seq=3, max_pages=4, max_len=150)
        dq, dk, dv, do = put(q), put(k), put(v), put(np.zeros_like(q))
        ctx.gd_kv_append_rope(kv, s, dq, H * hd, dq, H, dk, hkv * hd, dv, hkv * hd, ga.F32, 64, 1e6)
        ko, vo = put(np.zeros_like(k)), put(np.zeros_like(v))
        ctx.gd_kv_read(kv, s, ko, vo, ga.F32)
        K, V = (ctx.get(p, k.shape, np.float32).astype(np.float64) for p in (ko, vo))
        for b in range(3):
            r = slice(start[b], start[b + 1])
            turned = rotate(k[r], np.arange(lens[b]), 64, 1e6)
            step = 2.0 ** exponent(turned) * 0.5001 if dtype == ga.I8 else np.abs(turned).max() * 2.0 ** -10.9
            assert np.abs(K[r] - turned).max() <= step
            assert np.abs(V[r] - v[r]).max() <= (2.0 ** exponent(v[r]) * 0.5 if dtype == ga.I8 else np.abs(v[r]).max() * 2.0 ** -11)
        qr, scale = ctx.get(dq, q.shape, np.float32), hd ** -0.5
        if which == "tokens":                               # the last row of each
            rows = [start[b + 1] - 1 for b in range(3)]
            s = ga.Seqs(n_rows=3, row_start=None, pos=put(np.array(lens, np.int32) - 1), rope_shift=None, page_table=dt,
                        n_seq=3, max_pages=4, max_len=0)
            ctx.set(dq, np.ascontiguousarray(qr[rows]))
        ctx.gd_kv_attn(kv, s, dq, H * hd, None, 0, do, ga.F32, H, scale, 0, 0)
        got = ctx.get(do, (s.n_rows, H, hd), np.float32)
        for b in range(3):
            r = slice(start[b], start[b + 1])
            want = attend(qr[r], K[r], V[r], 0, np.float32(scale), 0, 0, None)
            mine, want = (got[b:b + 1], want[-1:]) if which == "tokens" else (got[r], want)
            assert np.abs(mine - want).max() <= bound(qr[r], K[r], V[r], scale, False), b
    finally:
        for p in bufs:
            ctx.free(p)
        ctx.gd_kv_free(C.byref(kv))


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("tokens", [True, False], ids=["tokens", "chunk"])
def test_positions_up_to_2_31(ctx, dtype, tokens):
    """Pages of 2^22 positions, the last of a table of 2^31: rows appended behind others and attended
    to under a window, sinks on a page that is not there; the last position of all is past the table's
    end (positions are below 2^31 - 1)."""
    hd, hkv, H, page, n_rot, window = 128, 1, 3, 1 << 22, 128, 50
    end, kv, bufs = (1 << 31) - 1, ga.KV(), []
    put = lambda a: bufs.append(ctx.put(a)) or bufs[-1]  # noqa: E731
    ctx.gd_kv_alloc(dtype, hkv, hd, page, 2, C.byref(kv))
    try:
        rng = np.random.default_rng(3)
        table = np.full((1, 512), -1, np.int32)
        table[0, 511] = 1
        dt, N = put(table), 100
        p0 = end - 99                                       # 99 rows there, and one that is not
        q, k, v = (rng.standard_normal((N, h, hd)).astype(np.float32) for h in (H, hkv, hkv))
        dq, dk, dv, do = put(q), put(k), put(v), put(np.zeros_like(q))
        s = ga.Seqs(n_rows=N, row_start=put(np.array([0, N], np.int32)), pos=put(np.array([p0], np.int32)), rope_shift=None,
                    page_table=dt, n_seq=1, max_pages=512, max_len=0)
        ctx.gd_kv_append_rope(kv, s, dq, H * hd, dq, H, dk, hkv * hd, dv, hkv * hd, ga.F32, n_rot, 1e4)
        qr = ctx.get(dq, q.shape, np.float32)
        p = p0 + np.arange(N)
        # (angles p base^-x in f64 are off by 2^-53 of themselves, 2^31 2^-53 of a radian)
        assert np.abs(qr - rotate(q, p, n_rot, 1e4)).max() <= np.abs(q).max() * 2 * (4 * 2.0 ** -24 + 2.0 ** -21)
        ko, vo = put(np.full_like(k, 9)), put(np.full_like(v, 9))
        ctx.gd_kv_read(kv, s, ko, vo, ga.F32)
        K, V = (ctx.get(x, k.shape, np.float32).astype(np.float64) for x in (ko, vo))
        assert not K[99].any() and not V[99].any() and K[:99].any(axis=(1, 2)).all()
        turned = rotate(k[:99], p[:99], n_rot, 1e4)
        step = 2.0 ** exponent(turned) * 0.501 if dtype == ga.I8 else np.abs(turned).max() * 2.0 ** -10.9
        assert np.abs(K[:99] - turned).max() <= step
        scale = hd ** -0.5
        if tokens:
            for r in (60, 98):
                s = ga.Seqs(n_rows=1, row_start=None, pos=put(np.array([p0 + r], np.int32)), rope_shift=None, page_table=dt,
                            n_seq=1, max_pages=512, max_len=0)
                ctx.gd_kv_attn(kv, s, dq + r * H * hd * 4, H * hd, None, 0, do, ga.F32, H, scale, window, 4)
                got = ctx.get(do, (1, H, hd), np.float32)
                want = attend(qr[r:r + 1], K[:99], V[:99], r, np.float32(scale), window, 0, None)
                assert np.abs(got - want).max() <= bound(qr[r:r + 1], K[:99], V[:99], scale, False)
        else:
            s = ga.Seqs(n_rows=50, row_start=put(np.array([0, 50], np.int32)), pos=put(np.array([p0 + 49], np.int32)),
                        rope_shift=None, page_table=dt, n_seq=1, max_pages=512, max_len=0)
            ctx.gd_kv_attn(kv, s, dq + 49 * H * hd * 4, H * hd, None, 0, do, ga.F32, H, scale, window, 4)
            got = ctx.get(do, (50, H, hd), np.float32)
            want = attend(qr[49:99], K[:99], V[:99], 49, np.float32(scale), window, 0, None)
            assert np.abs(got - want).max() <= bound(qr[49:99], K[:99], V[:99], scale, False)
    finally:
        for x in bufs:
            ctx.free(x)
        ctx.gd_kv_free(C.byref(kv))


@pytest.mark.parametrize("dtype", [ga.I8, ga.F16], ids=["i8", "f16"])
@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd,H,hkv", [(128, 300, 1), (256, 130, 1), (128, 64, 64), (256, 33, 3)])
def test_head_layouts(ctx, dtype, x16, hd, H, hkv):
    """More query heads to a kv head than a unit has columns, one each, and odd counts."""
    check_attention(ctx, [(0, 3), (37, 1), (5, 70), (700, 2)], dtype, x16, hd, H, hkv, 16, 0, 0, True)
    check_attention(ctx, [(0, 1), (37, 1), (1500, 1), (700, 1)], dtype, x16, hd, H, hkv, 16, 0, 0, True, row_start=False)
