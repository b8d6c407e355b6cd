"""The exponent of an 8-bit block where its largest turned key lies next to 127 2^e: the
definition's, by the value in 64 bits, on either side of the border."""
import ctypes as C

import numpy as np
import pytest

import gadeon_amd as ga
from test_gpu_kv_cache import Batch, exponent, raw, rotate

pytestmark = pytest.mark.gpu
N = 64


def next_to_the_border(rng, x16, n_rot, base):
    """Positions and pairs (a, b) whose turn's first element lies within 4e-6 of 127, some of them
    under it and some over it, and by over 1e-9 (a phase in f64 moves it by less than 1e-11)."""
    kept = [np.zeros((0, 3))] * 2
    while min(map(len, kept)) < N // 2:
        p = rng.integers(1, 300, 400000)
        b = rng.uniform(-60, 60, p.size)
        b = (b.astype(np.float16) if x16 else b.astype(np.float32)).astype(np.float64)
        c, s = np.cos(p.astype(np.float64)), np.sin(p.astype(np.float64))
        with np.errstate(divide="ignore"):
            a = (127 + b * s) / c
        a = np.where(np.abs(a) < 126, a, 0)
        a = (a.astype(np.float16) if x16 else a.astype(np.float32)).astype(np.float64)
        y, other = a * c - b * s, np.abs(a * s + b * c)
        near = (np.abs(y - 127) < 4e-6) & (np.abs(y - 127) > 1e-9) & (other < 126)
        for i, side in enumerate((y > 127, y < 127)):
            at = near & side
            kept[i] = np.concatenate([kept[i], np.stack([p[at], a[at], b[at]], 1)])[:N // 2]
    return np.concatenate(kept)


@pytest.mark.parametrize("x16", [False, True], ids=["f32rows", "f16rows"])
@pytest.mark.parametrize("hd,n_rot,offset", [(128, 64, 0), (256, 64, 0), (128, 6, 0), (256, 256, 4)])
def test_exponents_next_to_a_border(ctx, x16, hd, n_rot, offset):
    rng, base, hkv = np.random.default_rng(n_rot + hd), 1e6, 2
    case = next_to_the_border(rng, x16, n_rot, base)
    p = case[:, 0].astype(int)
    up = 2.0 ** rng.integers(-3, 4, N)                      # borders of other exponents
    k = rng.uniform(-1, 1, (N, hkv, hd)).astype(np.float16 if x16 else np.float32)
    for h in range(hkv):                                    # (the first pair turns by the position itself)
        k[:, h, 0], k[:, h, n_rot // 2] = case[:, 1] * up, case[:, 2] * up
    k[:, 1, 0] *= -1
    k[:, 1, n_rot // 2] *= -1
    if n_rot < hd:                                          # on the border, but not turned
        k[3::4, :, hd - 1] = 127 * up[3::4, None]
    with Batch(ctx, [(int(x), 1) for x in p], ga.I8, hkv, hd, 16, row_start=False) as bt:
        # Rows before these, at steps of less, the same and more.
        old = rng.integers(-127, 128, (bt.pages, hkv, 16, hd)).astype(np.int8)
        e_old = rng.integers(-5, 6, (bt.pages, hkv, 1))
        for c, e in ((bt.kv.k, bt.kv.k_exp), (bt.kv.v, bt.kv.v_exp)):
            ctx.set(c, old)
            ctx.set(e, (e_old + 127).astype(np.uint8))
        flat = np.zeros(k.size + 8, k.dtype)                # (a row start off the wide accesses' alignment)
        flat[offset // k.itemsize:][:k.size] = k.ravel()
        d = bt.put(raw(flat)) + offset
        x = ga.F16 if x16 else ga.F32
        ctx.gd_kv_append_rope(*bt.ref, None, 0, None, 0, d, hkv * hd, d, hkv * hd, x, n_rot, base)
        codes, _, exps, _ = bt.planes()
        turned = rotate(k, p, n_rot, base)
        for b in range(N):
            pg, sl = bt.table[b, p[b] // 16], p[b] % 16
            for h in range(hkv):
                e = exponent(turned[b, h])
                if sl:
                    e = max(e, e_old[pg, h, 0])
                    was = np.rint(old[pg, h, :sl] * 2.0 ** (e_old[pg, h, 0] - e))
                    assert np.array_equal(codes[pg, h, :sl], was), (b, h)
                assert int(exps[pg, h, 0]) - 127 == e, (b, h, p[b], turned[b, h, 0])
                assert np.abs(codes[pg, h, sl] - turned[b, h] * 2.0 ** -e).max() <= 0.5001
                assert np.array_equal(codes[pg, h, sl + 1:], old[pg, h, sl + 1:])
