"""Where gd_kv_attn splits its rows' keys and where it leaves them whole, next to the borders, on
the CPU: the number of splits that it launches with, through the stand-in for the HIP runtime."""
import pytest

from test_kv_cache_memory import run

BODY = r"""
def splits(rows, positions, tokens, hd=128, hkv=8, window=0, n_seq=None, dtype=ga.I8, heads=2):
    kv = ga.KV(k=P, v=P, k_exp=P, v_exp=P, n_pages=10, dtype=dtype, n_head_kv=hkv, head_dim=hd, page_size=16)
    s = ga.Seqs(n_rows=rows, row_start=None if tokens else P, pos=P, rope_shift=None, page_table=P,
                n_seq=rows if tokens else n_seq, max_pages=2000, max_len=positions)
    i("launches").value = 0
    H = heads * hkv
    ctx.gd_kv_attn(kv, s, P, H * hd, None, 0, P + (1 << 32), ga.F32, H, 0.1, window, 4)
    n = i("splits").value
    assert i("launches").value == (2 if n > 1 else 1)
    return n
ctx = ga.Context(0)
"""


def test_tokens(tmp_path):
    """(256 CUs: the stand-in tells none, and that is what is taken.)"""
    run(tmp_path, BODY + r"""
# few blocks of 32 keys are left whole: 20 at head dim 128, 16 at 256
assert splits(1, 640, True) == 1 < splits(1, 641, True)
assert splits(1, 512, True, hd=256) == 1 < splits(1, 513, True, hd=256)
# up to 36 where the workgroups fill three quarters of the CUs, or seven eighths
assert splits(24, 1152, True) == 1 < splits(23, 1152, True) and splits(24, 1153, True) > 1
assert splits(31, 16000, True, window=1024) == 1 < splits(16, 16000, True, window=1024)
assert splits(56, 1152, True, hd=256, hkv=4) == 1 < splits(55, 1152, True, hd=256, hkv=4)
# any of a full chip's, times over
assert splits(256, 30000, True) == 1 < splits(255, 30000, True)
""")


def test_rows(tmp_path):
    """A unit is 128 columns (64 at head dim 256), a workgroup one of a kv head, a block 64 keys (32)."""
    run(tmp_path, BODY + r"""
chunks = lambda n, positions, window=0, hd=256: splits(16 * n, positions, False, hd=hd, hkv=4, window=window, n_seq=n, heads=4)
# 16 rows of 4 heads: a unit each, and one a sequence besides
assert chunks(60, 320) == 1 < chunks(4, 321)               # 10 blocks
assert chunks(30, 480) == 1 < chunks(29, 480)              # 15 blocks from 240 workgroups on
assert chunks(26, 16000, 400) == 1 < chunks(25, 16000, 400)               # .. under a window from 208
assert chunks(24, 0, 0) > 1                                # no bound known: the tables' 32000 positions
assert chunks(42, 768) > 1 and chunks(43, 768) == 1        # 24 blocks: 344
assert chunks(95, 769) > 1 and chunks(96, 769) == 1        # up to 128: 768
assert chunks(96, 4097) > 1 and chunks(256, 4097) == 1     # 2048
""")


@pytest.mark.parametrize("entry", ["append", "read", "attn"])
def test_more_ragged_sequences_than_are_walked(entry):
    import test_kv_cache_args as args
    call = getattr(args, entry)
    args.refused(call(s=args.seqs(n_rows=70000, n_seq=65537)), "65537 sequences with row_start (65536 at most)")
    args.refused(call(s=args.seqs(n_rows=6, n_seq=2**31 - 1)), "65536 at most")
    before = args.ga.load().gd_last_error(None)
    kw = {"append": dict(q=None, q_out=None), "read": {}, "attn": dict(q=args.P, out=args.P, gate=None)}[entry]
    for s in (args.seqs(n_rows=70000, n_seq=65536), args.seqs(n_rows=70000, n_seq=70000, row_start=None)):
        assert call(s=s, **kw) == args.ga.GD_EINVAL and args.ga.load().gd_last_error(None) == before   # the context alone
