"""What memory and how many launches the entries of the cache's pages take, on the CPU, in the
process of test_kv_cache_memory.py with a stand-in for the HIP runtime."""
import re

import pytest

import test_kv_cache_memory as memory

SETUP = r"""
def pages(n_seq, width, n_pages):
    return ga.KVPages(refs=P, table=4 * P, n_pages=n_pages, n_seq=n_seq, max_pages=width, page_size=16)
def reserve(ctx, n_seq, n_pages, rows=0):
    s = ga.Seqs(n_rows=rows or n_seq, row_start=P if rows else None, pos=P, rope_shift=None, page_table=4 * P, n_seq=n_seq,
                max_pages=100, max_len=0)
    ctx.gd_kv_reserve(pages(n_seq, 100, n_pages), s, P, P, P)
def launched(call):
    i("launches").value, before = 0, i("mallocs").value
    call()
    return i("launches").value, i("mallocs").value - before
ctx = ga.Context(0)
"""


@pytest.fixture
def run(tmp_path, monkeypatch):
    # (Its look at attention kernels' arguments left out.)
    source = re.sub(r"if \(launches\+\+ % 2 == 0\) \{.*?\n    \}", "launches++;", memory.HIP, flags=re.S)
    assert source != memory.HIP
    monkeypatch.setattr(memory, "HIP", source)
    return lambda body: memory.run(tmp_path, SETUP + body)


def test_reserve(run):
    """Up to 4096 sequences and entries no memory; beyond, what the header says, once."""
    run(r"""
assert launched(lambda: reserve(ctx, 4096, 10**6)) == (1, 0)
assert launched(lambda: reserve(ctx, 100, 10**6, 60000)) == (1, 0)       # 3750 + 200 entries
assert launched(lambda: reserve(ctx, 4097, 10**6)) == (1, 1)
size = live[i("n_live").value - 1].size
assert 8 * 10**6 + 28 * 4097 <= size <= 8 * 10**6 + 28 * 4097 + MB, size
assert launched(lambda: reserve(ctx, 4097, 10**6)) == (1, 0)
assert launched(lambda: reserve(ctx, 100, 10**6, 64000)) == (1, 0)       # 4200 entries
""")


def test_a_recording_does_not_grow_the_workspace(run):
    run(r"""
ctx.gd_graph_begin()
reserve(ctx, 4096, 10**6)                                  # needs none
for call in (lambda: reserve(ctx, 5000, 1000), lambda: ctx.gd_kv_compact(pages(3, 100, 5000), P, P)):
    try:
        call()
        assert False
    except ga.GDError as e:
        assert e.code == ga.GD_ENOMEM and "recording" in str(e)
g = C.c_void_p()
assert ctx.lib.gd_graph_end(ctx.h, C.byref(g)) != 0        # discarded
reserve(ctx, 5000, 1000)
ctx.gd_graph_begin()
reserve(ctx, 5000, 1000)
ctx.gd_graph_end(C.byref(g))
held = i("n_live").value
ctx.gd_kv_compact(pages(3, 100, 10**6), P, P)              # a larger workspace beside the one that g holds
assert i("n_live").value == held + 1
ctx.lib.gd_graph_destroy(g)
assert i("n_live").value == held
""")


def test_compact_and_copies(run):
    run(r"""
for n_seq, width, n_pages, launches, mallocs in ((60, 100, 4096, 1, 0), (0, 1, 1, 1, 0), (62, 100, 4096, 2, 1), (3, 100, 16384, 2, 1),
                                                 (3, 100, 16385, 3, 1), (3, 100, 10**6, 3, 1), (3, 100, 16384, 2, 0)):
    assert launched(lambda: ctx.gd_kv_compact(pages(n_seq, width, n_pages), P, P)) == (launches, mallocs), n_pages
kv = lambda n: (ga.KV * n)(*[ga.KV(k=P, v=P, k_exp=P, v_exp=P, n_pages=10, dtype=ga.I8, n_head_kv=2, head_dim=128, page_size=16)] * n)
for n, launches in ((0, 0), (1, 1), (64, 1), (65, 2), (200, 4)):
    assert launched(lambda: ctx.gd_kv_copy_pages(kv(n) if n else None, n, P, P, 10)) == (launches, 0)
    assert launched(lambda: ctx.gd_kv_copy_pages(kv(n) if n else None, n, None, None, 0)) == (0, 0)
assert launched(lambda: ctx.gd_kv_fork(pages(3, 100, 10), P, P, P, 5)) == (1, 0)
assert launched(lambda: ctx.gd_kv_fork(pages(3, 100, 10), None, None, None, 0)) == (0, 0)
assert launched(lambda: ctx.gd_kv_release(pages(3, 100, 10), P, None, P, 5)) == (1, 0)
""")
