"""What the entries of the cache's pages (gd_kv_fork, gd_kv_release, gd_kv_reserve,
gd_kv_compact, gd_kv_copy_pages) refuse, without a device (test_kv_cache_args.py's way)."""
import ctypes as C

import pytest

import gadeon_amd as ga
from test_kv_cache_args import BATCHES, CACHES, P, kv, refused

T = 4 * P                        # stands for a table


def pages(**kw):
    return ga.KVPages(**(dict(refs=P, table=T, n_pages=10, n_seq=3, max_pages=4, page_size=16) | kw))


def seqs(**kw):
    s = dict(n_rows=6, row_start=P, pos=P, rope_shift=None, page_table=T, n_seq=3, max_pages=4, max_len=0)
    return ga.Seqs(**(s | kw))


def call(name, pg, *args):
    return getattr(ga.load(), name)(None, pg if pg is not None else pages(), *args)


def fork(pg=None, **kw):
    return call("gd_kv_fork", pg, *(dict(src=P, dst=P, len=P, n=2) | kw).values())


def release(pg=None, **kw):
    return call("gd_kv_release", pg, *(dict(seq=P, frm=None, to=P, n=2) | kw).values())


def reserve(pg=None, s=None, **kw):
    return call("gd_kv_reserve", pg, s if s is not None else seqs(), *(dict(copies=P, n_copies=P, pos_out=P) | kw).values())


def compact(pg=None, **kw):
    return call("gd_kv_compact", pg, *(dict(moves=P, n_moves=P) | kw).values())


def copy(caches=None, **kw):
    caches = [kv()] if caches is None else caches
    a = dict(n=len(caches), pairs=P, n_pairs=P, most=4) | kw
    return ga.load().gd_kv_copy_pages(None, (ga.KV * len(caches))(*caches) if caches else None, *a.values())


PAGES = [(dict(refs=None), "null refs or table"), (dict(table=None), "null refs or table"), (dict(n_pages=0), "0 pages"),
         (dict(n_pages=-1), "-1 pages"), (dict(n_pages=1 << 31), "2147483648 pages"), (dict(n_seq=-1), "-1 sequences"),
         (dict(n_seq=1 << 24), "16777216 sequences"), (dict(max_pages=0), "of 0 pages"), (dict(page_size=0), "page size 0"),
         (dict(page_size=(1 << 24) + 1), "page size"), (dict(refs=P + 2), "4-byte aligned"), (dict(table=T + 1), "4-byte aligned")]


@pytest.mark.parametrize("entry", [fork, release, reserve, compact])
@pytest.mark.parametrize("what,words", PAGES)
def test_refused_pages(entry, what, words):
    refused(entry(pages(**what)), words)


@pytest.mark.parametrize("entry", [fork, release, reserve, compact])
def test_null_pages(entry):
    refused(entry(C.POINTER(ga.KVPages)()), "null pages")


@pytest.mark.parametrize("entry", [fork, release])
@pytest.mark.parametrize("n,words", [(-1, "-1 orders"), (65537, "65537 orders")])
def test_refused_orders(entry, n, words):
    refused(entry(n=n), words)


@pytest.mark.parametrize("call,words", [
    (lambda: fork(src=None), "null orders"), (lambda: fork(dst=None), "null orders"), (lambda: fork(len=None), "null orders"),
    (lambda: release(seq=None), "null orders"), (lambda: release(to=None), "null orders"), (lambda: fork(len=P + 1), "4-byte aligned"),
    (lambda: release(frm=P + 2), "4-byte aligned"), (lambda: release(pages(max_pages=1 << 27)), "over 134217728 pages each"),
    (lambda: fork(pages(max_pages=1 << 20), n=1 << 15), "32768 orders over 1048576 pages")])
def test_refused_order_arrays(call, words):
    refused(call(), words)


@pytest.mark.parametrize("what,words", [b for b in BATCHES if "page_table" not in b[0]])
def test_refused_sequences(what, words):
    refused(reserve(s=seqs(**what)), words)


@pytest.mark.parametrize("call,words", [
    (lambda: reserve(s=C.POINTER(ga.Seqs)()), "null sequences"), (lambda: reserve(s=seqs(page_table=P)), "not the pages'"),
    (lambda: reserve(s=seqs(page_table=None)), "page table"), (lambda: reserve(s=seqs(n_seq=2)), "not the pages'"),
    (lambda: reserve(s=seqs(max_pages=5)), "not the pages'"), (lambda: reserve(copies=None), "null copies"),
    (lambda: reserve(n_copies=None), "null copies"), (lambda: reserve(pos_out=None), "null copies"),
    (lambda: reserve(pos_out=P + 2), "4-byte aligned"), (lambda: reserve(s=seqs(n_rows=0, pos=None)), "null positions"),
    (lambda: compact(moves=None), "null moves"), (lambda: compact(n_moves=None), "null moves"),
    (lambda: compact(moves=P + 1), "4-byte aligned")])
def test_refused_outputs(call, words):
    refused(call(), words)


@pytest.mark.parametrize("what,words", CACHES)
def test_refused_caches(what, words):
    refused(copy([kv(**what)]), words)
    refused(copy([kv(), kv(**what)]), words)


@pytest.mark.parametrize("kw,words", [
    (dict(n=-1), "-1 caches"), (dict(caches=[], n=2), "2 caches"), (dict(caches=[kv(), kv(n_pages=11)]), "caches of 10 and 11 pages"),
    (dict(most=-1), "-1 pairs"), (dict(most=1 << 30), "1073741824 pairs"), (dict(pairs=None), "null pairs"),
    (dict(pairs=P + 2), "4-byte aligned"), (dict(n_pairs=P + 1), "4-byte aligned"),
    (dict(caches=[kv(page_size=1 << 24, n_head_kv=2, head_dim=128)], most=1), "pages of 4294967296 bytes")])
def test_refused_copies(kw, words):
    refused(copy(**kw), words)


@pytest.mark.parametrize("call", [fork, release, reserve, compact, copy, lambda: fork(n=0, src=None, dst=None, len=None),
                                  lambda: release(frm=P), lambda: copy(n_pairs=None), lambda: copy(most=0, pairs=None, n_pairs=None),
                                  lambda: copy([kv(), kv(dtype=ga.F16, head_dim=256, k_exp=None, v_exp=None)]),
                                  lambda: reserve(s=seqs(n_rows=3, row_start=None)),
                                  lambda: reserve(pages(n_seq=0), seqs(n_seq=0, n_rows=0), copies=None, pos_out=None),
                                  lambda: compact(pages(n_seq=0, table=None))])
def test_good_arguments_need_a_context_only(call):
    import os
    ga.load().gd_gguf_open(os.fsencode("/no/such/file"), C.byref(C.c_void_p()))
    before = ga.load().gd_last_error(None)
    assert call() == ga.GD_EINVAL and ga.load().gd_last_error(None) == before
