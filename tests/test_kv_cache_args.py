"""What the paged-cache entries (gd_kv_alloc, gd_kv_append_rope, gd_kv_read,
gd_kv_attn) refuse.  They check their arguments before the context, so a null
context shows each message (gd_last_error(NULL)) without a device; good arguments
then fail for the context alone."""
import ctypes as C

import pytest

import gadeon_amd as ga

P = 1 << 20                      # stands for device pointers: refused calls read none


def kv(**kw):
    c = dict(k=P, v=P, k_exp=P, v_exp=P, n_pages=10, dtype=ga.I8, n_head_kv=2, head_dim=128, page_size=16)
    return ga.KV(**(c | kw))


def seqs(**kw):
    s = dict(n_rows=6, row_start=P, pos=P, rope_shift=None, page_table=P, n_seq=3, max_pages=4, max_len=0)
    return ga.Seqs(**(s | kw))


def append(c=None, s=None, **kw):
    a = dict(q=P, q_stride=512, q_out=2 * P, n_head=4, k=P, k_stride=256, v=P, v_stride=256, x=ga.F32, n_rot=64,
             base=1e6) | kw
    return ga.load().gd_kv_append_rope(None, c if c is not None else kv(), s if s is not None else seqs(), *a.values())


def read(c=None, s=None, **kw):
    a = dict(k_out=P, v_out=P, dtype=ga.F32) | kw
    return ga.load().gd_kv_read(None, c if c is not None else kv(), s if s is not None else seqs(), *a.values())


def attn(c=None, s=None, **kw):
    a = dict(q=P, q_stride=512, gate=P, gate_stride=512, out=2 * P, x=ga.F32, n_head=4, scale=0.1, window=0,
             n_sink=0) | kw
    return ga.load().gd_kv_attn(None, c if c is not None else kv(), s if s is not None else seqs(), *a.values())


def alloc(**kw):
    a = dict(dtype=ga.I8, n_head_kv=2, head_dim=128, page_size=16, n_pages=4, out=C.byref(ga.KV())) | kw
    return ga.load().gd_kv_alloc(None, *a.values())


def refused(rc, words):
    msg = ga.load().gd_last_error(None).decode()
    assert rc == ga.GD_EINVAL and words in msg, (rc, msg)


CACHES = [(dict(k=None), "null cache plane"), (dict(v_exp=None), "null cache plane"), (dict(dtype=3), "cache dtype 3"),
          (dict(dtype=ga.F32), "cache dtype 0"), (dict(head_dim=64), "head_dim 64"), (dict(n_head_kv=0), "n_head_kv 0"),
          (dict(page_size=24), "page size 24"), (dict(page_size=0), "page size 0"), (dict(n_pages=0), "0 pages"),
          (dict(n_pages=1 << 31), "pages"), (dict(n_pages=-1), "-1 pages"), (dict(v=P + 8), "16-byte aligned"),
          (dict(page_size=1 << 24, n_head_kv=4096, n_pages=1 << 30), "pages")]
BATCHES = [(dict(n_seq=-1), "-1 sequences"), (dict(n_rows=-1), "-1 rows"), (dict(n_rows=1 << 24), "16777216 rows"),
           (dict(row_start=None), "need row_start"), (dict(pos=None), "null positions"),
           (dict(page_table=None), "page table"), (dict(max_pages=0), "max_pages 0"), (dict(max_len=-1), "max_len -1")]


@pytest.mark.parametrize("entry", [append, read, attn])
@pytest.mark.parametrize("what,words", CACHES)
def test_refused_caches(entry, what, words):
    refused(entry(c=kv(**what)), words)


@pytest.mark.parametrize("entry", [append, read, attn])
@pytest.mark.parametrize("what,words", BATCHES)
def test_refused_sequences(entry, what, words):
    refused(entry(s=seqs(**what)), words)


@pytest.mark.parametrize("entry", [append, read, attn])
def test_null_structs(entry):
    refused(entry(c=C.POINTER(ga.KV)()), "null cache")
    refused(entry(s=C.POINTER(ga.Seqs)()), "null sequences")


@pytest.mark.parametrize("kw,words", [
    (dict(k=None), "null k or v"), (dict(v=None), "null k or v"), (dict(k_stride=255), "overlap"),
    (dict(v_stride=0), "overlap"), (dict(v_stride=-256), "overlap"), (dict(n_rot=63), "n_rot 63"),
    (dict(n_rot=130), "n_rot 130"), (dict(n_rot=-2), "n_rot -2"), (dict(base=0.0), "base"),
    (dict(base=float("nan")), "base"), (dict(base=float("inf")), "base"), (dict(q_out=None), "without q_out"),
    (dict(n_head=0), "0 heads"), (dict(q_stride=511), "overlap"), (dict(q_out=P, q_stride=1024), "in place"),
    (dict(x=ga.I8), "row dtype 2"), (dict(k_stride=1 << 31), "row stride"),
    (dict(k=3 * P, q_out=3 * P), "place of k or v"), (dict(v=2 * P + 512 * 4 * 6 - 16), "place of k or v"),
    (dict(v=2 * P - 16), "place of k or v")])
def test_refused_appends(kw, words):
    refused(append(**kw), words)


@pytest.mark.parametrize("kw,words", [(dict(k_out=None), "null output"), (dict(v_out=None), "null output"),
                                      (dict(dtype=ga.I8), "row dtype 2"), (dict(v_out=P + 2), "aligned")])
def test_refused_reads(kw, words):
    refused(read(**kw), words)


@pytest.mark.parametrize("kw,words", [
    (dict(q=None), "null q or out"), (dict(out=None), "null q or out"), (dict(n_head=3), "n_head 3"),
    (dict(n_head=0), "n_head 0"), (dict(q_stride=511), "strides"), (dict(gate_stride=500), "strides"),
    (dict(q_stride=514), "aligned"), (dict(q=P + 4), "aligned"), (dict(gate=P + 8), "aligned"),
    (dict(x=ga.F16, q_stride=516), "aligned"), (dict(window=-1), "window -1"), (dict(n_sink=-1), "n_sink -1"),
    (dict(scale=float("inf")), "scale"), (dict(x=7), "row dtype 7"), (dict(out=P, q_stride=1024), "in place"),
    (dict(out=P + 512), "in place"), (dict(gate=2 * P, gate_stride=1024), "in place")])
def test_refused_attention(kw, words):
    refused(attn(**kw), words)


def test_rows_by_heads_past_31_bits():
    n = (1 << 24) - 1
    refused(attn(c=kv(n_head_kv=256), s=seqs(n_rows=n, max_pages=1), n_head=256, q=P << 8, q_stride=1 << 15, gate=None,
                 out=P << 30), "16777215 rows of 256 heads")


def test_more_workgroups_than_a_launch_has():
    refused(attn(s=seqs(n_rows=1 << 23, n_seq=1 << 23, row_start=None)), "8388608 rows of 4 heads")
    refused(attn(c=kv(n_head_kv=4096), s=seqs(n_rows=1 << 13, n_seq=1 << 13), n_head=4096, q=P << 8, q_stride=1 << 19,
                 gate=None, out=P << 30), "8192 rows of 4096 heads")


@pytest.mark.parametrize("kw,words", [(dict(dtype=ga.F32), "cache dtype"), (dict(head_dim=96), "head_dim 96"),
                                      (dict(page_size=8), "page size 8"), (dict(n_pages=0), "0 pages"),
                                      (dict(out=None), "null out pointer")])
def test_refused_allocations(kw, words):
    refused(alloc(**kw), words)


@pytest.mark.parametrize("call", [append, read, attn, alloc, lambda: append(q=None, q_out=None, n_head=0),
                                  lambda: append(c=kv(dtype=ga.F16, k_exp=None, v_exp=None, page_size=7)),
                                  lambda: append(n_rot=0, base=0.0), lambda: attn(gate=None),
                                  lambda: attn(out=P), lambda: attn(out=P, q=3 * P),
                                  lambda: attn(s=seqs(n_rows=3, row_start=None)),
                                  lambda: attn(s=seqs(n_rows=0, n_seq=0, pos=None, page_table=None))])
def test_good_arguments_need_a_context_only(call):
    import os
    ga.load().gd_gguf_open(os.fsencode("/no/such/file"), C.byref(C.c_void_p()))      # leaves a message of its own
    before = ga.load().gd_last_error(None)
    assert call() == ga.GD_EINVAL and ga.load().gd_last_error(None) == before
