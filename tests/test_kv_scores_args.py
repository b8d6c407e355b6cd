"""What gd_kv_attn_scored refuses, without a device (test_kv_cache_args.py's way)."""
import ctypes as C

import pytest

import gadeon_amd as ga
from test_kv_cache_args import BATCHES, CACHES, P, kv, refused, seqs


def scored(c=None, s=None, how=None, **kw):
    a = dict(q=P, q_stride=512, gate=P, gate_stride=512, out=2 * P, x=ga.F32, n_head=4, scale=0.1) | kw
    how = ga.Scores(cap=30.0, slope=P, first=P, prefix=P) if how is None else how
    return ga.load().gd_kv_attn_scored(None, c if c is not None else kv(), s if s is not None else seqs(), *a.values(), how)


@pytest.mark.parametrize("what,words", CACHES)
def test_refused_caches(what, words):
    refused(scored(c=kv(**what)), words)


@pytest.mark.parametrize("what,words", BATCHES)
def test_refused_sequences(what, words):
    refused(scored(s=seqs(**what)), words)


@pytest.mark.parametrize("kw,words", [
    (dict(q=None), "null q or out"), (dict(out=None), "null q or out"), (dict(n_head=3), "n_head 3"), (dict(q_stride=511), "strides"),
    (dict(gate_stride=500), "strides"), (dict(q=P + 4), "aligned"), (dict(x=ga.I8), "row dtype 2"),
    (dict(scale=float("nan")), "scale"), (dict(out=P, q_stride=1024), "in place")])
def test_refused_rows(kw, words):
    refused(scored(**kw), words)


@pytest.mark.parametrize("kw,words", [
    (dict(cap=-1.0), "cap -1"), (dict(cap=float("nan")), "cap nan"), (dict(cap=float("inf")), "cap inf"), (dict(cap=1e-31), "cap 1e-31"),
    (dict(cap=1e31), "cap 1e+31"), (dict(window=-1, cap=1.0), "window -1"), (dict(n_sink=-1, cap=1.0), "n_sink -1"),
    (dict(window=-1), "window -1"), (dict(slope=P + 2), "4-byte aligned"), (dict(first=P + 1), "4-byte aligned"),
    (dict(prefix=P + 3), "4-byte aligned")])
def test_refused_scores(kw, words):
    refused(scored(how=ga.Scores(**kw)), words)


def test_null_structs():
    refused(scored(how=C.POINTER(ga.Scores)()), "null scores")
    refused(scored(c=C.POINTER(ga.KV)()), "null cache")
    refused(scored(s=C.POINTER(ga.Seqs)()), "null sequences")


@pytest.mark.parametrize("how", [None, ga.Scores(), ga.Scores(cap=1e-30), ga.Scores(cap=1e30, window=5), ga.Scores(prefix=P),
                                 ga.Scores(first=P), ga.Scores(slope=P)])
def test_good_arguments_need_a_context_only(how):
    import os
    ga.load().gd_gguf_open(os.fsencode("/no/such/file"), C.byref(C.c_void_p()))
    before = ga.load().gd_last_error(None)
    assert scored(how=how) == ga.GD_EINVAL and ga.load().gd_last_error(None) == before
