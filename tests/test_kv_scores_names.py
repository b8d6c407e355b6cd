"""What gd_kv_attn_scored refuses bears its own name, with scores and without any
(test_kv_scores_args.py's way)."""
import pytest

import gadeon_amd as ga
from test_kv_cache_args import P, attn, refused
from test_kv_scores_args import scored


@pytest.mark.parametrize("how", [dict(), dict(cap=5.0), dict(first=P)], ids=["plain", "cap", "first"])
@pytest.mark.parametrize("kw", [dict(q=None), dict(n_head=3), dict(window=-1)], ids=str)
def test_name(how, kw):
    mask = {k: v for k, v in kw.items() if k == "window"}
    refused(scored(how=ga.Scores(**how, **mask), **{k: v for k, v in kw.items() if k != "window"}), "gd_kv_attn_scored: ")
    refused(attn(**kw), "gd_kv_attn: ")
