"""What gd_kv_release and its kin refuse of gd_kv_pages.keep, without a device
(test_kv_pages_args.py's way)."""
import pytest

import gadeon_amd as ga
from test_kv_cache_args import P, refused
from test_kv_pages_args import compact, fork, pages, release, reserve


@pytest.mark.parametrize("entry", [fork, release, reserve, compact])
def test_keep(entry):
    refused(entry(pages(keep=P + 2)), "keep must be 4-byte aligned")
    assert entry(pages(keep=P)) == ga.GD_EINVAL            # (for the context alone)
    assert "aligned" in ga.load().gd_last_error(None).decode()
