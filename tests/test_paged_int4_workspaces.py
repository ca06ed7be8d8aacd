"""Workspaces of attention over paged caches of 4 bits: none where no two workgroups can share a sequence."""
import importlib

import pytest

mynn = importlib.import_module("my-nn-engine_amd")

few = [(1, 8, 2), (2, 8, 2), (4, 32, 8), (1, 16, 1)]  # tokens, heads: up to 16 rows of a kv head


@pytest.mark.parametrize("S,Hq,Hkv", few)
def test_short_caches_need_none(S, Hq, Hkv):
    size = mynn.lib().mynn_attention_paged_int4_workspace_bytes
    for pages, rows in ((1, 32), (4, 32), (2, 64), (1, 128)):
        assert size(3, S, pages, rows, Hq, Hkv, 128) == 0
    for pages, rows in ((16, 32), (3, 256)):
        assert size(3, S, pages, rows, Hq, Hkv, 128) > 0


def test_a_call_over_a_short_cache_takes_no_workspace():
    """refused for its last argument but one, not for the workspace that is not there"""
    p = 0x10000
    a = [p, p, p, p, p, p, p, p, p, 4, 2, 32, 1.0, 1, 1, 1, p, None, 2, 1, 64, mynn.F16, 64, None, 0, p + 2]
    assert mynn.lib().mynn_attention_paged_int4(*a, None) == -1
    assert b"unaligned counters" in mynn.lib().mynn_last_error()
