"""Calls over paged caches whose sizes the library's numbers do not hold are refused, not cut off."""
import importlib

import pytest
import torch

mynn = importlib.import_module("my-nn-engine_amd")


def meta(*shape, t=torch.float16):
    return torch.empty(shape, dtype=t, device="meta")  # (sizes without memory)


def pools(n=4, H=1, P=32):
    return [meta(n, H, P, 32, t=torch.uint8) for _ in range(2)] + [meta(n, H, P, 1, t=t) for t in (torch.float16, torch.float16, torch.uint8, torch.uint8)]


BIG = (1 << 32) + 2  # an int's 2


@pytest.mark.parametrize("kw", [dict(pages=BIG), dict(n=BIG), dict(H=BIG), dict(P=BIG), dict(B=BIG), dict(Hq=BIG)], ids=str)
def test_sizes_past_an_int_are_refused(kw):
    a = dict(pages=2, n=4, H=1, P=32, B=1, Hq=2)
    a.update(kw)
    cache, table, lens = pools(a["n"], a["H"], a["P"]), meta(a["B"], a["pages"], t=torch.int32), meta(a["B"], t=torch.int32)
    q, k, cos = meta(a["B"], a["Hq"], 1, 64), meta(a["B"], a["H"], 1, 64), meta(8, 64)
    calls = [lambda: mynn.rope_append_paged(q, k, k, cos, cos, cache, table, lens), lambda: mynn.attention_paged_int4(q, cache, table, 1.0, lens),
             lambda: mynn.kv_rows_paged(cache, table, lens, 1)]
    space = lambda: mynn.attention_paged_int4_workspace(q, cache, table)
    # (a workspace does not ask how many pages there are; heads of q are looked at when the pools are known to be the GPU's, which these are not)
    for call in [space] if "Hq" in kw else calls if "n" in kw else calls + [space]:
        with pytest.raises(mynn.MynnError):
            call()
