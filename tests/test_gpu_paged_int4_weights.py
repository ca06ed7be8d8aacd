"""Attention over paged caches of 4 bits: its weights keep 20 bits and more on their way into the second product, whatever the rows of a kv head and the type are."""
import pytest
import torch

import paged_reference as ref
from test_gpu_attention_paged_int4 import cache, queries

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mynn():
    import gpu_util

    return gpu_util.mynn


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,group", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("S", [1, 4, 6, 16, 64, 140])
def test_weights_of_few_keys(mynn, dtype, D, group, S):
    """scores of a few hundredths and at most some 30 keys: what the bound allows besides the weights' rounding (32-bit sums of D products, of 30 weights) is 2^-16 of a result and less,
    so a weight rounded to 11 bits, 2^-12, does not pass it"""
    past = [0, 3, 30 - min(S, 30)]
    new = [min(S, 30), min(S, 7), min(S, 30)]
    pools, table = cache(3, 2, D, 64, group, dtype, [p + S for p in past], seed=S)
    q = queries(3, 16, S, D, dtype, size=0.02)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    want, slack = ref.attention(q, pools, table, D ** -0.5, past, new, False, 2.0 ** -20)
    ws = mynn.attention_paged_int4_workspace(q, pools, table)
    for workspace in (None, ws):
        ref.assert_close(mynn.attention_paged_int4(q, pools, table, D ** -0.5, dev(past), dev(new), False, workspace=workspace), want, slack)
