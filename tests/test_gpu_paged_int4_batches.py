"""Attention over paged caches of 4 bits: batches that are more than the lanes of a wave several times over, tables far wider than the sequences, zero points with more than
their four bits."""
import pytest
import torch

import paged_reference as ref
from test_gpu_attention_paged_int4 import cache, check, queries
from test_gpu_rope_append_paged import same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mynn():
    import gpu_util

    return gpu_util.mynn


def lengths(n, most, seed):
    return [int(x) for x in torch.randint(0, most, (n,), generator=torch.Generator().manual_seed(seed))]


@pytest.mark.parametrize("B,Hkv,most", [(400, 2, 300), (330, 1, 90), (640, 1, 500), (900, 8, 40)])
def test_one_token_of_many_sequences(mynn, B, Hkv, most):
    """their lengths are added up 256 at a time behind the first 64"""
    past = lengths(B, most, B)
    past[0], past[-1], past[320] = most, most, 0
    pools, table = cache(B, Hkv, 64, 32, 64, torch.float16, [p + 1 for p in past], seed=70)
    check(mynn, queries(B, 4 * Hkv, 1, 64, torch.float16), pools, table, past, new=[int(i % 11 != 5) for i in range(B)])


@pytest.mark.parametrize("B,G,S,dtype", [(70, 4, 5, torch.float16), (66, 8, 8, torch.bfloat16), (130, 4, 6, torch.bfloat16), (65, 4, 20, torch.float16)])
def test_ranges_of_keys_in_batches_past_64(mynn, B, G, S, dtype):
    """many rows, few blocks of them over long tables: how long a range is, is found from lengths added up 64 at a time"""
    past = [int(p) % 60 for p in lengths(B, 1000, B)]
    past[1], past[64], past[B - 1] = 2200, 2900, 2500
    pools, table = cache(B, 1, 128, 128, 64, dtype, [p + S for p in past], seed=71)
    check(mynn, queries(B, G, S, 128, dtype), pools, table, past, new=[S - (i % 3 == 1) for i in range(B)])


@pytest.mark.parametrize("B,Hq,Hkv,D,S,past", [(1, 32, 4, 64, 100, 0), (1, 32, 4, 64, 300, 0), (1, 32, 4, 64, 777, 0), (1, 32, 8, 128, 300, 0), (3, 32, 8, 128, 60, 0), (2, 32, 8, 128, 64, 500),
                                               (4, 32, 8, 128, 8, 500), (4, 16, 16, 64, 1, 60), (3, 8, 8, 128, 1, 130)])
def test_tables_far_wider_than_the_sequences(mynn, B, Hq, Hkv, D, S, past):
    """as a program allocates them, for the longest sequence that it takes: other tiles and ranges than for a table that fits, the same results but for the order of sums"""
    dtype = torch.bfloat16
    lens = [past - 7 * b if past else 0 for b in range(B)]
    pools, table = cache(B, Hkv, D, 64, 64, dtype, [p + S for p in lens], seed=72)
    q = queries(B, Hq, S, D, dtype)
    wide = torch.full((B, 128), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    if S < 300:
        check(mynn, q, pools, wide, lens)
    past_dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    a, b = (mynn.attention_paged_int4(q, pools, t, D ** -0.5, past_dev) for t in (table, wide))
    # (each within 2^-11 of the 64-bit result's magnitudes before it is rounded, which is half a step of 2^-8: two half steps and twice that)
    size = mynn.kv_rows_paged(pools, table, torch.zeros_like(past_dev), past + S, past_dev + S)[1].abs().amax()  # (of the sequences' own rows: others hold anything)
    assert bool(torch.isfinite(size))
    assert ((a.float() - b.float()).abs() <= 2.0 ** -8 * a.float().abs() + 2.0 ** -9 * size).all()


@pytest.mark.parametrize("S,Hq", [(1, 8), (4, 8), (6, 8), (40, 8)])
@pytest.mark.parametrize("D,group", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_only_the_low_four_bits_of_a_zero_point_count(mynn, dtype, D, group, S, Hq):
    past = [200, 31]
    pools, table = cache(2, 2, D, 64, group, dtype, [p + S for p in past], seed=73)
    q = queries(2, Hq, S, D, dtype)
    want = check(mynn, q, pools, table, past)
    rows = mynn.kv_rows_paged(pools, table, torch.zeros(2, dtype=torch.int32, device="cuda"), 31 + S)
    for z in pools[4:]:
        z |= torch.randint(0, 16, z.shape, dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) << 4
    assert same_bits(check(mynn, q, pools, table, past), want)
    for a, b in zip(mynn.kv_rows_paged(pools, table, torch.zeros(2, dtype=torch.int32, device="cuda"), 31 + S), rows):
        assert same_bits(a, b)
