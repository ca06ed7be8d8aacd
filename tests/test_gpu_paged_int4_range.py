"""Attention over paged caches of 4 bits whose scales reach over their type: groups and rows of zeros (their scale is 1) beside small values, groups of a row far
from each other, values that stand for no number, scales that change along a sequence, keys and queries at opposite ends of bf16."""
import pytest
import torch

import paged_reference as ref
from test_gpu_attention_paged_int4 import cache, queries
from test_gpu_rope_append_paged import same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mynn():
    import gpu_util

    return gpu_util.mynn


def attention(q, pools, table, scale, past, new, causal=True):
    """softmax(q k scale) v in 64 bits, and how far a result may be from it before it is rounded to its type, column by column:

    A weight's error relative to itself: a score is a sum of D products of exact operands in 32 bits, scaled in a few more steps, (D + 8) half steps of 2^-24 of the
    sum of the magnitudes; its exponential's argument is rounded at the size of the largest score, the exponential good to 2^-22; on its way into the second product a
    weight keeps 20 bits or more; n keys' sums have n half steps, joins a few more.  Numerator and denominator have them both: twice their sum, times sum(p |v|) / sum(p).
    And absolute: where the second product takes its weights as fp16 numbers, these are in units in which a scale next to the largest weight is 2^4 (few rows) or 1 (more
    than 16 of a kv head) or more, so a small one is off by 2^-25 of these: 2^-29 or 2^-25 of its own scale times the largest weight.  In bf16 parts: 2^-100 and less of its
    scale times the largest weight, and below 2^-133 in units of 2^-8 or more, nothing."""
    B, Hq, S, D = q.shape
    Hkv, P = pools[0].shape[1], pools[0].shape[2]
    G, half = Hq // Hkv, 2.0 ** -24
    tiny = 2.0 ** (-28 if G * S <= 16 else -24)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    slack = torch.zeros_like(out)
    for b in range(B):
        n = S if new is None else new[b]
        length = past[b] + n
        (k, there), (v, _) = ref.rows_of(pools, 0, table, b, 0, length), ref.rows_of(pools, 1, table, b, 0, length)
        at = torch.arange(length, device=q.device)
        for i in range(n):
            seen = there & (at < (past[b] + i + 1 if causal else length))
            for h in range(Hkv):
                x, kk, vv = q[b, h * G:(h + 1) * G, i].double(), k[h][seen], v[h][seen]
                s = torch.mm(x, kk.t().contiguous()) * scale
                size = (torch.mm(x.abs(), kk.abs().t().contiguous()) * abs(scale)).amax(-1, keepdim=True)
                p = torch.softmax(s, -1)
                weight = (D + 8) * half * size + 4 * half * s.abs().amax(-1, keepdim=True) + 2.0 ** -22 + 2.0 ** -20 + (kk.shape[0] + 64) * half
                out[b, h * G:(h + 1) * G, i] = torch.mm(p, vv)
                slack[b, h * G:(h + 1) * G, i] = 2 * weight * torch.mm(p, vv.abs()) + tiny * p.amax(-1, keepdim=True) * vv.abs().sum(0) + kk.shape[0] * 2.0 ** -120
    return out, slack


def check(mynn, q, pools, table, past, new=None, causal=True, scale=None, bad=None):
    """bad: which results stand for no number (the 64-bit ones are taken without what makes them so)"""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")
    ws = mynn.attention_paged_int4_workspace(q, pools, table)
    got = mynn.attention_paged_int4(q, pools, table, scale, dev(past), dev(new), causal, workspace=ws)
    again = mynn.attention_paged_int4(q, pools, table, scale, dev(past), dev(new), causal)
    if bad is None:
        want, slack = attention(q, pools, table, scale, past, new, causal)
        assert same_bits(got, again)
    else:
        clean = [torch.where(torch.isfinite(p), p, torch.ones_like(p)) if p.is_floating_point() else p for p in pools]
        want, slack = attention(q, clean, table, scale, past, new, causal)
        assert torch.equal(torch.isfinite(got), ~bad) and torch.equal(torch.isfinite(again), ~bad)
        got, again = (torch.where(bad, want.to(q.dtype), x) for x in (got, again))
        assert same_bits(got, again)
    ref.assert_close(got, want, slack)
    return got


def put_values(pools, table, side, x, group):
    """rows [B, n, Hkv, D] in the place of each sequence's first n"""
    P = pools[0].shape[2]
    parts = ref.quantize4(x.to(pools[2].dtype), group, pools[2].dtype)
    r = torch.arange(x.shape[1])
    for b in range(x.shape[0]):
        for n, t in enumerate(parts):
            pools[2 * n + side][table[b].long().cpu()[r // P], :, (r % P)] = t[b].to(pools[0].device)


def made(B, Hkv, D, P, group, dtype, n, values, seed, keys=None):
    """a cache of B sequences of n rows, values (and keys) as given"""
    pools, table = cache(B, Hkv, D, P, group, dtype, [n] * B, seed=seed)
    put_values(pools, table, 1, values, group)
    if keys is not None:
        put_values(pools, table, 0, keys, group)
    return pools, table


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# few rows of a kv head, up to 32, and many; heads, groups
ROWS = [(1, 8), (4, 8), (6, 8), (40, 8)]
SHAPES = [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)]


@pytest.mark.parametrize("S,Hq", ROWS)
@pytest.mark.parametrize("D,group", [s for s in SHAPES if s[1] < s[0]])
@pytest.mark.parametrize("dtype,size", [(torch.float16, -10), (torch.bfloat16, -10), (torch.bfloat16, -24), (torch.bfloat16, -36), (torch.bfloat16, -60), (torch.bfloat16, -100)])
def test_a_group_of_zeros_beside_small_values(mynn, dtype, size, D, group, S, Hq):
    """columns of a head that are always zero: their groups' scale is 1, by the rule"""
    v = normal(1, 2, 300 + S, 2, D) * 2.0 ** size
    v[..., :group] = 0.0
    pools, table = made(2, 2, D, 64, group, dtype, 300 + S, v, 2)
    assert bool((pools[3][int(table[0, 0]), :, :, 0] == 1).all())
    got = check(mynn, queries(2, Hq, S, D, dtype), pools, table, [300, 120], new=[S, S])
    assert not got[..., :group].any()


@pytest.mark.parametrize("S,Hq", ROWS)
@pytest.mark.parametrize("D,group", SHAPES)
@pytest.mark.parametrize("dtype,size", [(torch.float16, -10), (torch.bfloat16, -30), (torch.bfloat16, -70), (torch.bfloat16, -110)])
def test_rows_of_zeros_beside_small_values(mynn, dtype, size, D, group, S, Hq):
    """a token whose values are zero, at the front, in the middle of a tile and among the last"""
    v = normal(3, 1, 300 + S, 2, D) * 2.0 ** size
    v[:, [0, 77, 290]] = 0.0
    pools, table = made(1, 2, D, 64, group, dtype, 300 + S, v, 4)
    check(mynn, queries(1, Hq, S, D, dtype), pools, table, [300])


@pytest.mark.parametrize("S,Hq", ROWS)
@pytest.mark.parametrize("D,group", [s for s in SHAPES if s[1] < s[0]])
@pytest.mark.parametrize("dtype,low,high", [(torch.float16, -8, 8), (torch.float16, -12, 13), (torch.bfloat16, 0, 28), (torch.bfloat16, 0, 36), (torch.bfloat16, -40, 40), (torch.bfloat16, -90, 110)])
def test_groups_of_a_row_far_from_each_other(mynn, dtype, low, high, D, group, S, Hq):
    v = normal(5, 2, 200 + S, 1, D)
    if dtype == torch.float16:
        v = v.clamp(-3.5, 3.5)
    v[..., group:2 * group] *= 2.0 ** high
    v[..., :group] *= 2.0 ** low
    v[..., 2 * group:] *= 2.0 ** low
    pools, table = made(2, 1, D, 32, group, dtype, 200 + S, v, 6)
    check(mynn, queries(2, Hq, S, D, dtype), pools, table, [200, 33], new=[S, S])


@pytest.mark.parametrize("S,Hq", ROWS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,group,scale_of_it,longest", [(d, g, s, 150) for d, g in SHAPES for s in (float("nan"), float("inf"))] + [(64, 32, float("nan"), 3000), (128, 64, float("inf"), 3000),
                                                                                                                                    (128, 32, float("nan"), 3000), (64, 64, float("inf"), 3000)])
def test_a_group_of_values_that_stands_for_no_number(mynn, dtype, D, group, S, Hq, scale_of_it, longest):
    """only its own columns are none, and only for the rows that see it; 3000: sequences that several workgroups share"""
    past = [longest, 40]
    v = normal(7, 2, longest + S, 2, D) * 2.0 ** -9
    pools, table = made(2, 2, D, 64, group, dtype, longest + S, v, 8)
    at, g = longest + S // 2, D // group - 1
    page, r = int(table[0, at // 64]), at % 64
    pools[3][page, 1, r, g] = scale_of_it
    pools[1][page, 1, r] = 0x5A
    pools[5][page, 1, r] = 0  # (codes 5 and 10: an infinite scale stands for infinities)
    bad = torch.zeros(2, Hq, S, D, dtype=torch.bool, device="cuda")
    bad[0, Hq // 2:, S // 2:, g * group:] = True
    check(mynn, queries(2, Hq, S, D, dtype), pools, table, past, new=[S, S], bad=bad)


@pytest.mark.parametrize("S,Hq", ROWS)
@pytest.mark.parametrize("D,group", [(64, 64), (128, 64)])
@pytest.mark.parametrize("dtype,way", [(torch.float16, (0, 12, -6)), (torch.float16, (-10, 6, 10)), (torch.bfloat16, (0, 20, -20)), (torch.bfloat16, (-50, 0, 30)), (torch.bfloat16, (40, -20, 0)),
                                       (torch.bfloat16, (-100, -60, -80)), (torch.bfloat16, (-100, 100, 0)), (torch.bfloat16, (90, -90, 3)), (torch.bfloat16, (10, 50, 100))])
def test_scales_that_change_along_a_sequence(mynn, dtype, way, D, group, S, Hq):
    """powers of two of its thirds; the keys of the thirds with small values have the larger scores, so that all of them count"""
    n = 900 + S
    third = torch.arange(n) * 3 // n
    v = normal(9, 1, n, 1, D) * (2.0 ** torch.tensor(way, dtype=torch.float64)[third])[None, :, None, None]
    if dtype == torch.float16:
        v = v.clamp(-6e4, 6e4)
    direction = normal(10, D)
    order = torch.tensor(way).argsort(descending=True).argsort().float()
    k = 0.3 * normal(11, 1, n, 1, D) + (order[third] * 4.0)[None, :, None, None] * direction / direction.norm()
    pools, table = made(1, 1, D, 128, group, dtype, n, v, 12, keys=k)
    q = (direction + 0.2 * normal(13, 1, Hq, S, D)).to(dtype).cuda()
    check(mynn, q, pools, table, [900], scale=0.5)
    check(mynn, q, pools, table, [900], scale=0.0)


@pytest.mark.parametrize("S,Hq", ROWS)
@pytest.mark.parametrize("D,group", SHAPES)
@pytest.mark.parametrize("key", [-118, -100, 100, 112, 120])
@pytest.mark.parametrize("scale", [0.125, -0.125])
def test_keys_and_queries_at_opposite_ends(mynn, D, group, S, Hq, key, scale):
    """their products are ordinary scores"""
    dtype, n = torch.bfloat16, 150 + S
    k = normal(14, 2, n, 2, D) * 2.0 ** key
    pools, table = made(2, 2, D, 64, group, dtype, n, normal(15, 2, n, 2, D), 16, keys=k)
    q = (normal(17, 2, Hq, S, D) * 2.0 ** -key).to(dtype).cuda()
    q[:, 0] *= 0.001  # (rows of their own sizes, a row of zeros)
    q[:, 1] = 0.0
    check(mynn, q, pools, table, [150, 31], new=[S, S], scale=scale)


@pytest.mark.parametrize("S,Hq", ROWS)
def test_scores_that_are_very_large(mynn, S, Hq):
    """keys of 2^100 and queries of about 1: one key has all the weight"""
    dtype, D, n = torch.bfloat16, 128, 100 + S
    k = normal(18, 1, n, 1, D).abs() * 2.0 ** 100
    pools, table = made(1, 1, D, 64, 64, dtype, n, normal(19, 1, n, 1, D), 20, keys=k)
    q = normal(21, 1, Hq, S, D).abs().to(dtype).cuda()
    got = mynn.attention_paged_int4(q, pools, table, 0.125, torch.tensor([100], dtype=torch.int32, device="cuda"))
    (k, _), (v, _) = (ref.rows_of(pools, side, table, 0, 0, n) for side in (0, 1))
    for i in range(S):
        s = torch.mm(q[0, :, i].double(), k[0, :101 + i].t().contiguous())
        top = s.topk(2, -1)
        clear = top.values[:, 0] > top.values[:, 1] * (1 + 2.0 ** -16)  # (sums of 128 positive products in 32 bits)
        assert bool(clear.any()) and torch.equal(got[0, clear, i], v[0][top.indices[clear, 0]].to(dtype))


@pytest.mark.parametrize("S,Hq", ROWS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_captured_and_replayed_over_scales_that_change(mynn, dtype, S, Hq):
    """lengths grow past rows of zeros and of values 2^-14 and 2^12 of the others': what fits fp16 at one replay does not at the next"""
    D, group, n = 128, 64, 1300
    v = normal(22, 2, n, 2, D)
    v[:, 400:600] *= 2.0 ** 12
    v[:, 700:720] = 0.0
    v[:, 800:1000] *= 2.0 ** -14
    pools, table = made(2, 2, D, 64, group, dtype, n, v.clamp(-6e4, 6e4), 23)
    q = queries(2, Hq, S, D, dtype)
    past, new = torch.tensor([0, 150], dtype=torch.int32, device="cuda"), torch.tensor([S, S], dtype=torch.int32, device="cuda")
    ws, out, plain = mynn.attention_paged_int4_workspace(q, pools, table), torch.empty_like(q), torch.empty_like(q)
    calls = lambda: (mynn.attention_paged_int4(q, pools, table, 0.1, past, new, workspace=ws, out=out), mynn.attention_paged_int4(q, pools, table, 0.1, past, new, out=plain))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    for step in range(6):
        graph.replay()
        torch.cuda.synchronize()
        want = mynn.attention_paged_int4(q, pools, table, 0.1, past, new)
        assert same_bits(out, want) and same_bits(plain, want)
        exact, slack = attention(q, pools, table, 0.1, past.tolist(), new.tolist())
        ref.assert_close(out, exact, slack)
        past += 190
