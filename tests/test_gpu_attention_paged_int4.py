"""Attention over paged caches of 4 bits against 64 bits: few rows and many, sequences of all lengths, masks that leave nothing, pages that are
not there, values at the ends of their types."""
import pytest
import torch

import paged_reference as ref
from test_gpu_rope_append_paged import same_bits, tables

pytestmark = pytest.mark.gpu

# the weights' relative error on their way into the second product (test bound of paged_reference.attention): 16 rows and fewer a kv head, and results in fp16, keep 20 bits
# of them; more rows with results in bf16 round them to fp16
def weight_error(q, pools):
    return 2.0 ** -20 if q.dtype == torch.float16 or q.shape[1] // pools[0].shape[1] * q.shape[2] <= 16 else 2.0 ** -11


@pytest.fixture(scope="module")
def mynn():
    import gpu_util

    return gpu_util.mynn


def cache(B, Hkv, D, P, group, dtype, rows, seed=0, spare=2, size=1.0, pages=None):
    """pools of quantised normal values (some channels of the keys larger), a table in no order with -1 behind a sequence's rows; rows of a page behind a sequence's own
    hold anything, NaN scales among it"""
    g = torch.Generator().manual_seed(seed)
    need = [(r + P - 1) // P for r in rows]
    pages = pages or max(max(need), 1)
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((B, pages), -1, dtype=torch.int32)
    pools = list(ref.make_pools(n_pages, Hkv, P, D, dtype, 4, group, "cpu", seed))
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        for side in range(2):
            x = torch.randn(rows[b], Hkv, D, generator=g) * size
            if side == 0:
                x[..., ::17] *= 4.0
            parts = ref.quantize4(x.to(dtype), group, dtype)
            r = torch.arange(rows[b])
            for n, t in enumerate(parts):
                pools[2 * n + side][table[b].long()[r // P], :, r % P] = t
    return [p.cuda() for p in pools], table.cuda()


def queries(B, Hq, S, D, dtype, seed=1, size=1.0):
    return (torch.randn(B, Hq, S, D, generator=torch.Generator().manual_seed(seed)) * size).to(dtype).cuda()


def check(mynn, q, pools, table, past, new=None, causal=True, scale=None, twice=True):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")
    want, slack = ref.attention(q, pools, table, scale, past, new, causal, weight_error(q, pools))
    got = mynn.attention_paged_int4(q, pools, table, scale, dev(past), dev(new), causal)
    ref.assert_close(got, want, slack)
    if twice:  # with a kept workspace, twice: the same bits
        ws = mynn.attention_paged_int4_workspace(q, pools, table)
        for _ in range(2):
            assert same_bits(mynn.attention_paged_int4(q, pools, table, scale, dev(past), dev(new), causal, workspace=ws), got)
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,group", [(32, 4, 64, 64), (32, 4, 64, 32), (32, 8, 128, 128), (32, 8, 128, 64), (32, 8, 128, 32), (3, 1, 64, 64), (8, 8, 128, 64), (16, 1, 128, 128)])
@pytest.mark.parametrize("past", [[0], [30, 31, 32, 0, 127], [1000, 5]])
def test_one_token(mynn, dtype, Hq, Hkv, D, group, past):
    pools, table = cache(len(past), Hkv, D, 64, group, dtype, [p + 1 for p in past])
    check(mynn, queries(len(past), Hq, 1, D, dtype), pools, table, past)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,group,S,P", [
    (32, 8, 128, 32, 4, 128),    # 16 rows of a kv head
    (8, 8, 64, 64, 13, 32),
    (32, 4, 64, 32, 3, 32),      # 24
    (32, 8, 128, 128, 5, 256),   # 20
    (4, 1, 128, 64, 40, 64),     # 160
    (12, 4, 64, 64, 100, 32),    # 300
    (32, 1, 64, 64, 1, 32),      # one token, 32 rows
])
@pytest.mark.parametrize("causal", [True, False])
def test_several_tokens(mynn, dtype, Hq, Hkv, D, group, S, P, causal):
    past = [0, 77, 300]
    pools, table = cache(3, Hkv, D, P, group, dtype, [p + S for p in past], seed=2)
    check(mynn, queries(3, Hq, S, D, dtype), pools, table, past, causal=causal)
    check(mynn, queries(3, Hq, S, D, dtype), pools, table, past, new=[S, max(S // 2, 1), 0], causal=causal)


@pytest.mark.parametrize("S,Hq", [(1, 8), (5, 8), (70, 8)])
def test_rows_that_see_nothing_are_zeros(mynn, S, Hq):
    """empty sequences, none of the call's tokens, lengths below zero and past the cache, pages that are not there: some, and all of a sequence"""
    B, Hkv, D, P = 7, 2, 128, 32
    past = [0, 40, -3, 200, 2 ** 31 - 1, 100, -2 ** 31]
    rows = [S, 40 + S, S, 256, 256, 100 + S, 0]
    pools, table = cache(B, Hkv, D, P, 64, torch.float16, rows, seed=3, pages=8)
    table[1, 0], table[5, :] = pools[0].shape[0], -1
    q = queries(B, Hq, S, D, torch.float16)
    for new in (None, [S, 0, S, S, S, S, S], [0, 1, 1, 1, -4, 1, 1]):
        got = check(mynn, q, pools, table, past, new)
        assert not got[5].any() and not got[6].any()
        assert new is None or new[0] or not got[0].any()


@pytest.mark.parametrize("S", [1, 33])
def test_what_lies_behind_the_rows_does_not_count(mynn, S):
    """the same call over pools whose other bytes are something else"""
    past = [45, 3]
    pools, table = cache(2, 2, 64, 64, 32, torch.bfloat16, [p + S for p in past], seed=4)
    other, _ = cache(2, 2, 64, 64, 32, torch.bfloat16, [p + S for p in past], seed=4)
    for side in range(6):
        for b in range(2):
            other[side][int(table[b, 0]), :, past[b] + S:] = 0xFF if other[side].dtype == torch.uint8 else float("nan")
    q = queries(2, 8, S, 64, torch.bfloat16)
    lens = torch.tensor(past, dtype=torch.int32, device="cuda")
    a = mynn.attention_paged_int4(q, pools, table, 0.125, lens)
    assert torch.isfinite(a).all() and same_bits(a, mynn.attention_paged_int4(q, other, table, 0.125, lens))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales_of_either_sign(mynn, dtype, S, scale):
    """2.0: scores of some dozens, one key has nearly all the weight"""
    past = [150, 20]
    pools, table = cache(2, 2, 128, 64, 64, dtype, [p + S for p in past], seed=5)
    check(mynn, queries(2, 8, S, 128, dtype), pools, table, past, scale=scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("kv,qs", [(1e-3, 1.0), (200.0, 2.0 ** -8), (2e3, 2.0 ** -12)])
def test_large_and_small_values(mynn, dtype, S, kv, qs):
    past = [150, 20]
    pools, table = cache(2, 2, 128, 64, 32, dtype, [p + S for p in past], seed=6, size=kv)
    check(mynn, queries(2, 8, S, 128, dtype, size=qs), pools, table, past)


@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("kv,qs", [(1e30, 1e-28), (1e-30, 1e28)])
def test_values_that_only_bf16_reaches(mynn, S, kv, qs):
    past = [150, 20]
    pools, table = cache(2, 2, 128, 64, 64, torch.bfloat16, [p + S for p in past], seed=7, size=kv)
    check(mynn, queries(2, 8, S, 128, torch.bfloat16, size=qs), pools, table, past)


@pytest.mark.parametrize("dtype,big", [(torch.float16, 2.0 ** 12), (torch.bfloat16, 2.0 ** 60)])
@pytest.mark.parametrize("S", [1, 40])
def test_a_huge_value_row_without_weight_does_not_hide_the_others(mynn, dtype, big, S):
    """one row of values is `big` times the others', and its key next to opposite to every query: its weight times its values is nothing"""
    past = [90]
    D = 128
    pools, table = cache(1, 1, D, 64, 64, dtype, [90 + S], seed=8)
    direction = torch.randn(D, generator=torch.Generator().manual_seed(2))
    rows = {0: -8.0 * direction[None], 1: big * torch.randn(1, D, generator=torch.Generator().manual_seed(3))}
    for side, x in rows.items():
        for n, t in enumerate(ref.quantize4(x.to(dtype), 64, dtype)):
            pools[2 * n + side][int(table[0, 0]), 0, 37] = t[0].cuda()
    q = (direction + 0.1 * torch.randn(1, 8, S, D, generator=torch.Generator().manual_seed(4))).to(dtype).cuda()
    check(mynn, q, pools, table, past, scale=0.3)


def test_a_row_that_stands_for_nan_is_seen_and_only_by_those_who_see_it(mynn):
    for S, seen in ((1, 20), (40, 30)):
        pools, table = cache(2, 2, 128, 32, 64, torch.float16, [seen + S, seen + S], seed=9)
        at = seen + S // 2
        for side in (2, 3):
            pools[side][int(table[1, at // 32]), 1, at % 32, 0] = float("nan")
        q = queries(2, 4, S, 128, torch.float16)
        got = mynn.attention_paged_int4(q, pools, table, 0.1, torch.tensor([seen, seen], dtype=torch.int32, device="cuda"))
        bad = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
        bad[1, 2:, S // 2:] = True
        assert torch.equal(torch.isnan(got), bad)


def test_long_caches(mynn):
    """a long sequence among short ones: parts of it on many workgroups, joined"""
    past = [20000, 0, 300, 7]
    pools, table = cache(4, 2, 128, 256, 128, torch.bfloat16, [p + 1 for p in past], seed=10)
    check(mynn, queries(4, 16, 1, 128, torch.bfloat16), pools, table, past)
    pools, table = cache(1, 2, 64, 64, 32, torch.float16, [9000 + 20], seed=11)
    check(mynn, queries(1, 8, 20, 64, torch.float16), pools, table, [9000])


def test_many_sequences(mynn):
    """more of them than a wave has lanes"""
    g = torch.Generator().manual_seed(0)
    past = [int(x) for x in torch.randint(0, 400, (150,), generator=g)]
    pools, table = cache(150, 2, 64, 32, 64, torch.float16, [p + 1 for p in past], seed=12)
    check(mynn, queries(150, 8, 1, 64, torch.float16), pools, table, past)


@pytest.mark.parametrize("S", [1, 48])
def test_captured_and_replayed_over_growing_lengths(mynn, S):
    B, Hq, Hkv, D, P, dtype = 3, 8, 2, 128, 64, torch.bfloat16
    pools, table = cache(B, Hkv, D, P, 64, dtype, [1200, 1200, 1200], seed=13)
    q = queries(B, Hq, S, D, dtype)
    past = torch.tensor([0, 5, 300], dtype=torch.int32, device="cuda")
    new = torch.tensor([S, 1, S], dtype=torch.int32, device="cuda")
    ws, out = mynn.attention_paged_int4_workspace(q, pools, table), torch.empty_like(q)
    plain = torch.empty_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        mynn.attention_paged_int4(q, pools, table, 0.1, past, new, workspace=ws, out=out)
        mynn.attention_paged_int4(q, pools, table, 0.1, past, new, out=plain)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        mynn.attention_paged_int4(q, pools, table, 0.1, past, new, workspace=ws, out=out)
        mynn.attention_paged_int4(q, pools, table, 0.1, past, new, out=plain)
    for step in range(5):
        graph.replay()
        torch.cuda.synchronize()
        want = mynn.attention_paged_int4(q, pools, table, 0.1, past, new)
        assert same_bits(out, want) and same_bits(plain, want)
        full, slack = ref.attention(q, pools, table, 0.1, past.tolist(), new.tolist(), True, weight_error(q, pools))
        ref.assert_close(out, full, slack)
        past += 211


def test_on_two_streams_at_once(mynn):
    """each with a workspace of its own, and without any"""
    past = [3000, 100]
    pools, table = cache(2, 4, 128, 64, 64, torch.float16, [p + 1 for p in past], seed=14)
    q = [queries(2, 16, 1, 128, torch.float16, seed=s) for s in (20, 21)]
    lens = torch.tensor(past, dtype=torch.int32, device="cuda")
    want = [mynn.attention_paged_int4(x, pools, table, 0.1, lens) for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    ws = [mynn.attention_paged_int4_workspace(x, pools, table) for x in q]
    torch.cuda.synchronize()
    got = [[], []]
    for turn in range(6):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(mynn.attention_paged_int4(q[n], pools, table, 0.1, lens, workspace=ws[n] if turn % 2 else None))
    torch.cuda.synchronize()
    for n in range(2):
        for x in got[n]:
            assert same_bits(x, want[n])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32)])
def test_generation_prompt_then_tokens(mynn, dtype, D, group):
    """as a program uses them together: two prompts of their own lengths in one padded call, then tokens one by one, rows appended and attended to; the cache's rows read
    back and attended to in 64 bits give the same"""
    B, Hq, Hkv, P, S = 2, 8, 2, 32, 45
    pool = mynn.KvPool(20, P)
    pages = mynn.KvPages(pool, B, 128)
    pages.reserve(S + 6)
    pools, = pool.buffers(1, Hkv, D, dtype, kv_int4_group=group)
    table = torch.from_numpy(pages.table()).cuda()
    cos, sin = tables(128, D, dtype)
    g = torch.Generator().manual_seed(5)
    past = torch.zeros(B, dtype=torch.int32, device="cuda")
    new = torch.tensor([45, 21], dtype=torch.int32, device="cuda")
    for step in range(6):
        n = S if step == 0 else 1
        rows = torch.randn(B, n, (Hq + 2 * Hkv) * D, generator=g).to(dtype).cuda().view(B, n, -1, D).transpose(1, 2)
        fresh = new if step == 0 else None
        q = mynn.rope_append_paged(rows[:, :Hq], rows[:, Hq:Hq + Hkv], rows[:, Hq + Hkv:], cos, sin, pools, pages, past, fresh)
        got = mynn.attention_paged_int4(q, pools, pages, D ** -0.5, past, fresh)
        want, slack = ref.attention(q, pools, table, D ** -0.5, past.tolist(), None if fresh is None else fresh.tolist(), True, weight_error(q, pools))
        ref.assert_close(got, want, slack)
        k, v = mynn.kv_rows_paged(pools, pages, past, n, fresh)
        kr = ref.rotate(rows[:, Hq:Hq + Hkv], cos[past.long()[:, None].clamp(max=127) + torch.arange(n, device="cuda")], sin[past.long()[:, None] + torch.arange(n, device="cuda")])
        for b in range(B):
            m = n if fresh is None else int(fresh[b])
            for have, put in ((k, kr.to(dtype)), (v, rows[:, Hq + Hkv:])):
                span = (put[b, :, :m].float().unflatten(-1, (-1, group)).amax(-1).clamp_min(0) - put[b, :, :m].float().unflatten(-1, (-1, group)).amin(-1).clamp_max(0)) / 15
                # (a code at the end of the range is a step off at most, in a scale and a value that are rounded)
                assert ((have[b, :, :m].float() - put[b, :, :m].float()).abs().unflatten(-1, (-1, group)) <= span[..., None] * 1.2 + 1e-6).all()
        past += new if step == 0 else 1
    pages.close()
    pool.close()


@pytest.mark.parametrize("D,group", [(64, 32), (128, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("G,S", [(4, 1), (5, 1), (1, 5), (2, 4), (9, 1), (3, 3), (8, 2), (17, 1), (1, 16), (1, 17), (16, 4), (13, 5), (2, 64), (43, 3)])
def test_rows_of_a_kv_head_around_the_tiles(mynn, D, group, G, S):
    """4, 8, 16, 64 and 128 rows are a tile's: as many, and one more"""
    past = [0, 129, 511]
    pools, table = cache(3, 2, D, 64, group, torch.float16, [p + S for p in past], seed=30 + S)
    check(mynn, queries(3, 2 * G, S, D, torch.float16), pools, table, past, new=[S, max(S - 1, 1), S])


@pytest.mark.parametrize("S", [30, 130])
@pytest.mark.parametrize("causal", [True, False])
def test_ranges_of_keys_of_ragged_prompts(mynn, S, causal):
    """few blocks of rows over many keys: their ranges are on workgroups of their own, as many as a sequence's length asks for"""
    past = [5000, 0, 700, 63, 2600]
    pools, table = cache(5, 1, 128, 128, 128, torch.bfloat16, [p + S for p in past], seed=31)
    q = queries(5, 4, S, 128, torch.bfloat16)
    check(mynn, q, pools, table, past, new=[S, S, 1, 0, S - 1], causal=causal)
    check(mynn, q, pools, table, past, causal=causal)
    one = [t[:1].contiguous() for t in (q, table)]
    check(mynn, one[0], pools, one[1], past[:1], causal=causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,group", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("B,G,S,longest", [(2, 4, 5, 2300), (2, 8, 4, 2500), (130, 4, 8, 300), (130, 17, 1, 150), (2, 3, 7, 4000)])
def test_drafts(mynn, dtype, D, group, B, G, S, longest):
    """17 to 32 rows of a kv head, over long caches and in large batches: tiles of 128 keys; pages that are not there among them"""
    g = torch.Generator().manual_seed(B + S)
    past = [int(x) for x in torch.randint(0, longest // 4 if B > 2 else longest, (B,), generator=g)]
    past[0], past[1] = longest, 100
    pools, table = cache(B, 2, D, 32 if B > 2 else 128, group, dtype, [p + S for p in past], seed=60 + G)
    q = queries(B, 2 * G, S, D, dtype)
    new = [S - i % (S + 1) for i in range(B)]
    check(mynn, q, pools, table, past, new=new)
    table[0, 1] = -1
    check(mynn, q, pools, table, past, new=new, causal=False)
    check(mynn, q[:2], pools, table[:2].contiguous(), past[:2], twice=False)


def test_many_parts_of_one_sequence(mynn):
    """more than 64 of them in a join"""
    pools, table = cache(1, 1, 64, 256, 64, torch.float16, [60001], seed=32)
    for Hq in (4, 7, 16):
        check(mynn, queries(1, Hq, 1, 64, torch.float16), pools, table, [60000])


@pytest.mark.parametrize("dtype,B,Hq,Hkv,D,group,P,most", [
    (torch.float16, 130, 64, 16, 128, 128, 64, 700),   # 2080 (sequence, kv head)s: a wave each
    (torch.bfloat16, 300, 32, 8, 64, 32, 32, 300),
    (torch.bfloat16, 70, 256, 32, 64, 64, 128, 200),   # 8 rows
    (torch.float16, 260, 8, 8, 128, 32, 256, 900),     # one row, four groups
    (torch.float16, 64, 16, 16, 128, 64, 64, 511),     # 1024, and caches of 512 rows
    (torch.bfloat16, 64, 32, 8, 128, 128, 32, 127),    # 512, and caches of 128
])
def test_a_wave_for_each_sequence_and_kv_head(mynn, dtype, B, Hq, Hkv, D, group, P, most):
    g = torch.Generator().manual_seed(B)
    past = [int(x) for x in torch.randint(0, most, (B,), generator=g)]
    past[0], past[1], past[-1] = most, 0, 1
    pools, table = cache(B, Hkv, D, P, group, dtype, [p + 1 for p in past], seed=40)
    table[B // 2, 0] = -1
    q = queries(B, Hq, 1, D, dtype)
    check(mynn, q, pools, table, past, new=[int(i % 7 != 3) for i in range(B)])


def test_one_workspace_for_calls_of_every_shape(mynn):
    """kept from the call that needs most of it, in any order, rows few and many; one that is too small is refused"""
    past = [4000, 900, 17, 0, 300, 2222]
    pools, table = cache(6, 4, 128, 64, 64, torch.float16, [p + 40 for p in past], seed=33)
    calls = []
    for B, S in ((1, 1), (6, 1), (2, 1), (1, 4), (6, 2), (3, 40), (1, 40), (6, 1), (6, 40)):
        q, lens = queries(B, 16, S, 128, torch.float16, seed=B + S), torch.tensor(past[:B], dtype=torch.int32, device="cuda")
        calls.append((q, pools, table[:B].contiguous(), 0.1, lens))
    spaces = [mynn.attention_paged_int4_workspace(*c[:3]) for c in calls]
    ws = max(spaces, key=lambda t: t.numel())
    want = [mynn.attention_paged_int4(*c) for c in calls]
    for turn in range(3):
        for n in torch.randperm(len(calls), generator=torch.Generator().manual_seed(turn)).tolist():
            assert same_bits(mynn.attention_paged_int4(*calls[n], workspace=ws), want[n]), (turn, n)
    assert not ws[:mynn.PAGED_INT4_COUNTER_BYTES].any()
    for bad in (ws[:mynn.PAGED_INT4_COUNTER_BYTES], ws[:spaces[1].numel() - 1], ws.float()):
        with pytest.raises(mynn.MynnError):
            mynn.attention_paged_int4(*calls[1], workspace=bad)
    with pytest.raises(mynn.MynnError):
        mynn.attention_paged_int4(*calls[1], workspace=ws[1:])


def test_two_captured_calls_share_a_workspace(mynn):
    """of different shapes, replayed in turn with eager calls between them"""
    past = [3000, 100, 1500]
    pools, table = cache(3, 2, 128, 64, 128, torch.bfloat16, [p + 60 for p in past], seed=34)
    calls = []
    for B, S in ((3, 1), (1, 1), (3, 24)):
        calls.append((queries(B, 8, S, 128, torch.bfloat16, seed=S + B), pools, table[:B].contiguous(), 0.1, torch.tensor(past[:B], dtype=torch.int32, device="cuda")))
    ws = max((mynn.attention_paged_int4_workspace(*c[:3]) for c in calls), key=lambda t: t.numel())
    outs = [torch.empty_like(c[0]) for c in calls]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for c, o in zip(calls, outs):
            mynn.attention_paged_int4(*c, workspace=ws, out=o)
    torch.cuda.synchronize()
    graphs = []
    for c, o in zip(calls, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            mynn.attention_paged_int4(*c, workspace=ws, out=o)
    for turn in range(4):
        for n in ((0, 1, 2), (2, 1, 0), (1, 0, 2), (0, 2, 1))[turn]:
            outs[n].zero_()
            graphs[n].replay()
            torch.cuda.synchronize()
            assert same_bits(outs[n], mynn.attention_paged_int4(*calls[n])), (turn, n)
        for c in calls:
            c[4].add_(7)


def test_pools_of_more_than_32_bits_of_bytes(mynn):
    """pages at the end of pools whose codes, scales and zero points lie past 2^32 bytes of the first: appended, read back, attended to, the same bits as in small pools"""
    Hq, Hkv, D, P, S = 8, 2, 128, 256, 40
    n_pages = (1 << 32) // (Hkv * P * D // 2) + 8
    group = 32
    lead = (n_pages, Hkv, P)
    big = [torch.empty(lead + (D // 2,), dtype=torch.uint8, device="cuda") for _ in range(2)]
    big += [torch.empty(lead + (D // group,), dtype=t, device="cuda") for t in (torch.float16, torch.float16, torch.uint8, torch.uint8)]
    pages = [n_pages - 1, 3, n_pages - 5, n_pages - 2, 0, n_pages - 3]
    small = [torch.empty((6,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in big]
    g = torch.Generator().manual_seed(35)
    cos, sin = tables(1024, D, torch.float16)
    where = [torch.tensor(x, dtype=torch.int32, device="cuda").view(2, 3) for x in (pages, list(range(6)))]
    past = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    for step in range(4):
        n = (300, S, 1, 5)[step]
        rows = torch.randn(2, n, (Hq + 2 * Hkv) * D, generator=g).to(torch.float16).cuda().view(2, n, -1, D).transpose(1, 2)
        got = []
        for pools, table in zip((big, small), where):
            q = mynn.rope_append_paged(rows[:, :Hq], rows[:, Hq:Hq + Hkv], rows[:, Hq + Hkv:], cos, sin, pools, table, past)
            got.append((q, mynn.attention_paged_int4(q, pools, table, 0.1, past), *mynn.kv_rows_paged(pools, table, past, n)))
        for a, b in zip(*got):
            assert same_bits(a, b), step
        past += n
    check(mynn, got[1][0], small, where[1], (past - n).tolist())


@pytest.mark.parametrize("S", [1, 33])
def test_sequences_that_share_pages(mynn, S):
    """a prompt's pages in the tables of several sequences"""
    past = [200, 170, 128]
    pools, table = cache(3, 2, 64, 32, 64, torch.bfloat16, [p + S for p in past], seed=41)
    table[1:, :4] = table[0, :4]
    check(mynn, queries(3, 16, S, 64, torch.bfloat16), pools, table, past)


def test_calls_from_two_threads(mynn):
    """each on a stream of its own, appends into pages of its own and attention behind them"""
    import threading

    Hq, Hkv, D, P, steps = 8, 2, 128, 32, 12
    cos, sin = tables(64, D, torch.float16)
    state = []
    for n in range(2):
        pools, table = cache(2, Hkv, D, P, 128, torch.float16, [64, 64], seed=50 + n)
        rows = torch.randn(steps, 2, 1, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(n)).half().cuda()
        ws = mynn.attention_paged_int4_workspace(torch.empty(2, Hq, 1, D, dtype=torch.float16, device="cuda"), pools, table)
        state.append((pools, table, rows.view(steps, 2, 1, -1, D).transpose(2, 3), ws))

    def run(n, out):
        pools, table, rows, ws = state[n]
        pools = [p.clone() for p in pools]
        past = torch.tensor([3, 20], dtype=torch.int32, device="cuda")
        for i in range(steps):
            q = mynn.rope_append_paged(rows[i][:, :Hq], rows[i][:, Hq:Hq + Hkv], rows[i][:, Hq + Hkv:], cos, sin, pools, table, past)
            out.append(mynn.attention_paged_int4(q, pools, table, 0.1, past, workspace=ws))
            past = past + 1

    want = [[], []]
    for n in range(2):
        run(n, want[n])
    torch.cuda.synchronize()
    got, bad = [[], []], []

    def thread(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                run(n, got[n])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # (shown below: an exception in a thread ends only that)
            bad.append(e)

    threads = [threading.Thread(target=thread, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not bad
    for n in range(2):
        assert len(got[n]) == steps and all(same_bits(a, b) for a, b in zip(got[n], want[n]))
