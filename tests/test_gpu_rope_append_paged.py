"""RoPE of q and k with the append of k and v to paged caches of 16, 8 and 4 bits: the rotated q and every byte of the pools against the
same steps in plain 32-bit operations, the rows that come back against 64 bits."""
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

KINDS = [(16, 0), (8, 0), (4, 128), (4, 64), (4, 32)]


@pytest.fixture(scope="module")
def mynn():
    import gpu_util

    return gpu_util.mynn


def tables(n, D, dtype, device="cuda"):
    angle = torch.arange(n, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(D // 2, dtype=torch.float64) * 2 / D)
    angle = torch.cat((angle, angle), 1)
    return angle.cos().to(dtype).to(device), angle.sin().to(dtype).to(device)


def case(B, S, Hq, Hkv, D, P, dtype, bits, group, past, seed=0, pages=None, spare=3):
    """operands in the GPU's memory: views of the projection's rows, pools full of something, a table in no order"""
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(B, S, (Hq + 2 * Hkv) * D, generator=g)
    rows.view(B, S, -1, D)[:, :, Hq:, ::13] *= 6.0
    rows = rows.to(dtype).cuda()
    x = rows.view(B, S, Hq + 2 * Hkv, D).transpose(1, 2)
    pages = pages or max((p + S + P - 1) // P for p in past)
    table = torch.randperm(B * pages + spare, generator=g)[:B * pages].to(torch.int32).view(B, pages).cuda()
    pools = ref.make_pools(B * pages + spare, Hkv, P, D, dtype, bits, group, "cuda", seed)
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], pools, table, torch.tensor(past, dtype=torch.int32, device="cuda")


def same_bits(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def check(mynn, q, k, v, cos, sin, pools, table, past, new=None, positions=None, out=None):
    new_dev = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    cpu = lambda t: None if t is None else t.cpu()
    want, want_pools = ref.append(cpu(q), cpu(k), cpu(v), cos.cpu(), sin.cpu(), [p.cpu() for p in pools], table.cpu(), past.cpu(), new, cpu(positions))
    got = mynn.rope_append_paged(q, k, v, cos, sin, pools, table, past, new_dev, positions, out)
    torch.cuda.synchronize()
    if q is not None:
        assert same_bits(got.cpu(), want)
    else:
        assert got is None
    for n, (a, b) in enumerate(zip(pools, want_pools)):
        if not same_bits(a.cpu(), b):
            pytest.fail("pool %d" % n)
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits,group", KINDS)
@pytest.mark.parametrize("B,S,Hq,Hkv,D,P,past", [
    (1, 1, 32, 4, 64, 32, [0]),
    (5, 1, 32, 8, 128, 64, [63, 64, 0, 200, 31]),
    (2, 37, 8, 8, 64, 32, [20, 0]),          # pages that begin and end inside the call's rows
    (3, 9, 4, 1, 128, 256, [250, 0, 255]),
    (1, 3, 6, 2, 64, 32, [95]),              # head counts that are no power of two
])
def test_rows_and_pools_bit_for_bit(mynn, dtype, bits, group, B, S, Hq, Hkv, D, P, past):
    if group > D:
        pytest.skip("groups of at most a row")
    q, k, v, pools, table, past_dev = case(B, S, Hq, Hkv, D, P, dtype, bits, group, past)
    cos, sin = tables(400, D, dtype)
    check(mynn, q, k, v, cos, sin, pools, table, past_dev)


@pytest.mark.parametrize("bits,group", KINDS)
def test_ragged_batches_leave_every_other_row_alone(mynn, bits, group):
    """sequences with all, some and none of the call's tokens, more than there are, and lengths below zero"""
    B, S, D, dtype = 6, 11, 128, torch.bfloat16
    q, k, v, pools, table, past = case(B, S, 8, 2, D, 32, dtype, bits, group, [0, 30, 5, 64, 33, 1], seed=3)
    cos, sin = tables(120, D, dtype)
    check(mynn, q, k, v, cos, sin, pools, table, past, new=[11, 4, 0, 1, 200, -7])


@pytest.mark.parametrize("bits,group", KINDS)
def test_rows_past_the_cache_the_table_and_the_pages_are_not_there(mynn, bits, group):
    """the last page is full, tables end, pages are unmapped or none of the pool's: nothing but what is there is written"""
    B, S, D, dtype = 5, 6, 64, torch.float16
    if group > D:
        pytest.skip("groups of at most a row")
    q, k, v, pools, table, past = case(B, S, 4, 2, D, 32, dtype, bits, group, [61, 30, 30, -3, 2 ** 31 - 1], seed=4, pages=2)
    table[1, 1], table[2, 0] = -1, pools[0].shape[0]
    cos, sin = tables(63, D, dtype)
    check(mynn, q, k, v, cos, sin, pools, table, past)
    past[4] = -2 ** 31
    check(mynn, q, k, v, cos, sin, pools, table, past)


def test_positions_of_their_own(mynn):
    B, S, D, dtype = 2, 5, 128, torch.bfloat16
    q, k, v, pools, table, past = case(B, S, 4, 4, D, 64, dtype, 4, 64, [7, 100], seed=5)
    cos, sin = tables(50, D, dtype)
    positions = torch.tensor([[0, 49, 3, 50, -1], [12, 12, 2 ** 40, 1, 0]], dtype=torch.int64, device="cuda")
    check(mynn, q, k, v, cos, sin, pools, table, past, positions=positions)


@pytest.mark.parametrize("bits,group", KINDS)
def test_rows_at_odd_places(mynn, bits, group):
    """projection rows of an odd pitch that begin two bytes past a 16-byte line; heads last; one row for every token"""
    B, S, Hq, Hkv, D, dtype = 2, 3, 4, 2, 64, torch.float16
    if group > D:
        pytest.skip("groups of at most a row")
    q, k, v, pools, table, past = case(B, S, Hq, Hkv, D, 32, dtype, bits, group, [1, 40], seed=6)
    wide = torch.empty(B, S, (Hq + 2 * Hkv) * D + 3, dtype=dtype, device="cuda")
    x = torch.as_strided(wide, (B, Hq + 2 * Hkv, S, D), (wide.stride(0), D, wide.stride(1), 1), 1)
    x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:] = q, k, v
    cos, sin = tables(60, D, dtype)
    check(mynn, x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], cos, sin, pools, table, past)
    check(mynn, q.contiguous(), k.transpose(1, 2).contiguous().transpose(1, 2), v[:, :, :1].expand(-1, -1, S, -1), cos, sin, pools, table, past)


def test_in_place_and_without_queries(mynn):
    B, S, D, dtype = 3, 4, 128, torch.float16
    q, k, v, pools, table, past = case(B, S, 8, 2, D, 32, dtype, 4, 32, [0, 31, 77], seed=7)
    cos, sin = tables(100, D, dtype)
    q = q.contiguous()
    want = mynn.rope_append_paged(q, k, v, cos, sin, [p.clone() for p in pools], table, past)
    kept = q.clone()
    got = mynn.rope_append_paged(q, k, v, cos, sin, [p.clone() for p in pools], table, past, out=q)
    assert got.data_ptr() == q.data_ptr() and same_bits(got, want) and not torch.equal(got, kept)
    check(mynn, None, k, v, cos, sin, pools, table, past)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [128, 64, 32])
def test_extreme_rows_of_four_bits(mynn, dtype, group):
    """zeros, one value, values of one sign, the type's largest and smallest, infinities and NaN"""
    D, dtype_max, least = 128, torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    rows = torch.zeros(1, 1, 12, D)
    rows[0, 0, 1, 5] = 3.0
    rows[0, 0, 2] = torch.linspace(1.0, 2.0, D)
    rows[0, 0, 3] = -torch.linspace(1.0, 2.0, D)
    rows[0, 0, 4, ::2], rows[0, 0, 4, 1::2] = dtype_max, -dtype_max
    rows[0, 0, 5, 7] = least
    rows[0, 0, 6, ::3], rows[0, 0, 6, 1::3] = least * 40, -least * 7
    rows[0, 0, 7, 70] = float("inf")
    rows[0, 0, 8, 3] = float("nan")
    rows[0, 0, 9, 31], rows[0, 0, 9, 32] = float("-inf"), 2.0
    rows[0, 0, 10] = torch.arange(D) / 2.0 - 20.0  # halves: ties
    rows[0, 0, 11] = dtype_max
    v = rows.to(dtype).cuda()
    k = torch.randn(1, 1, 12, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    pools = ref.make_pools(2, 1, 32, D, dtype, 4, group, "cuda")
    table, past = torch.tensor([[1]], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    cos, sin = tables(32, D, dtype)
    before = [p.clone() for p in pools]
    mynn.rope_append_paged(None, k, v, cos, sin, pools, table, past)
    _, want = ref.append(None, k.cpu(), v.cpu(), cos.cpu(), sin.cpu(), [p.cpu() for p in before], table.cpu(), past.cpu(), None)
    for n, (a, b) in enumerate(zip(pools, want)):
        if a.is_floating_point():  # (a NaN's bits are no one's business)
            a, b = a.cpu(), b
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)), "pool %d" % n
        else:
            assert torch.equal(a.cpu(), b), "pool %d" % n


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits,group", KINDS)
def test_rows_come_back_as_what_they_stand_for(mynn, dtype, bits, group):
    B, S, Hkv, D, P = 3, 40, 3, 128, 32
    q, k, v, pools, table, past = case(B, S, 3, Hkv, D, P, dtype, bits, group, [0, 17, 50], seed=8)
    cos, sin = tables(120, D, dtype)
    mynn.rope_append_paged(q, k, v, cos, sin, pools, table, past)
    table[1, 1] = -1
    for first, n, count in (([0, 17, 50], 40, None), ([5, 0, 126], 3, [1, 3, 9]), ([-2, 130, 60], 5, None)):
        dev = torch.tensor(first, dtype=torch.int32, device="cuda")
        got = mynn.kv_rows_paged(pools, table, dev, n, None if count is None else torch.tensor(count, dtype=torch.int32, device="cuda"))
        for side in range(2):
            for b in range(B):
                want, there = ref.rows_of(pools, side, table, b, first[b], n)
                there = there & (torch.arange(n, device="cuda") < (n if count is None else count[b]))
                want = torch.where(there[None, :, None], want, torch.zeros_like(want))
                # (a whole number times a scale is exact in 32 bits; rows that no one wrote may hold NaN)
                want = want.float().to(dtype)
                if not (torch.equal(torch.isnan(got[side][b]), torch.isnan(want)) and torch.equal(torch.nan_to_num(got[side][b]), torch.nan_to_num(want))):
                    pytest.fail("rows of side %d, sequence %d, from %d" % (side, b, first[b]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_against_64_bits(mynn, dtype):
    """q: two products and their sum in 32 bits, then half a step of the type.  The 4-bit rows: a value in range is at most half a step of its scale from what its
    code stands for, and a whole one at the ends, where the zero point's rounding cuts the range short; 15 steps of a scale that is itself rounded."""
    B, S, Hq, Hkv, D, group = 2, 8, 4, 2, 128, 64
    q, k, v, pools, table, past = case(B, S, Hq, Hkv, D, 32, dtype, 4, group, [3, 40], seed=9)
    cos, sin = tables(60, D, dtype)
    got = mynn.rope_append_paged(q, k, v, cos, sin, pools, table, past)
    at = past.long()[:, None] + torch.arange(S, device="cuda")
    eps = torch.finfo(dtype).eps / 2
    for x, y in ((q, got),):
        want = ref.rotate(x, cos[at], sin[at], torch.float64)
        size = ref.rotate(x.abs(), cos[at].abs(), -sin[at].abs(), torch.float64).abs() + ref.rotate(x.abs(), cos[at].abs(), sin[at].abs(), torch.float64).abs()
        assert ((y.double() - want).abs() <= want.abs() * eps + size * 3 * 2.0 ** -24 + 1e-30).all()
    kr = ref.rotate(k, cos[at], sin[at]).to(dtype).double()
    for side, x in enumerate((kr, v.double())):
        for b in range(B):
            have, _ = ref.rows_of(pools, side, table, b, int(past[b]), S)
            step = torch.stack([pools[2 + side][int(table[b, r // 32]), :, r % 32] for r in range(int(past[b]), int(past[b]) + S)], 1).double()  # [Hkv, S, groups]
            limit = step.repeat_interleave(group, -1) * (1 + 30 * eps)
            assert ((have - x[b]).abs() <= limit).all()


def test_a_captured_call_follows_the_lengths(mynn):
    """lengths, tables and operands are read on the device: replays append where the lengths say, each equal to the eager call"""
    B, S, D, dtype = 4, 2, 128, torch.bfloat16
    q, k, v, pools, table, past = case(B, S, 8, 2, D, 32, dtype, 4, 64, [0, 1, 30, 62], seed=10, pages=6)
    new = torch.tensor([2, 1, 2, 0], dtype=torch.int32, device="cuda")
    cos, sin = tables(200, D, dtype)
    out = torch.empty(q.shape, dtype=dtype, device="cuda")
    stream = torch.cuda.Stream()
    eager = [p.clone() for p in pools]
    with torch.cuda.stream(stream):
        mynn.rope_append_paged(q, k, v, cos, sin, [p.clone() for p in pools], table, past, new, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        mynn.rope_append_paged(q, k, v, cos, sin, pools, table, past, new, out=out)
    for step in range(4):
        graph.replay()
        want = mynn.rope_append_paged(q, k, v, cos, sin, eager, table, past, new)
        torch.cuda.synchronize()
        assert same_bits(out, want)
        for a, b in zip(pools, eager):
            assert same_bits(a, b)
        past += new
        table.copy_(table.flip(1))


def test_pages_of_a_session_and_uniform_lengths_meet_the_other_paged_operators(mynn):
    """16-bit pools filled by one call are what mynn_kvcache_update_paged leaves, and mynn_attention_paged reads them; the table of a page set"""
    B, S, Hq, Hkv, D, P, dtype = 2, 70, 8, 2, 128, 64, torch.float16
    pool = mynn.KvPool(12, P)
    pages = mynn.KvPages(pool, B, 256)
    pages.reserve(S)
    (kp, vp), = pool.buffers(1, Hkv, D, dtype)
    table = torch.from_numpy(pages.table()).cuda()
    q, k, v, _, _, past = case(B, S, Hq, Hkv, D, P, dtype, 16, 0, [0, 0], seed=11)
    cos, sin = tables(256, D, dtype)
    got = mynn.rope_append_paged(q, k, v, cos, sin, (kp, vp), pages, past)
    k2, v2 = torch.zeros_like(kp), torch.zeros_like(vp)
    pos = torch.arange(S, device="cuda")
    mynn.kvcache_update_paged(k2, mynn.rope(k.contiguous(), cos, sin, pos), 0, table, P)
    mynn.kvcache_update_paged(v2, v.contiguous(), 0, table, P)
    assert same_bits(got, mynn.rope(q.contiguous(), cos, sin, pos)) and same_bits(kp, k2) and same_bits(vp, v2)
    out = mynn.attention_paged(got, kp, vp, table, P, D ** -0.5, True, S)
    want, slack = ref.attention(got, (kp, vp), table, D ** -0.5, [0, 0], None, True, 2.0 ** -10)
    ref.assert_close(out, want, slack)
    pages.close()
    pool.close()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [128, 64, 32])
def test_values_halfway_between_two_codes(mynn, dtype, group):
    """rows whose scale is known (15 of it between least and largest) and whose values are its halves, and the type's next numbers on either side of them: scales of few
    bits, whose halves the type holds, and of all, of every magnitude down to its least numbers"""
    D, P = 128, 32
    info = torch.finfo(dtype)
    bits = 10 if dtype == torch.float16 else 7
    least, most = (-24, 11) if dtype == torch.float16 else (-133, 120)
    scales = [2.0 ** e * m for e in list(range(least, least + 14)) + list(range(least + 14, most, 5)) for m in (1.0, 1.5, 1.25, 1.75, 1.0 + 2.0 ** -bits, 2.0 - 2.0 ** -bits, 1.0 + 2.0 ** -3)]
    rows = []
    for s in scales:
        s = float(torch.tensor(s, dtype=torch.float64).to(dtype).double())
        if not 0 < s or 15 * s > info.max:
            continue
        for z in (0, 4, 15):
            n = torch.arange(-z, 16 - z, dtype=torch.float64)
            x = ((n + 0.5) * s).to(dtype)
            row = torch.cat((x[:-1], n.mul(s).to(dtype)[-1:], n.mul(s).to(dtype)[:1], torch.zeros(15, dtype=dtype)))
            up, down = row.clone(), row.clone()
            for t, step in ((up, 1), (down, -1)):  # (one step of the type away from zero, towards it; not the ends, which make the scale)
                w = t[:15].view(torch.int16)
                w += step * (w.bitwise_and(0x7FFF) > 1).to(torch.int16)
            rows += [torch.cat((row, up, down, row))]
    S = len(rows)
    v = torch.stack(rows)[None, None].cuda()
    k = v.flip(-1).contiguous()
    cos, sin = torch.ones(S, D, dtype=dtype, device="cuda"), torch.zeros(S, D, dtype=dtype, device="cuda")
    pages = (S + P - 1) // P
    pools = ref.make_pools(pages, 1, P, D, dtype, 4, group, "cuda", 3)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    check(mynn, None, k, v, cos, sin, pools, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    codes = torch.stack((pools[1] & 15, pools[1] >> 4), -1).flatten(-2)
    assert all(int((codes == c).sum()) > S for c in range(16))
