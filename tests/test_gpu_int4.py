"""Products with 4-bit weights against 64 bits: 16-bit and int8 activations, groups of 32, 64, 128 and more, with and without zero
points, from one row to many, ragged in every direction."""
import importlib

import pytest
import torch

import int4_reference as ref

mynn = importlib.import_module("my-nn-engine_amd")
pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def generator(seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def operands(kind, M, N, K, group, dtype, zero, seed=1):
    g = generator(seed)
    weight = ref.matrix(N, K, group, dtype, zero, g)
    if kind == "linear":
        return (torch.randn((M, K), generator=g, device="cuda").to(dtype),) + weight
    lhs = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device="cuda")
    return (lhs, ((torch.rand((M,), generator=g, device="cuda") + 0.5) / 64).to(dtype)) + weight


def call(kind, ops):
    return mynn.dequant_matmul_int4(*ops) if kind == "linear" else mynn.quantized_matmul_int4(*ops)


def want(kind, ops):
    return ref.product(*ops) if kind == "linear" else ref.product(ops[0], *ops[2:], row_scale=ops[1])


KINDS = pytest.mark.parametrize("kind", ["linear", "qlinear"])


# one row, two, three, odd ones, whole and broken tiles of 16, 32, 64, 128 rows
@KINDS
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 96, 127, 128, 129, 200, 257, 500])
@pytest.mark.parametrize("N,K,group,zero,dtype", [(200, 512, 128, True, F16), (131, 416, 32, False, BF16), (72, 832, 64, True, BF16), (400, 2048, 128, False, BF16)])
def test_rows(kind, M, N, K, group, zero, dtype):
    ops = operands(kind, M, N, K, group, dtype, zero)
    ref.assert_close(call(kind, ops), *want(kind, ops))


# few and many weight rows, one group and many, K that ends inside every power of two a kernel might step by
@KINDS
@pytest.mark.parametrize("M", [1, 6, 20, 50, 150])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 33, 64, 65, 127, 256, 300])
@pytest.mark.parametrize("K,group", [(32, 32), (64, 64), (128, 128), (96, 32), (192, 64), (160, 32), (384, 128), (640, 128), (1024, 1024), (768, 384),
                                     (1056, 32), (2112, 64), (4224, 128)])
def test_columns(kind, M, N, K, group):
    dtype = F16 if (N + K) % 3 else BF16
    ops = operands(kind, M, N, K, group, dtype, N % 2 == 0)
    ref.assert_close(call(kind, ops), *want(kind, ops))


# the shapes of decoders
@KINDS
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K,group", [(1, 2048, 2048, 128), (1, 4096, 14336, 32), (1, 32000, 2048, 64), (2, 28672, 4096, 128), (7, 4096, 4096, 32),
                                         (16, 6144, 4096, 64), (31, 4096, 14336, 128), (64, 11264, 2048, 128), (300, 5632, 2048, 64), (1024, 4096, 4096, 128),
                                         (777, 2048, 5632, 32)])
def test_decoder_shapes(kind, dtype, M, N, K, group):
    ops = operands(kind, M, N, K, group, dtype, (M + N) % 3 == 0)
    ref.assert_close(call(kind, ops), *want(kind, ops))


# rows so long that a workgroup goes over K in rounds, and matrices of so many rows that a wave goes through a ring of them
@KINDS
@pytest.mark.parametrize("M,N,K,group,zero", [(1, 70, 40960, 64, True), (2, 100, 24576, 32, False), (3, 66, 32768, 128, True), (8, 40, 14336, 64, True),
                                              (5, 41, 20480, 32, True), (7, 33, 16512, 128, False), (1, 128256, 256, 128, True), (12, 70000, 512, 64, False),
                                              (20, 40000, 384, 32, True), (6, 50001, 640, 128, True)])
def test_long_rows_and_many(kind, M, N, K, group, zero):
    ops = operands(kind, M, N, K, group, BF16 if M % 2 else F16, zero)
    ref.assert_close(call(kind, ops), *want(kind, ops))
    if kind == "linear" and N <= 100:
        clean = call(kind, ops)
        ops[0][M - 1, K - 5] = float("-inf")
        out = call(kind, ops)
        d, _ = ref.differences(*ops[1:])
        expected = d[:, K - 5] * float("-inf")
        assert torch.equal(out[: M - 1], clean[: M - 1]) and torch.equal(out[M - 1].isnan(), expected.isnan())
        assert torch.equal(out[M - 1].double().nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0), expected.sign().nan_to_num(nan=0.0))


# both sides of every border between the forms: rows, columns, lengths, groups
@KINDS
@pytest.mark.parametrize("M", [8, 9, 16, 17, 32, 33])
@pytest.mark.parametrize("N", [15, 16, 17])
@pytest.mark.parametrize("K,group", [(1024, 32), (1152, 32), (2048, 128), (2176, 64), (4096, 32), (4096, 128), (4224, 128), (4128, 32)])
def test_borders(kind, M, N, K, group):
    ops = operands(kind, M, N, K, group, F16, True)
    ref.assert_close(call(kind, ops), *want(kind, ops))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_leading_dimensions(dtype):
    act, wq, scale, zero = operands("linear", 30, 48, 256, 64, dtype, True)
    out = mynn.dequant_matmul_int4(act.view(2, 3, 5, 256), wq, scale, zero)
    assert out.shape == (2, 3, 5, 48) and torch.equal(out.view(30, 48), mynn.dequant_matmul_int4(act, wq, scale, zero))


# every code with every zero point, by hand: act of ones in one column
@KINDS
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_each_code_and_zero_point_exactly(kind, dtype):
    K = 128
    wq = torch.randint(0, 256, (256, K // 2), generator=generator(), dtype=torch.uint8, device="cuda")
    wq[:, 5] = torch.arange(256, device="cuda").to(torch.uint8)
    zero = (torch.arange(256, device="cuda") * 7 % 256).to(torch.uint8)[:, None]  # (the high four bits mean nothing)
    scale = torch.full((256, 1), 0.25, dtype=dtype, device="cuda")
    for col in (10, 11):
        d = ((wq[:, 5].int() >> (4 * (col - 10))) & 15) - (zero[:, 0].int() & 15)
        if kind == "linear":
            act = torch.zeros((3, K), dtype=dtype, device="cuda")
            act[:, col] = 1.0
            out = mynn.dequant_matmul_int4(act, wq, scale, zero)
        else:
            lhs = torch.zeros((3, K), dtype=torch.int8, device="cuda")
            lhs[:, col] = 1
            out = mynn.quantized_matmul_int4(lhs, torch.ones((3,), dtype=dtype, device="cuda"), wq, scale, zero)
        assert torch.equal(out, (d * 0.25).to(dtype).expand(3, 256))


@KINDS
def test_extreme_int8_sums(kind):
    """a group's sum at its largest: 128 * 128 * 15, and groups of several times that"""
    K, group = 1024, 512
    wq = torch.full((40, K // 2), 0xFF, dtype=torch.uint8, device="cuda")
    scale = torch.full((40, 2), 2.0**-14, dtype=F16, device="cuda")
    zero = torch.zeros((40, 2), dtype=torch.uint8, device="cuda")
    for M in (1, 20, 130):
        if kind == "linear":
            out = mynn.dequant_matmul_int4(torch.full((M, K), -128.0, dtype=F16, device="cuda"), wq, scale, zero)
        else:
            lhs = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
            out = mynn.quantized_matmul_int4(lhs, torch.ones((M,), dtype=F16, device="cuda"), wq, scale, zero)
        assert torch.equal(out, torch.full((M, 40), -128.0 * 15 * K / 2**14, dtype=F16, device="cuda"))


# what is not finite goes where the formula takes it, and to its own row alone
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 3, 20, 70, 140])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("zero", [False, True])
def test_infinities_and_nan(dtype, M, group, zero):
    act, wq, scale, z = operands("linear", M, 100, 512, group, dtype, zero)
    last = M - 1
    act[last, 300] = float("inf")
    clean = mynn.dequant_matmul_int4(operands("linear", M, 100, 512, group, dtype, zero)[0], wq, scale, z)
    out = mynn.dequant_matmul_int4(act, wq, scale, z)
    assert torch.equal(out[:last], clean[:last])
    d, _ = ref.differences(wq, scale, z)
    expected = d[:, 300] * float("inf")  # (a difference of zero: NaN)
    assert torch.equal(out[last].isnan(), expected.isnan())
    assert torch.equal(out[last].double().nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0), expected.sign().nan_to_num(nan=0.0))
    act[last, 300] = float("nan")
    out = mynn.dequant_matmul_int4(act, wq, scale, z)
    assert torch.equal(out[:last], clean[:last]) and bool(out[last].isnan().all())


@pytest.mark.parametrize("M", [1, 5, 40, 130])
def test_large_bf16_activations_do_not_overflow_by_their_offset(M):
    """act * code alone would overflow where act * (code - zero) does not"""
    act = torch.zeros((M, 128), dtype=BF16, device="cuda")
    act[:, 3] = 3e38
    act[:, 77] = 1e38
    wq = torch.full((24, 64), 0x99, dtype=torch.uint8, device="cuda")  # (every difference 1)
    wq[:, 38] = 0x89                                                   # (column 76: 9, 77: 8, a difference of 0)
    scale = torch.full((24, 1), 1.0, dtype=BF16, device="cuda")
    out = mynn.dequant_matmul_int4(act, wq, scale)
    assert torch.equal(out, act[:, 3:4].expand(M, 24))


@KINDS
def test_scales_that_are_not_finite(kind):
    for M in (1, 20, 130):
        ops = operands(kind, M, 50, 256, 128, BF16, False)
        clean = call(kind, ops)
        ops[-2][7, 1] = float("nan")
        out = call(kind, ops)
        assert bool(out[:, 7].isnan().all())
        out[:, 7] = clean[:, 7]
        assert torch.equal(out, clean)
        if kind == "qlinear":
            ops[1][M - 1] = float("nan")
            out = call(kind, ops)
            assert bool(out[M - 1].isnan().all()) and not bool(out[: M - 1, :7].isnan().any())


# small values: rows of subnormal fp16 products, and of zeros
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 30, 140])
def test_small_values(dtype, M):
    act, wq, scale, zero = operands("linear", M, 70, 512, 64, dtype, True)
    act = act * 2.0**-13
    scale = scale * 2.0**-6
    ref.assert_close(mynn.dequant_matmul_int4(act, wq, scale, zero), *ref.product(act, wq, scale, zero))
    assert not bool(mynn.dequant_matmul_int4(torch.zeros_like(act), wq, scale, zero).any())


# scales, zero points and outputs at any element; what lies around the output stays as it was
@KINDS
@pytest.mark.parametrize("M,N,K,group", [(1, 37, 160, 32), (3, 37, 256, 32), (9, 50, 384, 128), (33, 65, 192, 64), (33, 65, 256, 64), (40, 70, 384, 32), (140, 131, 256, 128)])
def test_odd_places(kind, M, N, K, group):
    ops = list(operands(kind, M, N, K, group, BF16, True))
    expected = call(kind, ops)

    def moved(t):
        buf = torch.empty((t.numel() + 3,), dtype=t.dtype, device="cuda")
        buf[1 : 1 + t.numel()] = t.flatten()
        return buf[1 : 1 + t.numel()].view(t.shape)

    scale, zero = moved(ops[-2]), moved(ops[-1])
    buf = torch.full((M * N + 64,), 7.0, dtype=BF16, device="cuda")
    p = buf.data_ptr() + 2 * 31
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "linear":
        rc = mynn.lib().mynn_dequant_matmul_int4(p, ops[0].data_ptr(), ops[1].data_ptr(), scale.data_ptr(), zero.data_ptr(), M, N, K, group, mynn.BF16, stream)
    else:
        ls = moved(ops[1])
        rc = mynn.lib().mynn_quantized_matmul_int4(p, ops[0].data_ptr(), ls.data_ptr(), ops[2].data_ptr(), scale.data_ptr(), zero.data_ptr(), M, N, K, group,
                                                   mynn.BF16, stream)
    assert rc == 0
    assert torch.equal(buf[31 : 31 + M * N].view(M, N), expected)
    assert bool((buf[:31] == 7.0).all()) and bool((buf[31 + M * N :] == 7.0).all())


@KINDS
def test_offsets_beyond_32_bits(kind):
    """a matrix of more than 2^31 bytes, and an output of more than 2^31 values"""
    N, K = 66000, 65536
    assert N * K // 2 > 2**31
    ops = list(operands(kind, 1, N, K, 128, F16, False))
    out = call(kind, ops)
    rows = torch.tensor([0, 1, 32767, 32768, 65534, 65535, 65536, N - 2, N - 1], device="cuda")
    part = [x[rows] if x is ops[-3] or x is ops[-2] else x for x in ops]
    ref.assert_close(out[:, rows], *want(kind, part))
    del ops, part, out
    M, N, K = 66000, 33000, 32
    assert M * N > 2**31
    ops = list(operands(kind, M, N, K, 32, F16, True))
    out = call(kind, ops)
    pick = torch.tensor([0, 1, 32767, 32768, 65071, 65072, 65535, 65536, M - 2, M - 1], device="cuda")
    ops[0] = ops[0][pick]
    if kind == "qlinear":
        ops[1] = ops[1][pick]
    ref.assert_close(out[pick], *want(kind, ops))


# the same bits from call to call, from a captured graph, and beside another stream's calls
@KINDS
@pytest.mark.parametrize("M,N,K,group", [(1, 4096, 4096, 128), (5, 300, 8192, 64), (40, 2048, 4096, 32), (200, 1000, 2048, 128)])
def test_same_bits_everywhere(kind, M, N, K, group):
    ops, other = operands(kind, M, N, K, group, F16, True), operands(kind, M, N, K, group, F16, True, seed=2)
    expected, expected_other = call(kind, ops), call(kind, other)
    assert not torch.equal(expected, expected_other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call(kind, ops)
    with torch.cuda.graph(second, stream=side):
        out_other = call(kind, other)
    for _ in range(4):
        out.zero_(), out_other.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            second.replay()
            beside = call(kind, other)
        eager = call(kind, ops)
        torch.cuda.synchronize()
        assert torch.equal(out, expected) and torch.equal(out_other, expected_other) and torch.equal(beside, expected_other) and torch.equal(eager, expected)


def raw(kind, ops, out, workspace=None):
    """the library's own call: without a workspace, or with one of so many bytes at so many bytes behind the start of a tensor"""
    M, K = ops[0].shape
    N, groups = ops[-2].shape
    name = "mynn_dequant_matmul_int4" if kind == "linear" else "mynn_quantized_matmul_int4"
    args = [out.data_ptr()] + [t.data_ptr() if t is not None else None for t in ops] + [M, N, K, K // groups, mynn.F16]
    stream = torch.cuda.current_stream().cuda_stream
    if workspace is None:
        return getattr(mynn.lib(), name)(*args, stream)
    return getattr(mynn.lib(), name + "_ws")(*args, *workspace, stream)


# K in ranges (of whole pieces and not, one tile of rows and several) and not: every form of a call has the same bits, eager and captured
@KINDS
@pytest.mark.parametrize("M,N,K,group,ranges", [(12, 300, 4096, 32, True), (33, 1000, 4096, 64, True), (100, 520, 16384, 128, True), (40, 256, 2080, 32, True),
                                                (200, 256, 8192, 128, True), (64, 28672, 1024, 128, False), (16, 512, 4096, 128, False), (500, 4096, 512, 128, False)])
def test_every_form_of_a_call(kind, M, N, K, group, ranges):
    ops = operands(kind, M, N, K, group, F16, True)
    need = mynn.lib().mynn_matmul_int4_workspace_bytes(M, N, K, group)
    assert need % (M * N * 4) == 0 and (need >= 2 * M * N * 4 if ranges else need == 0)
    expected = call(kind, ops)
    ref.assert_close(expected, *want(kind, ops))
    out = torch.empty_like(expected)
    assert raw(kind, ops, out.zero_()) == 0 and torch.equal(out, expected)
    ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
    assert raw(kind, ops, out.zero_(), (ws.data_ptr() + 2048, need)) == 0 and torch.equal(out, expected)
    assert bool((ws[:2048] == 77).all()) and bool((ws[2048 + need :] == 77).all())
    if need:
        assert raw(kind, ops, out, (ws.data_ptr(), need - 1)) == -1 and b"workspace" in mynn.lib().mynn_last_error()
        assert raw(kind, ops, out, (None, need)) == -1 and raw(kind, ops, out, (ws.data_ptr() + 8, need)) == -1
    else:
        assert raw(kind, ops, out.zero_(), (None, 0)) == 0 and torch.equal(out, expected)
    # three graphs: the plain call (no memory of the library's), the caller's workspace, the wrapper's; replayed side by side
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], [torch.empty_like(out) for _ in range(2)]
    for f in (lambda: (raw(kind, ops, outs[0]), outs[0])[1], lambda: (raw(kind, ops, outs[1], (ws.data_ptr(), need)), outs[1])[1], lambda: call(kind, ops)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o = f()
        graphs.append((g, o))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for _, o in graphs:
            o.zero_()
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = call(kind, ops)
        torch.cuda.synchronize()
        assert torch.equal(eager, expected) and all(torch.equal(o, expected) for _, o in graphs)


def test_threads_on_streams_of_their_own():
    import threading

    shapes = [(12, 300, 2048, 32), (40, 1024, 4096, 64), (3, 4096, 4096, 128), (200, 256, 8192, 128)]
    sets = [operands("linear", *s, F16, True, seed=i) for i, s in enumerate(shapes)]
    expected = [call("linear", o) for o in sets]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                out = torch.empty_like(expected[i])
                if raw("linear", sets[i], out) != 0 or not torch.equal(out, expected[i]) or not torch.equal(call("linear", sets[i]), expected[i]):
                    failures.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


@KINDS
@pytest.mark.parametrize("M", [1, 40])
def test_the_way_without_the_module(kind, M, monkeypatch):
    """through ctypes: the same results and the same refusals as through the module of C++"""
    ops = operands(kind, M, 300, 4096, 64, F16, True)
    expected = call(kind, ops)
    monkeypatch.setattr(mynn, "_ops", mynn._NoHostOps())
    assert torch.equal(call(kind, ops), expected)
    with pytest.raises(mynn.MynnError, match="fit together"):
        call(kind, (ops[0][:, :64].contiguous(),) + ops[1:])


@KINDS
def test_wrapper_refuses_what_does_not_fit(kind):
    ops = operands(kind, 4, 32, 256, 64, F16, True)
    assert call(kind, ops) is not None

    def refused(**change):
        o = list(ops)
        for i, v in change.items():
            o[int(i[1:])] = v
        with pytest.raises((mynn.MynnError, AssertionError)):
            call(kind, o)

    w = len(ops) - 3
    refused(**{"_0": ops[0][:, :128].contiguous()})                      # K
    refused(**{"_0": ops[0].float()})                                    # type
    refused(**{"_0": ops[0].t().contiguous().t()})                       # order
    refused(**{"_0": ops[0][:0]})                                        # no rows
    refused(**{"_%d" % w: ops[w].to(torch.int8)})                        # codes of another type
    refused(**{"_%d" % w: ops[w][:31].contiguous()})                     # N
    refused(**{"_%d" % (w + 1): ops[w + 1][:, :3].contiguous()})         # groups that do not divide K
    refused(**{"_%d" % (w + 1): ops[w + 1].float()})                     # scales of another type
    refused(**{"_%d" % (w + 2): ops[w + 2].to(torch.int32)})             # zero points of another type
    refused(**{"_%d" % (w + 2): ops[w + 2][:16].contiguous()})
    refused(**{"_%d" % w: ops[w].cpu()})                                 # another device
    if kind == "qlinear":
        refused(_1=ops[1][:3].contiguous())
        refused(_1=ops[1].float())


def test_host_quantiser_round_trip():
    """codes, scales and zero points of the host quantiser multiplied by the identity: every weight within half a step, the scale's rounding
    and the output's of what it was"""
    g = torch.Generator().manual_seed(3)
    w = torch.randn((48, 256), generator=g)
    w[3] = w[3].abs() + 0.1  # (one sign alone)
    for dt, T in ((mynn.F16, F16), (mynn.BF16, BF16)):
        for group in (32, 128):
            for symmetric in (True, False):
                q, s, z = mynn.quantize_int4_groups(w.numpy(), group, dt, symmetric)
                scale = torch.from_numpy(s.view("int16")).view(T).cuda()
                out = mynn.dequant_matmul_int4(torch.eye(256, dtype=T, device="cuda"), torch.from_numpy(q).cuda(), scale, None if z is None else torch.from_numpy(z).cuda())
                steps = scale.float().repeat_interleave(group, 1).t()
                eps = torch.finfo(T).eps / 2
                # (symmetric codes reach 7 steps, asymmetric ones 15, of a step that may be rounded down by eps; zero points take half a step more)
                most = steps * (0.5 + (0 if symmetric else 0.5) + 15 * eps) + eps * 16 * steps
                assert bool(((out.float() - w.t().cuda()).abs() <= most * 1.0001).all())
