"""Products of few rows with 4-bit weights: what one weight row or one row of activations holds does not reach the others."""
import importlib

import pytest
import torch

import int4_reference as ref

mynn = importlib.import_module("my-nn-engine_amd")
pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def slots(M):
    """weight rows of a tile"""
    return 1 if M == 1 else 2 if M == 2 else 4 if M <= 4 else 8 if M <= 8 else 16


# a last tile that begins inside the one before it: the rows that both hold are the earlier one's, whatever the later one's scales are
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [2, 3, 4, 7, 8, 16, 24])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_that_two_tiles_hold(dtype, M, group):
    rows, K = slots(M), 1024
    for seed, more in enumerate((1, rows // 2, rows - 1)):
        N = 16 * rows + 32 + more
        g = generator(seed)
        wq, scale, zero = ref.matrix(N, K, group, dtype, True, g)
        act = torch.randn((M, K), generator=g, device="cuda").to(dtype)
        clean = mynn.dequant_matmul_int4(act, wq, scale, zero)
        scale[N - 1, 0] = float("nan")
        out = mynn.dequant_matmul_int4(act, wq, scale, zero)
        assert bool(out[:, N - 1].isnan().all())
        earlier = N // rows * rows
        assert torch.equal(out[:, :earlier], clean[:, :earlier])


MANY = [1, 2, 3, 4, 7, 8, 9, 16, 20, 32, 40, 140]


# an activation whose codes are the zero point counts for nothing, however large it is: the bits are those of a zero in its place
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", MANY)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zero", [False, True])
def test_outliers_where_the_code_is_the_zero_point(dtype, M, group, zero):
    N, K = 61, 1024
    g = generator(7)
    wq, scale, z = ref.matrix(N, K, group, dtype, zero, g)
    act = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    at = [3, 40, 200, 515, 1022]
    zeros = torch.full((N, K // group), 8, dtype=torch.uint8, device="cuda") if z is None else z
    for c in at:
        code = zeros[:, c // group]
        wq[:, c // 2] = (wq[:, c // 2] & 0xF0) | code if c % 2 == 0 else (wq[:, c // 2] & 0x0F) | (code << 4)
    act[:, at] = 0
    clean = mynn.dequant_matmul_int4(act, wq, scale, z)
    act[:, at] = torch.tensor([2.0**24, -(2.0**24), 2.0**30, 2.0**20, 2.0**16] if dtype == BF16 else [60000.0, -50000.0, 40000.0, 65504.0, 1000.0], device="cuda").to(dtype)
    assert torch.equal(mynn.dequant_matmul_int4(act, wq, scale, z), clean)
    # one unit each in 127 columns
    act, wq = torch.ones((M, 128), dtype=dtype, device="cuda"), torch.full((20, 64), 0xFF, dtype=torch.uint8, device="cuda")
    act[:, 5], wq[:, 2] = (2.0**24 if dtype == BF16 else 65504.0), 0xEF
    z = torch.full((20, 1), 14, dtype=torch.uint8, device="cuda")
    assert torch.equal(mynn.dequant_matmul_int4(act, wq, torch.ones((20, 1), dtype=dtype, device="cuda"), z), torch.full((M, 20), 127.0, dtype=dtype, device="cuda"))


# the bound of a 32-bit sum over act * (code - zero), which knows of no sums of codes and zero points apart
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", MANY)
@pytest.mark.parametrize("N,K,group,zero", [(200, 1024, 32, True), (75, 2048, 64, False), (100, 2048, 128, True)])
def test_sums_of_differences(dtype, M, N, K, group, zero):
    g = generator(M)
    wq, scale, z = ref.matrix(N, K, group, dtype, zero, g)
    # codes near the zero point, activations of one sign with a few large ones
    near = torch.full((N, K // group), 8, dtype=torch.uint8, device="cuda") if z is None else z
    code = (near.repeat_interleave(group, 1).int() + torch.randint(-1, 2, (N, K), generator=g, device="cuda")).clamp(0, 15).to(torch.uint8)
    wq = code[:, 0::2] | (code[:, 1::2] << 4)
    act = (torch.rand((M, K), generator=g, device="cuda") * (1 + 999 * (torch.rand((K,), generator=g, device="cuda") < 0.01))).to(dtype)
    d, s = ref.differences(wq, scale, z)
    exact = act.double() @ (d * s).t().contiguous()
    # (a term goes through 128 additions of a group, two for the scale, K / 32 partial sums and those of 32 waves, each at most 2^-23 off)
    bound = act.double().abs() @ (d.abs() * s.abs()).t().contiguous() * (128 + 3 + K / 32 + 32) * 2.0**-23
    eps = torch.finfo(dtype).eps / 2
    out = mynn.dequant_matmul_int4(act, wq, scale, z).double()
    assert bool(((out - exact).abs() <= bound + eps * (exact.abs() + bound) + torch.finfo(dtype).smallest_normal * eps).all())


# a row that is not finite, or one weight row's scale: every other value of the product keeps its bits
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", MANY)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zero", [False, True])
def test_other_rows_keep_their_bits(dtype, M, group, zero):
    N, K = 203, 2048
    for seed in range(6):
        g = generator(seed)
        wq, scale, z = ref.matrix(N, K, group, dtype, zero, g)
        act = (torch.randn((M, K), generator=g, device="cuda") * 30).to(dtype)
        clean = mynn.dequant_matmul_int4(act, wq, scale, z)
        row, column = seed * 5 % M, (37 * seed + N - 1) % N
        bad = act.clone()
        bad[row, 1000] = float("inf") if seed % 2 else float("nan")
        out = mynn.dequant_matmul_int4(bad, wq, scale, z)
        assert not bool(out[row].isfinite().any())
        assert torch.equal(out[:row], clean[:row]) and torch.equal(out[row + 1 :], clean[row + 1 :])
        bad = scale.clone()
        bad[column, 1] = float("nan") if seed % 2 else float("inf")
        out = mynn.dequant_matmul_int4(act, wq, bad, z)
        assert not bool(out[:, column].isfinite().any())
        assert torch.equal(out[:, :column], clean[:, :column]) and torch.equal(out[:, column + 1 :], clean[:, column + 1 :])


# bf16 rows of all magnitudes: each weight row has its differences in columns of one magnitude alone, however much larger the others are
@pytest.mark.parametrize("M", MANY)
@pytest.mark.parametrize("N,K,group,zero", [(57, 1024, 32, True), (57, 1024, 128, False), (57, 16384, 64, True)])
@pytest.mark.parametrize("far", [40, 31, 13])
def test_rows_of_all_magnitudes(M, N, K, group, zero, far):
    g = generator(M)
    wq, scale, z = ref.matrix(N, K, group, BF16, zero, g)
    exponents = torch.arange(-100, 101, far, device="cuda")
    which = torch.randint(0, len(exponents), (K,), generator=g, device="cuda")
    which[: len(exponents)] = torch.arange(len(exponents), device="cuda")
    act = (torch.randn((M, K), generator=g, device="cuda") * 2.0 ** exponents[which].float()).to(BF16)
    act[0, 5::7] = 0
    if M > 2:
        act[1] = 0
        act[2] = torch.randn((K,), generator=g, device="cuda").to(BF16)
    near = torch.full((N, K // group), 8, dtype=torch.uint8, device="cuda") if z is None else z
    code = near.repeat_interleave(group, 1)
    mine = torch.arange(N, device="cuda")[:, None] % len(exponents) == which[None, :]
    code = torch.where(mine, ref.codes(wq), code)
    wq = code[:, 0::2] | (code[:, 1::2] << 4)
    d, s = ref.differences(wq, scale, z)
    exact = act.double() @ (d * s).t().contiguous()
    bound = act.double().abs() @ (d.abs() * s.abs()).t().contiguous() * (128 + 3 + K / 32 + 32) * 2.0**-23
    eps = torch.finfo(BF16).eps / 2
    out = mynn.dequant_matmul_int4(act, wq, scale, z).double()
    assert bool(((out - exact).abs() <= bound + eps * (exact.abs() + bound) + torch.finfo(BF16).smallest_normal * eps).all())
    # rows of their own: the bits do not depend on the others' magnitudes
    if 2 < M <= 32:
        act[0] = act[2]
        assert torch.equal(mynn.dequant_matmul_int4(act, wq, scale, z)[2], out[2].to(BF16))
        alone = mynn.dequant_matmul_int4(act[2:3].expand(M, K).contiguous(), wq, scale, z)
        assert torch.equal(alone[2], out[2].to(BF16))


# the smallest bf16 numbers, and rows that end at the largest
@pytest.mark.parametrize("M", MANY)
def test_the_ends_of_bf16(M):
    K, N = 512, 33
    wq = torch.full((N, K // 2), 0x99, dtype=torch.uint8, device="cuda")  # (every difference 1)
    scale = torch.ones((N, 4), dtype=BF16, device="cuda")
    act = torch.zeros((M, K), dtype=BF16, device="cuda")
    act[:, 7] = 2.0**-133  # (the smallest)
    act[:, 300] = 2.0**-130
    assert torch.equal(mynn.dequant_matmul_int4(act, wq, scale), torch.full((M, N), 2.0**-133 + 2.0**-130, device="cuda").to(BF16))
    act[:, 400] = 3.3e38
    act[:, 401] = -3.3e38
    act[:, 300] = 1.0
    act[:, 7] = 0
    wq[:, 200] = 0x89  # (column 400: 1, 401: 0)
    assert torch.equal(mynn.dequant_matmul_int4(act, wq, scale), act[:, 400:401].expand(M, N))
    wq[:, 200] = 0x88
    assert torch.equal(mynn.dequant_matmul_int4(act, wq, scale), torch.ones((M, N), dtype=BF16, device="cuda"))
