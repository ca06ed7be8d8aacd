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
