"""Codes of the normalised rows at the borders between two of them: those of the 32-bit quotient."""
import importlib

import numpy as np
import pytest
import torch

mynn = importlib.import_module("my-nn-engine_amd")
pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def normalised(x, w, eps):
    """the 32-bit values that are quantised: whole numbers whose squares add up exactly in any order, then one rounding for each operation"""
    x, w = x.numpy().astype(np.float32), w.float().numpy()
    mean = (x * x).sum(1, dtype=np.float64).astype(np.float32) / np.float32(x.shape[1])
    inv = np.float32(1) / np.sqrt(mean + np.float32(eps))
    return (x * inv[:, None]) * w


def codes_of(y):
    """y / step in 32 bits, rounded half away from zero; step = max|y| / 127 in 32 bits"""
    q = np.abs(y) / (np.abs(y).max(1) / np.float32(127))[:, None]
    assert q.dtype == np.float32
    n = np.floor(q.astype(np.float64) + 0.5)
    return np.where(y < 0, -n, n)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("dim", [64, 63])
def test_codes_are_the_quotients(dtype, dim):
    g = torch.Generator().manual_seed(3)
    rows, eps = 60000, 0.3
    x = torch.randint(-15, 16, (rows, dim), generator=g).float()
    w = (1.0 + 0.3 * torch.randn((dim,), generator=g)).to(F16 if dtype == F32 else dtype).to(dtype)
    y = normalised(x, w, eps)
    want = codes_of(y)
    # (the product with the rounded reciprocal is another code for some)
    per = np.float32(1) / (np.abs(y).max(1) / np.float32(127))
    assert (np.floor((np.abs(y) * per[:, None]).astype(np.float64) + 0.5) != np.abs(want)).sum() >= 3
    codes, _, _ = mynn.add_rms_norm_quantize(x.to(dtype).cuda(), None, w.cuda(), eps)
    assert np.array_equal(codes.cpu().numpy(), want)


def test_exact_ties_go_away_from_zero():
    """steps that are whole numbers, values of (n + 1/2) steps"""
    steps = [s for s in range(1, 4000, 2) if s % 127]
    for step in steps[::40] + [41, 1023, 2047]:
        w = torch.tensor([(n + 0.5) * step for n in range(127)] + [127.0 * step], dtype=F32)
        x = torch.ones((2, 128))
        x[1] = -1.0
        codes, scale, _ = mynn.add_rms_norm_quantize(x.cuda(), None, w.cuda(), 0.0)
        want = torch.tensor(list(range(1, 128)) + [127], dtype=torch.int8)
        assert torch.equal(codes.cpu(), torch.stack((want, -want))) and scale.cpu().tolist() == [float(step)] * 2
