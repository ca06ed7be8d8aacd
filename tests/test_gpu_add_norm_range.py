"""The norm of rows whose squares are too large, or with eps 0 too small, for a 32-bit sum."""
import importlib

import pytest
import torch

mynn = importlib.import_module("my-nn-engine_amd")
pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def exact(x, w, eps):
    """in 64 bits, and how far off 32 bits may be, relative: the sum of dim squares (each term in at most dim / 256 + 16 additions, its own rounding and that
    of its power of two's subnormal part, 2^-24 of the largest), the mean, the root, the quotient, three products; the root halves the sum's"""
    h = x.double()
    eps = float(torch.tensor(eps, dtype=F32))  # (the call's is a 32-bit number: 1e-40 is a subnormal one, 5e-6 of it off)
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return y, ((x.shape[-1] / 256 + 18) / 2 + 7) * 2.0**-24


def check(x, w, eps, rows=slice(None)):
    dtype = x.dtype
    out, _ = mynn.add_rms_norm(x, None, w, eps)
    codes, scale, _ = mynn.add_rms_norm_quantize(x, None, w, eps)
    y, rel = exact(x, w, eps)
    # (values of the largest rows that are 2^-94 and less are nothing: below 2^-150 normalised)
    tiny = torch.finfo(dtype).smallest_normal * half_step(dtype) + 2.0**-149
    assert bool(((out.double() - y).abs() <= y.abs() * (half_step(dtype) * (1 + rel) + rel) + tiny)[rows].all())
    step = y.abs().amax(-1) / 127
    assert bool(((scale.double() - step).abs() <= step * (half_step(dtype) + 2 * rel + 2.0**-23) + tiny)[rows].all())
    assert bool(((codes.double() - y / step[:, None]).abs() <= 0.5 + 127 * (2 * rel + 2.0**-22))[rows].all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [8, 63, 64, 2048, 4096, 8200, 14336, 20000, 40000])
@pytest.mark.parametrize("rows", [6, 300])
def test_large_rows(dtype, dim, rows):
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((rows, dim), generator=g, device="cuda").to(dtype)
    w = (1.0 + 0.3 * torch.randn((dim,), generator=g, device="cuda")).to(dtype)
    plain = mynn.add_rms_norm(x, None, w, 1e-5)[0]
    x[0] = 1e20
    x[1] *= 1e30
    x[2, 0] = 3e38                               # (one value alone)
    x[3] = 3.3e38 * torch.sign(x[3])
    x[4, :4] = torch.tensor([1e38, 1e10, 1e-10, 1e-38], device="cuda").to(dtype)
    check(x, w, 1e-5)
    assert torch.equal(mynn.add_rms_norm(x, None, w, 1e-5)[0][5:], plain[5:])
    check(x, w, 1e38)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [8, 63, 2048, 8200, 40000])
def test_small_rows_without_eps(dtype, dim):
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((5, dim), generator=g, device="cuda")
    x[0] *= 1e-15
    x[1] *= 1e-20
    x[2] *= 1e-30
    x[3] *= 1e-17
    x = x.to(dtype)
    w = (1.0 + 0.3 * torch.randn((dim,), generator=g, device="cuda")).to(dtype)
    check(x, w, 0.0)
    check(x, w, 1e-40)
    check(x, w, 1e-30)
    check(x, w, 1e-5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [63, 2048])
def test_infinities_stay(dtype, dim):
    x = torch.ones((3, dim), dtype=dtype, device="cuda")
    x[0, 3] = float("inf")
    x[1] = 3e38
    x[1, 5] = float("nan")
    w = torch.ones((dim,), dtype=dtype, device="cuda")
    out, _ = mynn.add_rms_norm(x, None, w, 1e-5)
    codes, scale, _ = mynn.add_rms_norm_quantize(x, None, w, 1e-5)
    assert bool(out[0, 3].isnan()) and not bool(out[0, 4:].any()) and bool(out[1].isnan().all())
    assert bool(scale[:2].isnan().all()) and not bool(codes[:2].any()) and bool((codes[2] == 127).all())
