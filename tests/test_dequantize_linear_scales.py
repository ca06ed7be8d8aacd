"""dequantize_linear: a scale for each row of the codes, in as many leading dimensions as there are."""
import importlib
import types

import pytest
import torch

mynn = importlib.import_module("my-nn-engine_amd")
BF16 = torch.bfloat16


def test_scales_that_do_not_fit_are_refused():
    """(before any memory is looked at: without a GPU too)"""
    for shape, n in (((4, 64), 3), ((4, 64), 5), ((4, 64), 2), ((2, 3, 64), 3), ((2, 3, 64), 5), ((2, 3, 64), 7), ((2, 3, 64), 1), ((0, 64), 0), ((4, 0), 4), ((), 1)):
        with pytest.raises(mynn.MynnError, match="fit together"):
            mynn.dequantize_linear(torch.zeros(shape, dtype=torch.int8), torch.ones((n,)))


def test_operands_of_another_device_are_refused(monkeypatch):
    on = [types.SimpleNamespace(device=torch.device("cuda", i), is_cuda=False, shape=(4, 8), dim=lambda: 2, numel=lambda n=n: n) for i, n in ((1, 32), (0, 4))]
    monkeypatch.setattr(mynn, "_t", lambda: types.SimpleNamespace(_C=types.SimpleNamespace(_cuda_getDevice=lambda: 1)))
    with pytest.raises(mynn.MynnError, match="cuda:0"):
        mynn.dequantize_linear(*on)


@pytest.mark.gpu
@pytest.mark.parametrize("module", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, BF16, torch.float32])
def test_leading_dimensions(dtype, module, monkeypatch):
    if not module:
        monkeypatch.setattr(mynn, "_ops", mynn._NoHostOps())
    g = torch.Generator(device="cuda").manual_seed(4)
    for shape, n in (((12, 640), 12), ((3, 4, 640), 12), ((3, 4, 640), 3), ((3, 4, 33), 12), ((2, 3, 5, 16), 6), ((2, 3, 5, 16), 30), ((1, 1, 64), 1), ((7,), 7), ((2, 3, 5), 30)):
        x = torch.randint(-128, 128, shape, generator=g, dtype=torch.int8, device="cuda")
        scale = torch.rand((n,), generator=g, device="cuda").to(dtype)
        want = (x.view(n, -1).float() * scale.float()[:, None]).to(dtype).view(shape)
        assert torch.equal(mynn.dequantize_linear(x, scale), want)
        for wrong in (n - 1, n + 1):
            if wrong not in (shape[0], shape[0] * (shape[1] if len(shape) > 1 else 1)):
                with pytest.raises(mynn.MynnError, match="fit together"):
                    mynn.dequantize_linear(x, torch.ones((wrong,), dtype=dtype, device="cuda"))


@pytest.mark.gpu
def test_codes_of_the_norm_in_three_dimensions():
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((3, 5, 640), generator=g, device="cuda").to(BF16)
    w = torch.ones((640,), dtype=BF16, device="cuda")
    codes, scale, _ = mynn.add_rms_norm_quantize(x, None, w, 1e-5)
    assert codes.shape == x.shape and scale.shape == (15,)
    flat = mynn.dequantize_linear(codes.view(15, 640), scale)
    assert torch.equal(mynn.dequantize_linear(codes, scale), flat.view(3, 5, 640))
