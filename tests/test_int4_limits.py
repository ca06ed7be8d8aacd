"""4-bit weights: sizes that an int of the C ABI would cut off are refused, and not taken for what is left of them."""
import importlib

import numpy as np
import pytest
import torch

mynn = importlib.import_module("my-nn-engine_amd")


@pytest.mark.parametrize("group", [(1 << 32) + 32, (1 << 32) + 64, 1 << 32, (1 << 31) + 128, -(1 << 32) + 32])
@pytest.mark.parametrize("symmetric", [True, False])
def test_groups_of_the_quantiser(group, symmetric):
    with pytest.raises(mynn.MynnError, match="group"):
        mynn.quantize_int4_groups(np.ones((2, 96), np.float32), group, mynn.F16, symmetric)


def test_columns_of_the_products():
    K = (1 << 32) + 128  # (broadcast views: no memory)
    wq = torch.zeros((1, 1), dtype=torch.uint8).expand(1, K // 2)
    scale = torch.ones((1, 1), dtype=torch.float16)
    with pytest.raises(mynn.MynnError, match="4-bit weights"):
        mynn.dequant_matmul_int4(torch.zeros((1, 1), dtype=torch.float16).expand(1, K), wq, scale)
    with pytest.raises(mynn.MynnError, match="4-bit weights"):
        mynn.quantized_matmul_int4(torch.zeros((1, 1), dtype=torch.int8).expand(1, K), scale[0], wq, scale)
