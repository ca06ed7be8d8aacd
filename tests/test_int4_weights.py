"""4-bit weights without a GPU: the host quantiser, and what the products refuse."""
import ctypes as C
import importlib

import numpy as np
import pytest

mynn = importlib.import_module("my-nn-engine_amd")


def value(bits, dt):
    return bits.view(np.float16).astype(np.float64) if dt == mynn.F16 else (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def unpack(q):
    return np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1).astype(np.float64)


@pytest.mark.parametrize("dt", [mynn.F16, mynn.BF16])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("symmetric", [True, False])
def test_weights_within_half_a_step(dt, group, symmetric):
    rng = np.random.default_rng(1)
    w = rng.standard_normal((7, 512)).astype(np.float32) * np.exp(rng.uniform(-3, 3, (7, 1))).astype(np.float32)
    w[2] = np.abs(w[2])
    w[3] = -np.abs(w[3])
    w[4, :group] = 0.0
    q, s, z = mynn.quantize_int4_groups(w, group, dt, symmetric)
    scale = value(s, dt).repeat(group, 1)
    zero = 8.0 if symmetric else z.astype(np.float64).repeat(group, 1)
    eps = {mynn.F16: 2.0**-11, mynn.BF16: 2.0**-8}[dt]
    back = (unpack(q) - zero) * scale
    # half a step; where the stored step is below the exact one by eps, the last code is short by up to 15 eps of it; a zero point is rounded too
    assert np.all(np.abs(back - w) <= scale * (0.5 + (0 if symmetric else 0.5) + 16 * eps))
    assert np.all(back[4, :group] == 0) and np.all(scale[4, :group] == 1.0)


def test_codes_by_hand():
    w = np.zeros((1, 32), np.float32)
    w[0, :6] = [7.0, -7.0, 0.5, -0.5, 3.49, 1.5]
    q, s, z = mynn.quantize_int4_groups(w, 32, mynn.F16)
    assert z is None and value(s, mynn.F16)[0, 0] == 1.0
    assert list(unpack(q)[0, :7]) == [15, 1, 9, 7, 11, 10, 8]
    assert q[0, 0] == 0x1F  # (the even column in the low four bits)
    w[0, :6] = [10.0, -5.0, 0.4, 0.6, -4.6, 9.4]
    q, s, z = mynn.quantize_int4_groups(w, 32, mynn.F16, symmetric=False)
    assert value(s, mynn.F16)[0, 0] == 1.0 and z[0, 0] == 5
    assert list(unpack(q)[0, :7]) == [15, 0, 5, 6, 0, 14, 5]


def test_quantiser_refuses():
    w = np.ones((2, 96), np.float32)
    for group in (0, -32, 16, 48, 96, 100, 64):  # (64: 96 columns are one and a half groups)
        with pytest.raises(mynn.MynnError, match="group"):
            mynn.quantize_int4_groups(w, group, mynn.F16)
    with pytest.raises(mynn.MynnError, match="dtype"):
        mynn.quantize_int4_groups(w, 32, mynn.F32)
    for bad in (np.inf, np.nan, 3e38):
        w[1, 40] = bad
        with pytest.raises(mynn.MynnError, match="not finite|reach"):
            mynn.quantize_int4_groups(w, 32, mynn.F16)
        with pytest.raises(mynn.MynnError, match="not finite|reach"):
            mynn.quantize_int4_groups(w, 32, mynn.F16, symmetric=False)
    lib = mynn.lib()
    assert lib.mynn_quantize_int4_groups(None, None, None, None, 1, 32, 32, mynn.F16) == -1


def test_products_refuse_before_they_launch():
    """(no GPU here: a call that got past its checks would fail in the launch, with a positive status)"""
    lib = mynn.lib()
    buf = C.create_string_buffer(4096 + 16)
    p = (C.addressof(buf) + 15) & ~15
    odd = p + 2

    def linear(out=p, act=p, wq=p, scale=p, zero=None, M=1, N=4, K=128, group=128, dtype=mynn.F16):
        return lib.mynn_dequant_matmul_int4(out, act, wq, scale, zero, M, N, K, group, dtype, None)

    def qlinear(out=p, act=p, ls=p, wq=p, scale=p, zero=None, M=1, N=4, K=128, group=128, dtype=mynn.F16):
        return lib.mynn_quantized_matmul_int4(out, act, ls, wq, scale, zero, M, N, K, group, dtype, None)

    for f in (linear, qlinear):
        for k in ("out", "act", "wq", "scale"):
            assert f(**{k: None}) == -1, k
        for k in ("M", "N", "K"):
            assert f(**{k: 0}) == -1 and f(**{k: -5}) == -1
        for group in (0, -128, 16, 48, 96, 130, 192):
            assert f(K=128 * 3 * 5 * 13, group=group) == -2, group
        assert f(K=192) == -1 and f(K=100, group=32) == -1
        assert f(K=(1 << 22) + 128) == -2
        assert f(M=(1 << 30) + 1) == -2 and f(N=(1 << 31) - 1) == -2
        assert f(act=odd) == -1 and f(wq=odd) == -1
        for dtype in (mynn.F32, mynn.I8, 9):
            assert f(dtype=dtype) == -2
    assert qlinear(ls=None) == -1


def test_wrappers_refuse_before_they_call():
    import types

    import torch

    act, ls = torch.zeros((2, 64), dtype=torch.float16), torch.ones((2,), dtype=torch.float16)
    wq, scale, zero = torch.zeros((4, 32), dtype=torch.uint8), torch.ones((4, 2), dtype=torch.float16), torch.zeros((4, 2), dtype=torch.uint8)
    for bad in ((wq[0], scale, zero), (wq[None], scale, zero), (wq, scale[0], None), (wq, scale, zero[:1]), (wq[:, :0], scale, zero), (wq, scale[:, :0], None)):
        with pytest.raises(mynn.MynnError, match="4-bit weights"):
            mynn.dequant_matmul_int4(act, *bad)
        with pytest.raises(mynn.MynnError, match="4-bit weights"):
            mynn.quantized_matmul_int4(act.to(torch.int8), ls, *bad)
    for bad in (act[0, 0], act[:, :32], act.float(), act[None, :, :0]):
        with pytest.raises(mynn.MynnError, match="fit together"):
            mynn.dequant_matmul_int4(bad, wq, scale, zero)
    for bad in ((act.to(torch.int8)[0], ls), (act, ls), (act.to(torch.int8), ls[:1])):
        with pytest.raises(mynn.MynnError, match="fit together"):
            mynn.quantized_matmul_int4(*bad, wq, scale, zero)
    # more rows than an int counts (a broadcast view: no memory)
    with pytest.raises(mynn.MynnError, match="fit together"):
        mynn.dequant_matmul_int4(act[:1].expand((1 << 32) + 2, 64), wq, scale, zero)
    for norm in (mynn.add_rms_norm, mynn.add_rms_norm_quantize):
        for x, w in ((act[0, 0], act[0]), (act, act[0, :32]), (act[:1].expand((1 << 32) + 2, 64), act[0])):
            with pytest.raises(mynn.MynnError, match="fit together"):
                norm(x, None, w, 1e-5)
    # an operand of another device than the current one
    current = types.SimpleNamespace(_cuda_getDevice=lambda: 1)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(mynn, "_t", lambda: types.SimpleNamespace(_C=current))
        on = [types.SimpleNamespace(device=torch.device("cuda", i)) for i in range(2)]
        mynn._on_current_device("f", on[1], None)
        with pytest.raises(mynn.MynnError, match="cuda:0"):
            mynn._on_current_device("f", on[1], on[0])


def test_norm_refuses_before_it_launches():
    lib = mynn.lib()
    buf = C.create_string_buffer(4096)
    p = C.addressof(buf)

    def norm(out=p, total=None, x=p, residual=p, w=p, rows=1, dim=8, dtype=mynn.F16):
        return lib.mynn_add_rms_norm(out, total, x, residual, w, rows, dim, 1e-5, dtype, None)

    def qnorm(out=p, ys=p, total=None, x=p, residual=p, w=p, rows=1, dim=8, dtype=mynn.F16):
        return lib.mynn_add_rms_norm_quantize(out, ys, total, x, residual, w, rows, dim, 1e-5, dtype, None)

    for f in (norm, qnorm):
        for k in ("out", "x", "w"):
            assert f(**{k: None}) == -1
        for k in ("rows", "dim"):
            assert f(**{k: 0}) == -1 and f(**{k: -1}) == -1
        assert f(dtype=9) == -1
    assert norm(total=p) == -1 and qnorm(ys=None) == -1


def test_workspaces_are_asked_for_before_a_launch():
    lib = mynn.lib()
    need = lib.mynn_matmul_int4_workspace_bytes(48, 4096, 4096, 128)
    assert need > 0 and need % (48 * 4096 * 4) == 0
    # (few rows, and tiles that fill the device: none)
    assert lib.mynn_matmul_int4_workspace_bytes(1, 4096, 4096, 128) == 0 and lib.mynn_matmul_int4_workspace_bytes(2048, 28672, 4096, 128) == 0
    for bad in ((0, 4096, 4096, 128), (48, 0, 4096, 128), (48, 4096, -1, 128), (48, 4096, 4096, 0)):
        assert lib.mynn_matmul_int4_workspace_bytes(*bad) == 0
    buf = C.create_string_buffer(4096 + 16)
    p = (C.addressof(buf) + 15) & ~15
    for ws, size in ((None, 1 << 40), (p, need - 1), (p + 4, need)):
        assert lib.mynn_dequant_matmul_int4_ws(p, p, p, p, None, 48, 4096, 4096, 128, mynn.F16, ws, size, None) == -1
        assert b"workspace" in lib.mynn_last_error()
        assert lib.mynn_quantized_matmul_int4_ws(p, p, p, p, p, None, 48, 4096, 4096, 128, mynn.F16, ws, size, None) == -1


def test_kernels_use_no_scratch_memory(tmp_path):
    """sums, fragments and codes are registers in every form"""
    import os
    import re
    import subprocess

    from test_kernel_registers import LIB, READELF, device_code

    if not (os.path.exists(READELF) and os.path.exists(LIB)):
        pytest.skip("needs the built library and llvm-readelf")
    forms = {}
    for code in device_code(open(LIB, "rb").read()):
        if b"int4_tile_kernel" not in code and b"add_norm_vec_kernel" not in code:
            continue
        (tmp_path / "code").write_bytes(code)
        notes = subprocess.check_output([READELF, "--notes", str(tmp_path / "code")], text=True)
        for name, scratch in re.findall(r"\.name:\s+(\S*(?:int4|add_norm)\S*)\n(?:(?!\.name:).)*?\.private_segment_fixed_size:\s+(\d+)", notes, re.S):
            forms[name] = int(scratch)
    assert sum("int4_tile" in n for n in forms) == 40 and sum("int4_stream" in n for n in forms) >= 72 and sum("add_norm_vec" in n for n in forms) == 24
    assert not {k: v for k, v in forms.items() if v}
