"""The residual's addition with the RMSNorm behind it, in 16 bits, 32 bits and in 8 with row scales, against 64 bits."""
import importlib

import pytest
import torch

import int4_reference as ref

mynn = importlib.import_module("my-nn-engine_amd")
pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-5


def operands(rows, dim, dtype, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn((rows, dim), generator=g, device="cuda").to(dtype)
    r = (torch.randn((rows, dim), generator=g, device="cuda") * 2).to(dtype)
    return x, r, (1.0 + 0.3 * torch.randn((dim,), generator=g, device="cuda")).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_sum(total, x, r):
    exact = x.double() + (r.double() if r is not None else 0.0)
    # (added in 32 bits, then rounded: half a step of each)
    assert bool(((total.double() - exact).abs() <= exact.abs() * (half_step(total.dtype) + 2.0**-23)).all())


def exact_norm(total, w):
    """in 64 bits, and how far off 32 bits may be, relative: the sum of dim squares (a term goes through at most dim/256 + 16 additions in any of the
    forms here, and its own rounding), the mean, the root, the reciprocal, two products, each half a unit; the root halves the sum's"""
    h = total.double()
    y = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    return y, ((h.shape[-1] / 256 + 17) / 2 + 6) * 2.0**-24


DIMS = [1, 2, 7, 8, 9, 64, 100, 512, 520, 1000, 2047, 2048, 2056, 4096, 5632, 8184, 8192, 8200, 14336, 16384, 16392, 20000]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [1, 2, 5, 130])
@pytest.mark.parametrize("dim", DIMS)
def test_norm(dtype, rows, dim):
    x, r, w = operands(rows, dim, dtype)
    for residual in (r, None):
        out, total = mynn.add_rms_norm(x, residual, w, EPS)
        check_sum(total, x, residual)
        y, rel = exact_norm(total, w)
        assert bool(((out.double() - y).abs() <= y.abs() * (half_step(dtype) * (1 + rel) + rel) + torch.finfo(dtype).smallest_normal * half_step(dtype)).all())


def check_codes(codes, scale, total, w):
    y, rel = exact_norm(total, w)
    amax = y.abs().amax(-1)
    step = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    tiny = torch.finfo(scale.dtype).smallest_normal * half_step(scale.dtype)
    assert bool(((scale.double() - step).abs() <= step * (half_step(scale.dtype) + 2 * rel + 2.0**-23) + tiny).all())
    # a code is the value over the unrounded step, rounded: half a step, and what 32 bits leave open of a quotient of up to 127
    off = (codes.double() - y / step[:, None]).abs()
    assert bool((off <= 0.5 + 127 * (2 * rel + 2.0**-22)).all()), float(off.max())
    assert bool((codes.int().abs().amax(-1) == torch.where(amax > 0, 127, 0)).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [1, 3, 130])
@pytest.mark.parametrize("dim", DIMS)
def test_norm_quantized(dtype, rows, dim):
    x, r, w = operands(rows, dim, dtype)
    for residual in (r, None):
        codes, scale, total = mynn.add_rms_norm_quantize(x, residual, w, EPS)
        check_sum(total, x, residual)
        check_codes(codes, scale, total, w)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,dim", [(2047, 2048), (2048, 2048), (5000, 1024), (2100, 4096), (2048, 8192), (3000, 264)])
def test_many_rows(dtype, rows, dim):
    x, r, w = operands(rows, dim, dtype)
    out, total = mynn.add_rms_norm(x, r, w, EPS)
    check_sum(total, x, r)
    y, rel = exact_norm(total, w)
    assert bool(((out.double() - y).abs() <= y.abs() * (half_step(dtype) * (1 + rel) + rel) + torch.finfo(dtype).smallest_normal * half_step(dtype)).all())
    codes, scale, again = mynn.add_rms_norm_quantize(x, r, w, EPS)
    assert torch.equal(total, again)
    check_codes(codes, scale, total, w)


def test_leading_dimensions():
    x, r, w = operands(12, 640, BF16)
    out, total = mynn.add_rms_norm(x, r, w, EPS)
    codes, scale, _ = mynn.add_rms_norm_quantize(x, r, w, EPS)
    o3, t3 = mynn.add_rms_norm(x.view(3, 4, 640), r.view(3, 4, 640), w, EPS)
    c3, s3, _ = mynn.add_rms_norm_quantize(x.view(3, 4, 640), r.view(3, 4, 640), w, EPS)
    assert torch.equal(o3.view(12, 640), out) and torch.equal(t3.view(12, 640), total) and torch.equal(c3.view(12, 640), codes) and torch.equal(s3, scale)


def raw(name, out, *args):
    rc = getattr(mynn.lib(), name)(out, *args, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, mynn.lib().mynn_last_error()


# in place, and at addresses that no vector load takes; what lies around the outputs stays as it was
@pytest.mark.parametrize("dtype,code", [(F16, mynn.F16), (BF16, mynn.BF16), (F32, mynn.F32)])
@pytest.mark.parametrize("rows,dim", [(1, 4096), (9, 2048), (3, 1001), (2500, 512)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_in_place_and_odd_places(dtype, code, rows, dim, shift):
    x, r, w = operands(rows, dim, dtype)
    out, total = mynn.add_rms_norm(x, r, w, EPS)
    codes, scale, _ = mynn.add_rms_norm_quantize(x, r, w, EPS)
    n = rows * dim

    def moved(t, dt=None):
        buf = torch.full((n + 16,), 5, dtype=t.dtype, device="cuda")
        view = buf[shift : shift + t.numel()]
        view.copy_(t.flatten())
        return buf, view

    def around(buf, n_=n):
        return bool((buf[:shift] == 5).all()) and bool((buf[shift + n_ :] == 5).all())

    close = dict(rtol=2 * half_step(dtype) + 1e-6, atol=1e-7)  # (another form may add the squares up in another order: a step of the output's type)
    for sum_is, out_is in (("x", "r"), ("r", "x"), ("x", None), ("r", None), (None, "x"), (None, "r")):
        (xb, xv), (rb, rv), (_, wv) = moved(x), moved(r), moved(w)
        ob, ov = moved(torch.zeros_like(x))
        where = {"x": xv, "r": rv}
        sum_p = where[sum_is].data_ptr() if sum_is else None
        o = where[out_is] if out_is else ov
        raw("mynn_add_rms_norm", o.data_ptr(), sum_p, xv.data_ptr(), rv.data_ptr(), wv.data_ptr(), rows, dim, EPS, code)
        assert torch.allclose(o.view(rows, dim).double(), out.double(), **close)
        if sum_is:
            assert torch.equal(where[sum_is].view(rows, dim), total)
        assert around(xb) and around(rb) and around(ob)
    for sum_is in ("x", "r", None):
        (xb, xv), (rb, rv), (_, wv) = moved(x), moved(r), moved(w)
        yb = torch.full((n + 16,), 5, dtype=torch.int8, device="cuda")
        sb = torch.full((rows + 16,), 5, dtype=dtype, device="cuda")
        where = {"x": xv, "r": rv}
        raw("mynn_add_rms_norm_quantize", yb.data_ptr() + shift, sb.data_ptr() + shift * sb.element_size(), where[sum_is].data_ptr() if sum_is else None,
            xv.data_ptr(), rv.data_ptr(), wv.data_ptr(), rows, dim, EPS, code)
        check_codes(yb[shift : shift + n].view(rows, dim), sb[shift : shift + rows], total, w)
        assert around(yb) and around(sb, rows) and around(xb) and around(rb)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,dim", [(4, 2048), (4, 777), (3000, 1024)])
def test_rows_of_zeros_and_what_is_not_finite(dtype, rows, dim):
    x, r, w = operands(rows, dim, dtype)
    clean = mynn.add_rms_norm(x, r, w, EPS)
    cleanq = mynn.add_rms_norm_quantize(x, r, w, EPS)
    x[0] = 1.5
    r[0] = -1.5
    x[1, 5] = float("nan")
    x[2, 9] = float("inf")
    out, total = mynn.add_rms_norm(x, r, w, EPS)
    codes, scale, _ = mynn.add_rms_norm_quantize(x, r, w, EPS)
    assert not bool(total[0].any()) and not bool(out[0].any()) and not bool(codes[0].any()) and float(scale[0]) == 1.0
    assert bool(out[1].isnan().all()) and bool(out[2, 9].isnan())
    assert bool(scale[1].isnan()) and bool(scale[2].isnan()) and not bool(codes[1:3].any())
    assert torch.equal(out[3:], clean[0][3:]) and torch.equal(codes[3:], cleanq[0][3:]) and torch.equal(scale[3:], cleanq[1][3:])


def test_offsets_beyond_32_bits():
    rows, dim = 70000, 32768
    assert rows * dim > 2**31
    x = torch.zeros((rows, dim), dtype=BF16, device="cuda")
    x[-3:] = torch.randn((3, dim), device="cuda").to(BF16)
    x[70] = 1.0
    w = torch.ones((dim,), dtype=BF16, device="cuda")
    out, _ = mynn.add_rms_norm(x, None, w, EPS)
    y, rel = exact_norm(x[-3:], w)
    assert bool(((out[-3:].double() - y).abs() <= y.abs() * (half_step(BF16) * (1 + rel) + rel)).all())
    del out
    codes, scale, _ = mynn.add_rms_norm_quantize(x, None, w, EPS)
    check_codes(codes[-3:], scale[-3:], x[-3:], w)
    assert not bool(codes[100].any())


@pytest.mark.parametrize("dtype,dim", [(F16, 8), (F32, 3)])
def test_more_rows_than_a_launch_has_room_for(dtype, dim):
    rows = (1 << 24) + 5
    x, r, w = operands(rows, dim, dtype)
    out, total = mynn.add_rms_norm(x, r, w, EPS)
    codes, scale, again = mynn.add_rms_norm_quantize(x, r, w, EPS)
    assert torch.equal(total, again)
    for at in (0, (1 << 21) - 3, (1 << 22) - 3, 5 << 21, (1 << 24) - 3):
        rows = slice(at, at + 8)
        check_sum(total[rows], x[rows], r[rows])
        y, rel = exact_norm(total[rows], w)
        assert bool(((out[rows].double() - y).abs() <= y.abs() * (half_step(dtype) * (1 + rel) + rel) + torch.finfo(dtype).smallest_normal * half_step(dtype)).all())
        check_codes(codes[rows], scale[rows], total[rows], w)


@pytest.mark.parametrize("rows,dim", [(1, 4096), (300, 2048), (4096, 1024)])
def test_captured_calls(rows, dim):
    x, r, w = operands(rows, dim, F16)
    out, total = mynn.add_rms_norm(x, r, w, EPS)
    codes, scale, _ = mynn.add_rms_norm_quantize(x, r, w, EPS)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o, t = mynn.add_rms_norm(x, r, w, EPS)
        c, s, _ = mynn.add_rms_norm_quantize(x, r, w, EPS)
    for _ in range(3):
        o.zero_(), t.zero_(), c.zero_(), s.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, out) and torch.equal(t, total) and torch.equal(c, codes) and torch.equal(s, scale)


def test_the_way_without_the_module(monkeypatch):
    x, r, w = operands(6, 640, F16)
    expected = [mynn.add_rms_norm(x, r, w, EPS), mynn.add_rms_norm_quantize(x, r, w, EPS), mynn.add_rms_norm(x, None, w, EPS), mynn.add_rms_norm_quantize(x, None, w, EPS)]
    codes, scale = expected[1][:2]
    values = mynn.dequantize_linear(codes, scale)
    monkeypatch.setattr(mynn, "_ops", mynn._NoHostOps())
    again = [mynn.add_rms_norm(x, r, w, EPS), mynn.add_rms_norm_quantize(x, r, w, EPS), mynn.add_rms_norm(x, None, w, EPS), mynn.add_rms_norm_quantize(x, None, w, EPS)]
    for a, b in zip(expected, again):
        assert len(a) == len(b) and all(torch.equal(u, v) for u, v in zip(a, b))
    assert expected[2][1] is not None and again[2][1] is x and torch.equal(mynn.dequantize_linear(codes, scale), values)


# dequantize_linear of whole pieces of eight and of others, at any address: code times scale, rounded once
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,cols,shift", [(1, 8, 0), (7, 4096, 0), (300, 200, 0), (5, 33, 0), (9, 64, 1), (3, 4096, 4)])
def test_dequantize_linear(dtype, rows, cols, shift):
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    buf = torch.randint(-128, 128, (rows * cols + 8,), generator=g, dtype=torch.int8, device="cuda")
    x = buf[shift : shift + rows * cols].view(rows, cols)
    scale = torch.rand((rows,), generator=g, device="cuda").to(dtype)
    assert torch.equal(mynn.dequantize_linear(x, scale), (x.float() * scale.float()[:, None]).to(dtype))


def test_wrapper_refuses_what_does_not_fit():
    x, r, w = operands(4, 64, F16)
    for f in (mynn.add_rms_norm, mynn.add_rms_norm_quantize):
        for bad in ((x, r[:3], w), (x, r.float(), w), (x, r, w[:32]), (x, r, w.float()), (x[:0], r[:0], w), (x.t(), r.t(), w[:4]), (x.cpu(), r, w),
                    (x, r.to(BF16), w)):
            with pytest.raises((mynn.MynnError, AssertionError)):
                f(*bad, EPS)
        with pytest.raises((mynn.MynnError, AssertionError, KeyError)):
            f(x.double(), r.double(), w.double(), EPS)


# a layer's 4-bit feed-forward block as it is used: the norm, the products and the existing operators between them, captured
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 6, 40, 200])
def test_feed_forward_block(dtype, rows):
    hidden, ffn, group = 512, 1408, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    x, r, w = operands(rows, hidden, dtype)
    gate, up, down = (ref.matrix(n, k, gr, dtype, z, g) for n, k, gr, z in ((ffn, hidden, group, True), (ffn, hidden, 128, False), (hidden, ffn, 128, True)))

    def block16():
        y, h = mynn.add_rms_norm(x, r, w, EPS)
        mid = mynn.swiglu(mynn.dequant_matmul_int4(y, *gate), mynn.dequant_matmul_int4(y, *up))
        return mynn.add_rms_norm(mynn.dequant_matmul_int4(mid, *down), h, w, EPS)

    def block8():
        y, s, h = mynn.add_rms_norm_quantize(x, r, w, EPS)
        mid = mynn.swiglu(mynn.quantized_matmul_int4(y, s, *gate), mynn.quantized_matmul_int4(y, s, *up))
        c, cs, _ = mynn.dynamic_quantize_linear(mid)
        return mynn.add_rms_norm(mynn.quantized_matmul_int4(c, cs, *down), h, w, EPS)

    def exact():
        h = x.double() + r.double()
        norm = lambda t: t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()  # noqa: E731
        times = lambda t, m: t @ (lambda d, s: d * s)(*ref.differences(*m)).t().contiguous()  # noqa: E731
        y = norm(h)
        h = h + times(torch.nn.functional.silu(times(y, gate)) * times(y, up), down)
        return norm(h), h

    want = exact()
    # roundings to T in a row of the 16-bit block, each at most half a step, seen from the end: y, gate, up, silu * up, down, h twice, out,
    # with gate and up meeting as a product; the 8-bit block rounds y and the middle to 1/254 of their row's largest value (of a row of
    # some 512 or 1408 values that is 3 to 4 deviations, an error of 4/254/sqrt(3) of the root mean square) and adds those of its scales
    eps = half_step(dtype)
    for block, most in ((block16, 9 * eps), (block8, 9 * eps + 4 * eps + 3 * 4 / 254 / 3**0.5)):
        eager = block()
        for got, exact_ in zip(eager, want):
            rel = float((got.double() - exact_).norm() / exact_.norm())
            assert rel <= most, (rel, most)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = block()
        for _ in range(3):
            for t in out:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
