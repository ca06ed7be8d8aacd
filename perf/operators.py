"""The operators of 4-bit decoder weights as cases that can be timed: products of 16-bit and of int8 activations with weights of
4 bits and group scales, and the RMSNorm behind a residual's addition, with its output in 16 bits or in 8 with row scales.

A case is a dict of plain values; "op" says which operator:

  linear   dequant_matmul_int4: M rows of 16-bit activations times one 4-bit matrix [N, K]
  qlinear  quantized_matmul_int4: the same for int8 activations with a scale per row
  norm     add_rms_norm: the residual's addition and the norm of the sum, both returned
  qnorm    add_rms_norm_quantize: the same, the normalised rows in 8 bits; what the codes stand for comes back through
           dequantize_linear

A 4-bit matrix: codes 0 .. 15, two to a byte (the even column in the low four bits), in groups of `group` columns; a weight is
scale[n, g] * (code - zero[n, g]), zero 8 where a matrix has no zero points.

With `own` false the operators are computed by elementary tensor operations in 32 bits, with `own` true by the framework.  The
shapes are those of the two decoders of this repository's benchmark (hidden 2048 / feed-forward 5632 / vocabulary 32000 and
4096 / 14336 / 128256).
"""
import importlib
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
# (N, K) of the decoders' linear layers: q|k|v, o, gate|up, down
LINEARS = [(2560, 2048), (2048, 2048), (11264, 2048), (2048, 5632), (6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336)]


def listed():
    return [
        # one token through gate|up of the small decoder: a few microseconds
        dict(name="linear_f16_m1_gate_up", op="linear", dtype="f16", m=1, n=11264, k=2048, group=128, zero=False),
        # one token through a down projection with long rows, finer groups and zero points
        dict(name="linear_bf16_m1_down", op="linear", dtype="bf16", m=1, n=4096, k=14336, group=64, zero=True),
        # one token through the output matrix of the large decoder: the longest stream of weights
        dict(name="linear_bf16_m1_head", op="linear", dtype="bf16", m=1, n=128256, k=4096, group=128, zero=False),
        # six sequences of a small serving batch, the finest groups
        dict(name="linear_f16_m6_gate_up", op="linear", dtype="f16", m=6, n=28672, k=4096, group=32, zero=True),
        # a batch of 48 sequences
        dict(name="linear_bf16_m48_o", op="linear", dtype="bf16", m=48, n=4096, k=4096, group=128, zero=True),
        # a prompt of no particular length
        dict(name="linear_f16_m777_gate_up", op="linear", dtype="f16", m=777, n=28672, k=4096, group=128, zero=False),
        # one token in 8 bits through q|k|v
        dict(name="qlinear_bf16_m1_qkv", op="qlinear", dtype="bf16", m=1, n=6144, k=4096, group=128, zero=False),
        # 24 sequences in 8 bits through a down projection
        dict(name="qlinear_f16_m24_down", op="qlinear", dtype="f16", m=24, n=4096, k=14336, group=64, zero=True),
        # prompts in 8 bits
        dict(name="qlinear_bf16_m1000_gate_up", op="qlinear", dtype="bf16", m=1000, n=11264, k=2048, group=128, zero=True),
        # the norm of one token
        dict(name="norm_bf16_r1", op="norm", dtype="bf16", rows=1, dim=4096),
        # the 8-bit rows of one prompt
        dict(name="qnorm_f16_r300", op="qnorm", dtype="f16", rows=300, dim=2048),
        # the 8-bit rows of prompts in bulk
        dict(name="qnorm_bf16_r8192", op="qnorm", dtype="bf16", rows=8192, dim=4096),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["linear", "linear", "linear", "qlinear", "qlinear", "norm", "qnorm"])
    dtype = rng.choice(["f16", "bf16"])
    if op in ("norm", "qnorm"):
        # rows of whole 16-byte pieces mostly, of any length now and then
        dim = rng.choice([2048, 4096, 8 * _log(rng, 64, 1024), _log(rng, 500, 9000)])
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 8192), dim=dim)
    group = rng.choice([32, 64, 128])
    if rng.random() < 0.6:
        n, k = rng.choice(LINEARS)
    else:  # matrices of other models: any number of rows, any number of groups
        n, k = _log(rng, 500, 32000), group * _log(rng, 512 // group, 16384 // group)
    return dict(op=op, dtype=dtype, m=_log(rng, 1, 1024), n=n, k=k, group=group, zero=rng.random() < 0.5)


def _cost(case):
    w = work(case)
    return w["bytes"] / 8e12 + w["flops"] / 2.5e15


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw_once(rng)
        if _cost(case) <= most:
            return case


# ------------------------------------------------------------------ inputs
def _weight(case, g):
    """A 4-bit matrix as a quantiser leaves normally distributed weights: codes around the zero point that use the range."""
    n, k, group = case["n"], case["k"], case["group"]
    groups = k // group
    zero = torch.randint(5, 12, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zero"] else None
    centre = 8.0 if zero is None else zero.repeat_interleave(group, 1)
    codes = torch.randn((n, k), generator=g, device="cuda").mul_(2.6).add_(centre).round_().clamp_(0, 15).to(torch.uint8)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scale = ((torch.rand((n, groups), generator=g, device="cuda") + 0.5) / (2.6 * math.sqrt(k))).to(DTYPES[case["dtype"]])
    return packed, scale, zero


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] in ("norm", "qnorm"):
        rows, dim = case["rows"], case["dim"]
        s["x"] = torch.randn((rows, dim), generator=g, device="cuda").to(dtype)
        s["residual"] = (torch.randn((rows, dim), generator=g, device="cuda") * 3.0).to(dtype)
        s["w"] = (1.0 + 0.2 * torch.randn((dim,), generator=g, device="cuda")).to(dtype)
        return s
    m, k = case["m"], case["k"]
    s["wq"], s["scale"], s["zeros"] = _weight(case, g)
    if case["op"] == "linear":
        # a few channels much larger than the rest, as hidden states have them
        channels = 1.0 + 9.0 * (torch.rand((k,), generator=g, device="cuda") < 0.01)
        s["act"] = (torch.randn((m, k), generator=g, device="cuda") * channels).to(dtype)
    else:
        s["act"] = (torch.randn((m, k), generator=g, device="cuda") * 36.0).round_().clamp_(-127, 127).to(torch.int8)
        s["act_scale"] = ((torch.rand((m,), generator=g, device="cuda") + 0.5) / 36.0).to(dtype)
    return s


# ------------------------------------------------------------------ the operators
def _plain_weight(s):
    """[N, K] in 32 bits"""
    wq, scale = s["wq"], s["scale"].float()
    n, groups = scale.shape
    codes = torch.stack((wq & 15, wq >> 4), -1).reshape(n, groups, s["group"]).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None]
    return ((codes - zero) * scale[:, :, None]).reshape(n, s["k"])


def _plain_norm(s):
    """the stored sum, and its normalised rows in 32 bits"""
    total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    h = total.float()
    inv = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    return total, h * inv * s["w"].float()


def _plain(s):
    dtype = DTYPES[s["dtype"]]
    if s["op"] == "linear":
        return (s["act"].float() @ _plain_weight(s).t()).to(dtype)
    if s["op"] == "qlinear":
        return ((s["act"].float() @ _plain_weight(s).t()) * s["act_scale"].float()[:, None]).to(dtype)
    total, y = _plain_norm(s)
    if s["op"] == "norm":
        return {"out": y.to(dtype), "sum": total}
    scale = y.abs().amax(-1, keepdim=True) / 127.0
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = y / scale
    q = (torch.sign(q) * torch.floor(q.abs() + 0.5)).clamp(-127, 127)
    return {"values": (q * scale.to(dtype).float()).to(dtype), "scale": scale.to(dtype)[:, 0], "sum": total}


_mynn = None


def _own(s):
    global _mynn
    if _mynn is None:
        _mynn = importlib.import_module("my-nn-engine_amd")
    mynn = _mynn
    if s["op"] == "linear":
        return mynn.dequant_matmul_int4(s["act"], s["wq"], s["scale"], s["zeros"])
    if s["op"] == "qlinear":
        return mynn.quantized_matmul_int4(s["act"], s["act_scale"], s["wq"], s["scale"], s["zeros"])
    if s["op"] == "norm":
        out, total = mynn.add_rms_norm(s["x"], s["residual"], s["w"], EPS)
        return {"out": out, "sum": total}
    codes, scale, total = mynn.add_rms_norm_quantize(s["x"], s["residual"], s["w"], EPS)
    return {"values": mynn.dequantize_linear(codes, scale), "scale": scale, "sum": total}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    if case["op"] in ("norm", "qnorm"):
        rows, dim = case["rows"], case["dim"]
        # (8 bits: the codes are written, read again and returned as 16-bit values)
        moved = rows * dim * (2 + 2 + 2 + (2 if case["op"] == "norm" else 4)) + dim * 2 + (0 if case["op"] == "norm" else 4 * rows)
        return {"bytes": moved, "flops": 6 * rows * dim}
    m, n, k = case["m"], case["n"], case["k"]
    weight = n * k // 2 + n * (k // case["group"]) * (3 if case["zero"] else 2)
    act = m * k * 2 if case["op"] == "linear" else m * (k + 2)
    return {"bytes": weight + act + m * n * 2, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "qnorm"):
        x, r, w = s["x"].double(), s["residual"].double(), s["w"].double()
        stored = (x + r).to(s["x"].dtype).double()  # (the norm is the stored sum's)
        rms = torch.linalg.vector_norm(stored, dim=1).square().div(case["dim"]).add(EPS).sqrt()
        y = stored / rms[:, None] * w
        if case["op"] == "norm":
            return {"out": y, "sum": x + r}
        peak = y.abs().max(1).values
        step = torch.where(peak > 0, peak / 127.0, torch.ones_like(peak))
        codes = torch.trunc(y / step[:, None] + torch.copysign(torch.full_like(y, 0.5), y)).clamp(-127, 127)
        return {"values": codes * step.to(s["x"].dtype).double()[:, None], "scale": step, "sum": x + r}
    n, k, group = case["n"], case["k"], case["group"]
    weight = torch.empty((n, k), dtype=torch.float64, device="cuda")
    weight[:, 0::2] = (s["wq"] % 16).double()
    weight[:, 1::2] = (s["wq"] // 16).double()
    offset = torch.full_like(s["scale"], 8.0).double() if s["zeros"] is None else s["zeros"].double()
    weight -= offset.repeat_interleave(group, 1)
    weight *= s["scale"].double().repeat_interleave(group, 1)
    out = torch.mm(weight, s["act"].double().t().contiguous()).t()
    return out * s["act_scale"].double()[:, None] if case["op"] == "qlinear" else out
