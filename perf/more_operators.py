"""Operators around a paged KV cache as cases that can be timed: the position rotation with the append of keys and values to pools
of 16, 8 or 4 bits, and attention over a cache that is held in 4 bits.

A case is a dict of plain values; "op" says which operator:

  append  rope_append_paged: q, k and v of S new tokens of B sequences, views of the projection's rows; q and k are rotated by their
          positions, k and v go to the pools.  Of 8- and 4-bit pools what the new rows stand for comes back through kv_rows_paged.
  attend  attention_paged_int4: S query rows of each of B sequences over its cached rows, those of the S new tokens the last of them

The pools of a 4-bit cache, for keys and for values: codes uint8 [pages, Hkv, rows, D/2] (the even column in the low four bits),
scales [pages, Hkv, rows, D/group] and zero points uint8 like the scales; a value is scale * (code - zero).  Sequence b has past[b]
rows in the cache and new[b] <= S new tokens; row r of it is row r % rows of page table[b, r / rows].

With `own` false the operators are computed by elementary tensor operations in 32 bits, with `own` true by the framework.  The
head shapes are those of the two decoders of this repository's benchmark (32 query heads over 4 kv heads of 64, over 8 of 128) and of
smaller ones in its tests.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# (query heads, kv heads, head size)
HEADS = [(32, 4, 64), (32, 8, 128), (32, 32, 128), (16, 4, 64), (8, 1, 128), (8, 8, 64)]


def listed():
    return [
        # one token of one sequence, 16-bit pools: the smallest call, nothing but latency
        dict(name="append_f16_b1", op="append", dtype="f16", b=1, s=1, past=1000, ragged=False, hq=32, hkv=4, d=64, page=64, bits=16, group=0),
        # a decode step of a serving batch whose sequences are of all lengths, 4-bit pools
        dict(name="append_bf16_int4_b32", op="append", dtype="bf16", b=32, s=1, past=4000, ragged=True, hq=32, hkv=8, d=128, page=256, bits=4, group=64),
        # three prompts of their own lengths in one padded call, 8-bit pools
        dict(name="append_f16_int8_3x333", op="append", dtype="f16", b=3, s=333, past=50, ragged=True, hq=32, hkv=4, d=64, page=64, bits=8, group=0),
        # prompts in bulk, 4-bit pools
        dict(name="append_bf16_int4_4x2048", op="append", dtype="bf16", b=4, s=2048, past=0, ragged=False, hq=32, hkv=8, d=128, page=256, bits=4, group=128),
        # the token of a chat: one sequence, a thousand rows
        dict(name="attend_f16_b1_1000", op="attend", dtype="f16", b=1, s=1, past=999, ragged=False, hq=32, hkv=4, d=64, page=64, group=64),
        # one sequence over a long document
        dict(name="attend_bf16_b1_32768", op="attend", dtype="bf16", b=1, s=1, past=32767, ragged=False, hq=32, hkv=8, d=128, page=256, group=128),
        # a serving batch of sequences of all lengths
        dict(name="attend_bf16_b32_ragged", op="attend", dtype="bf16", b=32, s=1, past=4096, ragged=True, hq=32, hkv=8, d=128, page=256, group=64),
        # four drafted tokens to be verified, the finest groups
        dict(name="attend_f16_b8_s4", op="attend", dtype="f16", b=8, s=4, past=2001, ragged=True, hq=32, hkv=8, d=128, page=128, group=32),
        # a full batch over long caches: what the memory gives
        dict(name="attend_f16_b64_8192", op="attend", dtype="f16", b=64, s=1, past=8191, ragged=False, hq=32, hkv=8, d=128, page=256, group=128),
        # one prompt of no particular length
        dict(name="attend_bf16_prompt_777", op="attend", dtype="bf16", b=1, s=777, past=0, ragged=False, hq=32, hkv=4, d=64, page=64, group=64),
        # pieces of two prompts behind what is cached of them
        dict(name="attend_f16_piece_2x512", op="attend", dtype="f16", b=2, s=512, past=3001, ragged=True, hq=32, hkv=8, d=128, page=256, group=128),
        # prompts in bulk
        dict(name="attend_bf16_prompts_4x2048", op="attend", dtype="bf16", b=4, s=2048, past=0, ragged=False, hq=32, hkv=8, d=128, page=256, group=128),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["append", "attend", "attend"])
    hq, hkv, d = rng.choice(HEADS)
    case = dict(op=op, dtype=rng.choice(["f16", "bf16"]), hq=hq, hkv=hkv, d=d, page=rng.choice([32, 64, 128, 256]), ragged=rng.random() < 0.6)
    case["group"] = rng.choice([g for g in (32, 64, 128) if g <= d])
    if op == "append":
        case["bits"] = rng.choice([16, 8, 4, 4])
        if case["bits"] != 4:
            case["group"] = 0
    kind = rng.choice(["token", "token", "drafts", "prompt"])
    if kind == "token":
        case.update(b=_log(rng, 1, 64), s=1, past=_log(rng, 1, 32768) - 1)
    elif kind == "drafts":
        case.update(b=_log(rng, 1, 32), s=rng.randint(2, 12), past=_log(rng, 1, 8192) - 1)
    else:
        case.update(b=_log(rng, 1, 8), s=_log(rng, 13, 2048), past=rng.choice([0, _log(rng, 1, 4096)]))
    return case


def _cost(case):
    w = work(case)
    return w["bytes"] / 8e12 + w["flops"] / 2.5e15


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw_once(rng)
        # (the plain form holds what the cache stands for in 32 bits, and every score of a prompt)
        rows = case["b"] * case["hkv"] * (case["past"] + case["s"]) * case["d"]
        scores = case["b"] * case["hq"] * case["s"] * (case["past"] + case["s"])
        if _cost(case) <= most and rows <= 64 * 8 * 8192 * 128 and scores <= 4 * 32 * 2048 * 2048:
            return case


# ------------------------------------------------------------------ inputs
def _lens(case):
    """(rows in the cache, new tokens) of each sequence: of all lengths up to the case's own where it is ragged, the first one full"""
    past, new = [], []
    for i in range(case["b"]):
        part = 1.0 if not case["ragged"] or i == 0 else (0.15 + 0.618034 * i) % 1.0
        past.append(int(round(case["past"] * part)))
        new.append(max(1, int(round(case["s"] * (1.0 if not case["ragged"] or i == 0 else (0.4 + 0.754878 * i) % 1.0)))))
    return past, new


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _round(x):
    """to the nearest whole number, halves away from zero"""
    t = x.trunc()
    return t + torch.where((x - t).abs() >= 0.5, x.sign(), torch.zeros_like(x))


def _quantize4(x, group, dtype):
    """rows [.., D] of 32-bit numbers -> (codes [.., D/2], scales [.., D/group], zero points like the scales)"""
    v = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    lo, hi = v.amin(-1).clamp_max(0.0), v.amax(-1).clamp_min(0.0)
    fifteen = torch.full_like(hi, 15.0)  # (by a number, a tensor is multiplied with its rounded reciprocal)
    s = (hi / fifteen - lo / fifteen).to(dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)
    z = _round(-lo / s.float()).clamp_max(15.0)
    c = (_round(v / s.float()[..., None]) + z[..., None]).clamp(0.0, 15.0).to(torch.uint8).reshape(x.shape)
    return c[..., 0::2] | (c[..., 1::2] << 4), s, z.to(torch.uint8)


def _table(case, g):
    """pages handed out in no order, -1 where a sequence has none"""
    past, new = _lens(case)
    pages = [(p + n + case["page"] - 1) // case["page"] for p, n in zip(past, new)]
    order = torch.randperm(sum(pages) + 5, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["b"], max(pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(pages) + 5


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    s = dict(case)
    past, new = _lens(case)
    s["past_lens"] = torch.tensor(past, dtype=torch.int32, device="cuda")
    s["new_lens"] = torch.tensor(new, dtype=torch.int32, device="cuda") if case["ragged"] and case["s"] > 1 else None
    s["table"], n_pages = _table(case, g)
    shape = (n_pages, hkv, case["page"])
    s["rows"] = case["past"] + case["s"]  # the longest sequence's
    # a few channels of keys are much larger than the rest, as projections of hidden states have them
    channels = 1.0 + 5.0 * (torch.rand((hkv, 1, d), generator=g, device="cuda") < 0.04)
    if case["op"] == "append":
        qkv = _normal(g, case["b"], case["s"], hq + 2 * hkv, d)
        qkv[:, :, hq:hq + hkv] *= channels[:, 0]
        s["qkv"] = qkv.to(dtype).reshape(case["b"], case["s"], (hq + 2 * hkv) * d)
        angle = torch.arange(s["rows"], dtype=torch.float64, device="cuda")[:, None] / 10000.0 ** (torch.arange(d // 2, dtype=torch.float64, device="cuda") * 2 / d)
        angle = torch.cat((angle, angle), 1)
        s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
        if case["bits"] == 16:
            s["pools"] = tuple(_normal(g, *shape, d).to(dtype) for _ in range(2))
        elif case["bits"] == 8:
            s["pools"] = (torch.zeros(shape + (d,), dtype=torch.int8, device="cuda"), torch.zeros(shape + (d,), dtype=torch.int8, device="cuda"),
                          torch.zeros(shape, dtype=dtype, device="cuda"), torch.zeros(shape, dtype=dtype, device="cuda"))
        else:
            s["pools"] = tuple(torch.zeros(shape + (n,), dtype=t, device="cuda") for n, t in ((d // 2, torch.uint8), (d // case["group"], dtype), (d // case["group"], torch.uint8))
                               for _ in range(2))
        return s
    s["q"] = _normal(g, case["b"], hq, case["s"], d).to(dtype)
    s["scale"] = d ** -0.5
    pools = []
    for part in (channels, torch.ones_like(channels)):
        codes, scale, zero = [], [], []
        for at in range(0, n_pages, 256):
            x = _normal(g, min(256, n_pages - at), hkv, case["page"], d) * part
            for to, t in zip((codes, scale, zero), _quantize4(x, case["group"], dtype)):
                to.append(t)
        pools.append([torch.cat(t) for t in (codes, scale, zero)])
    s["pools"] = tuple(t for pair in zip(*pools) for t in pair)
    s["workspace"] = None
    return s


# ------------------------------------------------------------------ the operators
def _plain_rotate(x, cos, sin):
    """rows [B, H, S, D] in 32 bits by table rows [B, S, D]"""
    half = x.shape[-1] // 2
    cos, sin = cos.float()[:, None], sin.float()[:, None]
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat((lo * cos[..., :half] - hi * sin[..., :half], hi * cos[..., half:] + lo * sin[..., half:]), -1)


def _views(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    x = s["qkv"].view(s["b"], s["s"], hq + 2 * hkv, d).transpose(1, 2)
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


def _plain_append(s):
    dtype = DTYPES[s["dtype"]]
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    q, k, v = _views(s)
    i = torch.arange(s["s"], device="cuda")
    row = s["past_lens"].long()[:, None] + i  # [B, S]
    there = torch.ones_like(row, dtype=torch.bool) if s["new_lens"] is None else i < s["new_lens"][:, None]
    at = torch.where(there, row, torch.zeros_like(row))
    cos, sin = s["cos"][at], s["sin"][at]
    q = torch.where(there[:, None, :, None], _plain_rotate(q.float(), cos, sin), torch.zeros((), device="cuda")).to(dtype)
    k = _plain_rotate(k.float(), cos, sin).to(dtype)
    page = s["table"].long().gather(1, at // s["page"])[there]
    put = (page[:, None], torch.arange(hkv, device="cuda"), (at % s["page"])[there][:, None])  # [tokens, Hkv]
    values = []
    for side, x in enumerate((k, v)):
        x = x.transpose(1, 2)[there]  # [tokens, Hkv, D]
        if s["bits"] == 16:
            s["pools"][side][put] = x
            continue
        x = x.float()
        if s["bits"] == 8:
            peak = x.abs().amax(-1, keepdim=True)
            y = x * torch.where(peak == 0, torch.zeros_like(peak), torch.full_like(peak, 127.0) / peak)
            codes, scale = (y + torch.where(y >= 0, 0.5, -0.5)).trunc().clamp(-128, 127).to(torch.int8), (peak * (1.0 / 127.0)).to(dtype)
            s["pools"][side][put], s["pools"][2 + side][put] = codes, scale[..., 0]
            x = codes.float() * scale.float()
        else:
            codes, scale, zero = _quantize4(x, s["group"], dtype)
            s["pools"][side][put], s["pools"][2 + side][put], s["pools"][4 + side][put] = codes, scale, zero
            x = _plain_values(codes, scale, zero)
        rows = torch.zeros((s["b"], s["s"], hkv, d), dtype=dtype, device="cuda")
        rows[there] = x.to(dtype)
        values.append(rows.transpose(1, 2))
    if s["bits"] == 16:
        return {"q": q, "k_pool": s["pools"][0], "v_pool": s["pools"][1]}
    return {"q": q, "k": values[0], "v": values[1]}


def _plain_values(codes, scale, zero):
    """what 4-bit rows [.., D/2] stand for, in 32 bits"""
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(*scale.shape, -1).float()
    return ((c - zero.float()[..., None]) * scale.float()[..., None]).reshape(*codes.shape[:-1], -1)


def _plain_attend(s):
    dtype = DTYPES[s["dtype"]]
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    b, rows = s["b"], s["rows"]
    pages = s["table"].long().clamp_min(0)  # [B, pages]
    kv = []
    for side in (0, 1):
        codes, scale, zero = (s["pools"][n + side][pages].transpose(1, 2).flatten(2, 3)[:, :, :rows] for n in (0, 2, 4))  # [B, Hkv, rows, ..]
        kv.append(_plain_values(codes, scale, zero))
    new = torch.full_like(s["past_lens"], s["s"]) if s["new_lens"] is None else s["new_lens"]
    i = torch.arange(s["s"], device="cuda")
    bound = torch.where(i < new[:, None], s["past_lens"][:, None] + i + 1, 0)  # [B, S] keys that a row sees
    hidden = torch.arange(rows, device="cuda") >= bound[..., None]  # [B, S, rows]
    q = s["q"].float().reshape(b, hkv, (hq // hkv) * s["s"], d)
    scores = torch.matmul(q, kv[0].transpose(2, 3)).view(b, hq, s["s"], rows) * s["scale"]
    scores.masked_fill_(hidden[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hkv, (hq // hkv) * s["s"], rows), kv[1]).view(b, hq, s["s"], d)
    return torch.where(total == 0, torch.zeros_like(out), out / total).to(dtype)


_mynn = None


def _own(s):
    global _mynn
    if _mynn is None:
        _mynn = importlib.import_module("my-nn-engine_amd")
    if s["op"] == "append":
        q, k, v = _views(s)
        q = _mynn.rope_append_paged(q, k, v, s["cos"], s["sin"], s["pools"], s["table"], s["past_lens"], s["new_lens"])
        if s["bits"] == 16:
            return {"q": q, "k_pool": s["pools"][0], "v_pool": s["pools"][1]}
        k, v = _mynn.kv_rows_paged(s["pools"], s["table"], s["past_lens"], s["s"], s["new_lens"])
        return {"q": q, "k": k, "v": v}
    if s["workspace"] is None:  # (kept by the program from one call to the next)
        s["workspace"] = _mynn.attention_paged_int4_workspace(s["q"], s["pools"], s["table"])
    return _mynn.attention_paged_int4(s["q"], s["pools"], s["table"], s["scale"], s["past_lens"], s["new_lens"], workspace=s["workspace"])


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["op"] == "append" else _plain_attend(state)


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    past, new = _lens(case)
    if case["op"] == "append":
        tokens, padded = sum(new), case["b"] * case["s"]
        row = {16: 2 * d, 8: d + 2, 4: d // 2 + 3 * (d // max(case["group"], 1))}[case["bits"]]
        # (8 and 4 bits: the new rows are read again and returned as 16-bit values)
        moved = tokens * ((hq + 2 * hkv) * d * 2 + 4 * d + 2 * hkv * row) + padded * hq * d * 2
        if case["bits"] != 16:
            moved += tokens * 2 * hkv * row + padded * 2 * hkv * d * 2
        return {"bytes": moved, "flops": tokens * ((hq + hkv) * d * 3 + 2 * hkv * d * (0 if case["bits"] == 16 else 6))}
    row = d // 2 + 3 * (d // case["group"])
    seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))  # (query, key) pairs of a head
    return {"bytes": 2 * hkv * row * sum(p + n for p, n in zip(past, new)) + (sum(new) + case["b"] * case["s"]) * hq * d * 2, "flops": 4 * d * hq * seen}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_values(codes, scale, zero):
    x = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device="cuda")
    x[..., 0::2], x[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    group = x.shape[-1] // scale.shape[-1]
    return (x - zero.double().repeat_interleave(group, -1)) * scale.double().repeat_interleave(group, -1)


def _exact_quantized(x, case):
    """what rows [n, Hkv, D] in 64 bits stand for in the pools"""
    dtype = DTYPES[case["dtype"]]
    half_away = lambda y: torch.sign(y) * torch.floor(y.abs() + 0.5)
    if case["bits"] == 8:
        peak = x.abs().max(-1, keepdim=True).values
        code = half_away(torch.where(peak > 0, x / peak * 127.0, torch.zeros_like(x))).clamp(-128, 127)
        return code * (peak / 127.0).to(dtype).double()
    y = x.unflatten(-1, (-1, case["group"]))
    least, most = y.min(-1, keepdim=True).values.clamp(max=0), y.max(-1, keepdim=True).values.clamp(min=0)
    step = ((most - least) / 15.0).to(dtype).double()
    step[step == 0] = 1.0
    zero = half_away(-least / step).clamp(max=15)
    return (((half_away(y / step) + zero).clamp(0, 15) - zero) * step).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    dtype = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    past, new = _lens(case)
    if case["op"] == "append":
        x = s["qkv"].view(case["b"], case["s"], hq + 2 * hkv, d).double()
        out = torch.zeros((3, case["b"], hq, case["s"], d), dtype=torch.float64, device="cuda")
        pools = [p.double() for p in s["pools"][:2]] if case["bits"] == 16 else None
        for b in range(case["b"]):
            n, p = new[b], past[b]
            # the pair (j, j + D/2) as a complex number, turned
            c, t = s["cos"][p:p + n].double()[:, None], s["sin"][p:p + n].double()[:, None]
            y = x[b, :n]
            turned = y * c + torch.cat((-y[..., d // 2:], y[..., :d // 2]), -1) * t
            out[0, b, :, :n] = turned[:, :hq].transpose(0, 1)
            for side, rows in enumerate((turned[:, hq:hq + hkv], y[:, hq + hkv:])):
                if case["bits"] == 16:
                    for r in range(n):
                        pools[side][int(s["table"][b, (p + r) // case["page"]]), :, (p + r) % case["page"]] = rows[r]
                else:  # (it is the stored row, in 16 bits, that is quantised)
                    out[1 + side, b, :hkv, :n] = _exact_quantized(rows.to(dtype).double(), case).transpose(0, 1)
        if case["bits"] == 16:
            return {"q": out[0], "k_pool": pools[0], "v_pool": pools[1]}
        return {"q": out[0], "k": out[1, :, :hkv], "v": out[2, :, :hkv]}
    out = torch.zeros((case["b"], hq, case["s"], d), dtype=torch.float64, device="cuda")
    for b in range(case["b"]):
        rows, n = past[b] + new[b], new[b]
        pages = s["table"][b, :(rows + case["page"] - 1) // case["page"]].long()
        sides = []
        for side in (0, 1):
            x = _exact_values(*(s["pools"][m + side][pages] for m in (0, 2, 4)))  # [pages, Hkv, page rows, D]
            sides.append(x.transpose(0, 1).reshape(hkv, -1, d)[:, :rows])
        allowed = torch.ones((n, rows), dtype=torch.bool, device="cuda").tril(past[b])
        for h in range(hkv):
            q = s["q"][b, h * (hq // hkv):(h + 1) * (hq // hkv), :n].double()
            w = torch.mm(q.reshape(-1, d), sides[0][h].t().contiguous()).view(-1, n, rows) * s["scale"]
            w = torch.softmax(w.masked_fill(~allowed, -math.inf), -1)
            out[b, h * (hq // hkv):(h + 1) * (hq // hkv), :n] = torch.mm(w.view(-1, rows), sides[1][h]).view(-1, n, d)
    return out
