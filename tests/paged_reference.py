"""Paged caches of 16, 8 and 4 bits and attention over the last, in plain tensor operations: 32 bits where bits are compared, 64 bits
where tolerances are.  Everything runs on the device of its operands."""
import math

import torch


def round_away(x):
    t = x.trunc()
    return t + torch.where((x - t).abs() >= 0.5, x.sign(), torch.zeros_like(x))


def quantize4(x, group, dtype):
    """rows [.., D] of `dtype` -> (codes [.., D/2], scales [.., D/group], zero points)"""
    v = x.float().unflatten(-1, (-1, group))
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], torch.zeros_like(v), v)
    lo, hi = v.amin(-1).clamp_max(0.0), v.amax(-1).clamp_min(0.0)
    fifteen = torch.full_like(hi, 15.0)  # (a number in the place of either operand makes the division a product with a rounded reciprocal)
    s = (hi / fifteen - lo / fifteen).to(dtype).float()
    s = torch.where(s == 0, torch.ones_like(s), s)
    z = round_away(-lo / s).clamp_max(15.0)
    c = (round_away(v / s[..., None]) + z[..., None]).clamp(0.0, 15.0)
    s, z, c = torch.where(bad, torch.full_like(s, math.nan), s), torch.where(bad, torch.zeros_like(z), z), torch.where(bad[..., None], torch.zeros_like(c), c)
    c = c.flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), s.to(dtype), z.to(torch.uint8)


def values4(codes, scale, zero, kind=torch.float64):
    """what rows of 4 bits stand for, exactly in 64 bits"""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(kind)
    return ((c.unflatten(-1, (scale.shape[-1], -1)) - (zero & 15).to(kind)[..., None]) * scale.to(kind)[..., None]).flatten(-2)


def quantize8(x, dtype):
    """the rule of QuantizingKVCacheUpdate"""
    v = x.float()
    peak = v.abs().amax(-1, keepdim=True)
    y = v * torch.where(peak == 0, torch.zeros_like(peak), torch.full_like(peak, 127.0) / peak)
    return (y + torch.where(y >= 0, 0.5, -0.5)).trunc().clamp(-128, 127).to(torch.int8), (peak * torch.tensor(1.0 / 127.0, dtype=torch.float32)).to(dtype)[..., 0]


def rotate(x, cos, sin, kind=torch.float32):
    """[B,H,S,D] by table rows [B,S,D]"""
    h = x.shape[-1] // 2
    x, cos, sin = x.to(kind), cos.to(kind)[:, None], sin.to(kind)[:, None]
    return torch.cat((x[..., :h] * cos[..., :h] - x[..., h:] * sin[..., :h], x[..., h:] * cos[..., h:] + x[..., :h] * sin[..., h:]), -1)


def make_pools(n_pages, heads, rows, dim, dtype, bits, group, device, seed=0):
    """pools whose every byte is something: what is not written has to stay"""
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def any_bits(shape, t):
        size = torch.empty((), dtype=t).element_size()
        return torch.randint(0, 256, shape + (size,), generator=g, device=device, dtype=torch.uint8).view(t)[..., 0]

    lead = (n_pages, heads, rows)
    if bits == 16:
        return tuple(any_bits(lead + (dim,), dtype) for _ in range(2))
    if bits == 8:
        return tuple(any_bits(lead + (dim,), torch.int8) for _ in range(2)) + tuple(any_bits(lead, dtype) for _ in range(2))
    return (tuple(any_bits(lead + (dim // 2,), torch.uint8) for _ in range(2)) + tuple(any_bits(lead + (dim // group,), dtype) for _ in range(2)) +
            tuple(any_bits(lead + (dim // group,), torch.uint8) for _ in range(2)))


def append(q, k, v, cos, sin, pools, table, past, new, positions=None):
    """(the rotated q, the pools behind the append), bit for bit what the operator documents"""
    pools = [p.clone() for p in pools]
    B, S, D = k.shape[0], k.shape[2], k.shape[3]
    P, n_pages = pools[0].shape[2], pools[0].shape[0]
    dtype = k.dtype
    out = torch.zeros_like(q, memory_format=torch.contiguous_format) if q is not None else None
    for b in range(B):
        n = S if new is None else min(max(int(new[b]), 0), S)
        for i in range(n):
            row = int(past[b]) + i
            pos = row if positions is None else int(positions[b, i])
            if not (0 <= row < table.shape[1] * P and 0 <= pos < cos.shape[0]):
                continue
            c, s = cos[pos][None, None], sin[pos][None, None]
            if q is not None:
                out[b, :, i] = rotate(q[b:b + 1, :, i:i + 1], c, s).to(dtype)[0, :, 0]
            page = int(table[b, row // P])
            if not 0 <= page < n_pages:
                continue
            sides = (rotate(k[b:b + 1, :, i:i + 1], c, s).to(dtype)[0, :, 0], v[b, :, i])
            for side, x in enumerate(sides):
                if len(pools) == 2:
                    pools[side][page, :, row % P] = x
                elif len(pools) == 4:
                    pools[side][page, :, row % P], pools[2 + side][page, :, row % P] = quantize8(x, dtype)
                else:
                    group = D // pools[2].shape[-1]
                    for n4, t in enumerate(quantize4(x, group, dtype)):
                        pools[2 * n4 + side][page, :, row % P] = t
    return out, pools


def rows_of(pools, side, table, b, first, n):
    """(values [Hkv, n, D] in 64 bits, which of the rows are there)"""
    P, n_pages = pools[0].shape[2], pools[0].shape[0]
    r = torch.arange(first, first + n, device=table.device)
    inside = (r >= 0) & (r < table.shape[1] * P)
    page = table[b][torch.where(inside, r // P, torch.zeros_like(r))].long()
    there = inside & (page >= 0) & (page < n_pages)
    page, at = torch.where(there, page, torch.zeros_like(page)), torch.where(there, r % P, torch.zeros_like(r))
    if len(pools) == 2:
        x = pools[side][page, :, at].double()
    elif len(pools) == 4:
        x = pools[side][page, :, at].double() * pools[2 + side][page, :, at].double()[..., None]
    else:
        x = values4(*(pools[m + side][page, :, at] for m in (0, 2, 4)))
    return x.transpose(0, 1), there


def attention(q, pools, table, scale, past, new, causal, weight_error):
    """softmax(q k scale) v in 64 bits, and how far the operator's result may be from it before it is rounded to its type.

    The operator's errors: a score is a sum of D products of exact operands in 32 bits, scaled in a few more steps -- off by at most
    (D + 8) half steps of 2^-24 of the sum of the products' magnitudes --, its exponential has an argument rounded at the size of the
    largest score and is itself good to 2^-22; a weight enters the second product off by weight_error (relative), the sums over n keys
    have n half steps at the most, the join of ranges a few more.  All of these scale a key's weight, so the result is off by at most
    their sum times sum(p |v|) / sum(p), twice, as numerator and denominator have them both.
    What is absolute: a weight times its value's scale is an fp16 number in units that make the largest of them 2^13 or more (so off by
    2^-25 where it is small: 2^-38 of the largest, times a code of at most 15), or, where the scales next to the largest weight are
    below 2^-86, units of 2^-100 of that weight (2^-125); a weight below the smallest 32-bit number, in the same units, is lost
    (2^-140 times the largest scale, times the value).  More than 16 rows a kv head: their reference may lag 2^4 behind the largest, which
    then is 2^9 or more in the units of fp16 and all of these are 16 times as large."""
    B, Hq, S, D = q.shape
    Hkv = pools[0].shape[1]
    G, P = Hq // Hkv, pools[0].shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    slack = torch.zeros_like(out)
    half = 2.0 ** -24
    lag = 1.0 if G * S <= 16 else 16.0
    for b in range(B):
        n = S if new is None else min(max(int(new[b]), 0), S)
        length = min(max(int(past[b]) + n, 0), table.shape[1] * pools[0].shape[2]) if n else 0
        if not length:
            continue
        (k, there), (v, _) = rows_of(pools, 0, table, b, 0, length), rows_of(pools, 1, table, b, 0, length)
        at = torch.arange(length, device=q.device)
        for i in range(n):
            seen = there & (at < (min(int(past[b]) + i + 1, length) if causal else length))
            if not bool(seen.any()):
                continue
            for h in range(Hkv):
                x = q[b, h * G:(h + 1) * G, i].double()
                kk, vv = k[h][seen], v[h][seen]
                s = torch.mm(x, kk.t().contiguous()) * scale
                size = (torch.mm(x.abs(), kk.abs().t().contiguous()) * abs(scale)).amax(-1, keepdim=True)
                p = torch.softmax(s, -1)
                vs = pools[3][table[b][at // P].long().clamp(0, pools[3].shape[0] - 1), h, at % P].double().amax(-1)[seen] if len(pools) == 6 else vv.abs().amax(-1)
                small = lag * kk.shape[0] * (15 * 2.0 ** -38 * (p * vs).amax(-1, keepdim=True) + 2.0 ** -120 + 2.0 ** -138 * vs.max() * vv.abs().max())
                out[b, h * G:(h + 1) * G, i] = torch.mm(p, vv)
                weight = (D + 8) * half * size + 4 * half * s.abs().amax(-1, keepdim=True) + 2.0 ** -22 + weight_error + (kk.shape[0] + 64) * half
                slack[b, h * G:(h + 1) * G, i] = 2 * weight * torch.mm(p, vv.abs()) + small
    return out, slack


def assert_close(got, want, slack):
    """rounded once to its type: half a step of what lies inside the slack"""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # half steps of subnormal results
    got = got.double()
    assert torch.isfinite(got).all()
    off = (got - want).abs() - (want.abs() * half + slack * (1 + half) + tiny)
    assert float(off.max()) <= 0, "off by %g more than the bound at %s of %s" % (float(off.max()), (off == off.max()).nonzero()[0].tolist(), tuple(off.shape))
