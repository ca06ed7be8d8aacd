"""4-bit matrices and the operators on them in 64 bits, for the tests."""
import torch


def matrix(N, K, group, dtype, zero, gen, device="cuda"):
    """(wq, scale, zero points or None): any code, scales around 1 / sqrt(K)"""
    wq = torch.randint(0, 256, (N, K // 2), generator=gen, dtype=torch.uint8, device=device)
    scale = ((torch.rand((N, K // group), generator=gen, device=device) + 0.5) / K**0.5).to(dtype)
    z = torch.randint(0, 16, (N, K // group), generator=gen, dtype=torch.uint8, device=device) if zero else None
    return wq, scale, z


def codes(wq):
    return torch.stack((wq & 15, wq >> 4), -1).flatten(1)


def differences(wq, scale, zero):
    """code - zero [N, K], and the scale of every column [N, K], in 64 bits"""
    group = 2 * wq.shape[1] // scale.shape[1]
    z = torch.full(scale.shape, 8, dtype=torch.uint8, device=wq.device) if zero is None else zero & 15
    return codes(wq).double() - z.double().repeat_interleave(group, 1), scale.double().repeat_interleave(group, 1)


def product(act, wq, scale, zero, row_scale=None):
    """(the product in 64 bits, how far a 32-bit sum may be off it).

    The bound: a sum of terms t_k taken in any order is off by at most (number of additions a term goes through) * u * sum |t_k|.  A
    term is multiplied (1), goes through at most 128 additions inside a group's sum, one for the zero point, two for the scale, and
    one for each of the K / 32 partial sums and of up to 32 waves behind it; u = 2^-23, a whole unit in the last place, because a matrix
    instruction need not round to nearest.  The terms may be act * code and act * zero apart: |code| + |zero| for |code - zero|."""
    d, s = differences(wq, scale, zero)
    a = act.double()
    z = 8 if zero is None else 15
    want = a @ (d * s).t().contiguous()
    size = a.abs() @ ((d.abs() + 2 * z) * s.abs()).t().contiguous()
    bound = size * (128 + 4 + act.shape[1] / 32 + 32) * 2.0**-23
    if row_scale is not None:
        r = row_scale.double()[:, None]
        want, bound = want * r, bound * r.abs()
    return want, bound


def assert_close(out, want, bound):
    """every value within the 32-bit bound and half a step of its type; the whole within half a step (of the type's normal numbers)"""
    eps = torch.finfo(out.dtype).eps / 2
    tiny = torch.finfo(out.dtype).smallest_normal * eps  # (half a step below the normal numbers)
    got = out.double()
    assert got.shape == want.shape
    off = (got - want).abs()
    # (the rounded value is the 32-bit sum's: half a step of it, not of the exact one)
    most = bound + eps * (want.abs() + bound) + tiny
    assert bool((off <= most).all()), float((off / most).max())
    assert float(off.norm()) <= eps * float(want.norm()) + tiny * want.numel() ** 0.5 + 1e-300, float(off.norm() / want.norm()) / eps
