"""Bounds of a page's keys in plain torch: rows of one sign keep their span (not collected by pytest)."""
import torch

HALF_STEP = 0.501   # of a code, and the fp32 roundings of scale, quotients and sums: at most 1020 steps times 2^-23 each, three of them


def _away(x):
    t = x.trunc()
    return t + ((x - t).abs() >= 0.5) * x.sign()


def _over(a, b):
    """The quotient rounded to 32 bits (that in 64 bits has more than twice as many)."""
    return (a.double() / b.double()).float()


def bound_rows(x):
    """Codes, scale and zero point of rows [..., D] of fp32 values."""
    x = x.float()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    mn = torch.where(low > 0, torch.minimum(low, 0.75 * high), low)
    mx = torch.where(high < 0, torch.maximum(high, 0.75 * low), high)
    scale = _over(mx - mn, torch.full_like(mn, 255))
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    zero = _away(-128 - _over(mn, scale)).clamp(-1024, 1023)
    return _away(_over(x, scale) + zero).clamp(-128, 127), scale, zero


def extremes(keys):
    """The low and the high row of keys [..., rows, D], as fp32 values: [..., 2, D]."""
    k = keys.float()
    return torch.stack([k.amin(-2), k.amax(-2)], -2)


def values(codes, scale, zero):
    return (codes.double() - zero.double()) * scale.double()
