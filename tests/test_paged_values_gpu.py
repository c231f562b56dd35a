"""Values of any size on a paged cache, alike for all keys or not, in blocks of 16, 64 and 128 rows and in a pass over a prefix: the scales carry the
values' magnitude, and enter the probabilities before these are rounded to binary16.

Bound: the output rounded once; probability times scale in binary16 (2^-11, twice for the fp32 exponentials and the joins), a rounding of the largest
score in the exponent, twice; the codes' offset of at most 1152 + 255 in fp32 sums, 32 roundings inside a tile and one per tile of 32
keys, weighted with p_j scale_j; and binary16's smallest step, 2^-24, of one of the largest p_j scale_j of the row, once per key, times
|code - zero point| <= 255."""
import pytest
import torch

import paged_model as m
from test_paged_attn_gpu import _with_prefix_pass

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 30, 130])
@pytest.mark.parametrize("prefix", [0, 700])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [1e-20, 1e20, "ramp", "masked out", "rising scores", "scales of zero"])
def test_size_of_the_values(qfa, N, prefix, D, size):
    B, H, L, page, sm = 2, 2, 1500, 64, m.sm_of(D)
    g = torch.Generator().manual_seed(D + N)
    q, k, v = (torch.randn(B, h, n, D, generator=g) for h, n in ((H, N), (1, L), (1, L)))
    ramp, scale_dtype = torch.arange(L).view(1, 1, -1, 1) / L, torch.float32
    if prefix:   # the same rows for both sequences
        k[1, :, :prefix], v[1, :, :prefix] = k[0, :, :prefix], v[0, :, :prefix]
    if size == "ramp":
        v = v * 2.0 ** (40 * ramp - 20)
    elif size == "masked out":     # scores near -40 at the keys with large values, in the first tile and later
        q = q.abs() + 0.5
        far = (ramp < 0.01) | ((ramp > 0.5) & (ramp < 0.52))
        k, v = torch.where(far, -40 * sm * torch.ones_like(k), k * 0.1), torch.where(far, v * 1e5, v)
    elif size == "rising scores":
        q = q.abs() + 0.5
        k, v = k * 0.1 + 40 * ramp, v * 2.0 ** (-60 * ramp)
    elif size == "scales of zero":   # fp16 has none for so small a range: the values stand for zero
        v, scale_dtype = v * 1e-9, torch.float16
    else:
        v = v * size
    q = q.bfloat16()
    table, pages = m.shared_pages(B, -(-L // page), prefix // page, N)
    cache = m.garbage_cache(pages, 1, page, D, scale_dtype, 1)
    hat, v_scale = [], None
    for side, x in ((0, k), (3, v)):
        c, s, z = m.quantized(x)
        s = s.to(scale_dtype)
        for b in range(B):
            m.place(cache, table, b, 0, c[b], s[b], z[b], side)
        hat.append(m.values(c, s, z))
        v_scale = s.double()
    starts = torch.full((B,), L - N, dtype=torch.int32)
    dev = lambda t: t.to(DEV)   # noqa: E731
    call = (dev(q), [dev(t) for t in cache], dev(table), dev(starts))
    o = (_with_prefix_pass(*call, None, True, sm, prefix) if prefix else qfa.quant_flash_attn_paged(*call, sm_scale=sm)).cpu()
    kh, vh = hat
    s = (m.values(*m.quantized(q.float())) @ kh.transpose(-1, -2)) * sm
    s = s.masked_fill(torch.arange(L) > torch.arange(N).view(-1, 1) + L - N, -float("inf"))
    p = torch.softmax(s, -1)
    want, size_of, ps = p @ vh, p @ vh.abs(), p * v_scale.transpose(-1, -2)
    top = float(s[s > -float("inf")].abs().max())
    bound = (m.HALF[torch.bfloat16] * want.abs() + (2.0 ** -10 + 2.0 ** -22 * top) * size_of + (32 + L / 32) * m.U32 * (1152 + 255) * ps.sum(-1, keepdim=True)
             + L * 255 * 2.0 ** -25 * ps.max(-1, keepdim=True).values + m.TINY[torch.bfloat16])
    excess = (o.double() - want).abs() - bound
    assert torch.isfinite(o).all() and excess.max() <= 0, f"over the bound by {excess.max().item():.3e} of {want.abs().max().item():.3e}"
    if size == "scales of zero":
        assert not o.any()
