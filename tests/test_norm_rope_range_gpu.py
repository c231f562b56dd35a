"""Norms of rows of any size that the types hold: squares that leave fp32's range, and r^3 in the gradient.

The bounds are those of test_norm_rope_gpu.py; the scaling by a power of two that such rows need is exact."""
import pytest
import torch

import paged_model as m
from test_norm_rope_gpu import _check

DEV = "cuda:0"
SIZES = [1.0, 1e13, 1e15, 3e37, 1e-14, 1e-36, 2e19, 5e-20, 1e-3, 1e25]   # of a token's row; one after the other, so that lanes of a wave differ


def _rows(H, N, D, dtype, g):
    x = torch.randn(2, H, N, D, generator=g).double()
    return (x * torch.tensor([SIZES[n % len(SIZES)] for n in range(N)], dtype=torch.float64)[:, None]).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("per_head,interleaved", [(False, False), (True, True)])
def test_rows_of_any_size(qfa, D, dtype, eps, per_head, interleaved):
    g = torch.Generator().manual_seed(D)
    H, Hk, N = 3, 2, 27
    x = [_rows(h, N, D, dtype, g) for h in (H, Hk)]
    dy = [torch.randn(2, h, N, D, generator=g).to(dtype) for h in (H, Hk)]
    w = [(1 + 0.3 * torch.randn(*((h, D) if per_head else (D,)), generator=g)).to(dtype) for h in (H, Hk)]
    cos, sin = m.table(N, D // 2)
    leaves = [t.to(DEV).requires_grad_(True) for t in (*x, *w)]
    out = qfa.norm_rope_pair(*leaves, cos.to(DEV), sin.to(DEV), eps=eps, interleaved=interleaved)
    grads = torch.autograd.grad(out, leaves, [t.to(DEV) for t in dy])
    for i, name in enumerate("qk"):
        want, size = m.norm_rope(x[i], w[i], cos, sin, None, eps, interleaved)
        _check(name, out[i].detach(), want, size, 32)
        dx, dx_size, dw, dw_size = m.norm_rope_grad(x[i], dy[i], w[i], cos, sin, None, eps, interleaved)
        for n in range(N):   # (each row by itself: a NaN counts as over its bound)
            assert torch.isfinite(grads[i][:, :, n]).all(), f"d{name}: rows of {SIZES[n % len(SIZES)]}"
            _check(f"d{name}, rows of {SIZES[n % len(SIZES)]}", grads[i][:, :, n], dx[:, :, n], dx_size[:, :, n], 64)
        _check(f"dw of {name}", grads[2 + i], dw, dw_size, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_appended_keys_of_any_size(qfa, dtype):
    """The keys' values after norm and rotation, within a code and the scale's rounding (the norm may round a code's way or the other)."""
    g = torch.Generator().manual_seed(1)
    H, N, D, page = 2, 30, 128, 16
    k, v = _rows(H, N, D, dtype, g), torch.randn(2, H, N, D, generator=g).to(dtype)
    w, (cos, sin) = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype), m.table(N, D)
    table, pages = m.shared_pages(2, 2, 0, 1)
    cache = qfa.make_paged_cache(pages, H, page, D, scale_dtype=torch.float32, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    qfa.paged_cache_append(cache, k.to(DEV), v.to(DEV), table.to(DEV), zero, k_weight=w.to(DEV), cos=cos.to(DEV), sin=sin.to(DEV), eps=0.0)
    got, _ = qfa.paged_cache_read(cache, table.to(DEV), zero, N, dtype=torch.float32)
    want, _ = m.norm_rope(k, w, cos, sin, None, 0.0, False)
    step = (want.amax(-1, keepdim=True) - want.amin(-1, keepdim=True)) / 255
    assert ((got.cpu().double() - want).abs() <= 1.2 * step).all()


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_row_that_is_not_finite_leaves_the_others(qfa, value):
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(1, 2, 9, 128, generator=g).to(DEV) for _ in range(2))
    w = torch.ones(128, device=DEV)

    def run(x):
        x = x.clone().requires_grad_(True)
        y = qfa.norm_rope(x, w, None, None)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]
    clean = run(x)
    x[0, 1, 4, 17] = value
    keep = torch.ones(1, 2, 9, dtype=torch.bool, device=DEV)
    keep[0, 1, 4] = False
    for a, b in zip(run(x), clean):
        assert torch.isnan(a[0, 1, 4, 17]) and torch.equal(a[keep], b[keep])
