"""The weights' gradient of norm_rope at the sizes where its sums change: heads per workgroup, and launches beyond the last-level cache.

Bounds as in test_norm_rope_gpu.py: a thread adds up 8 heads at most, a workgroup 64 tokens, the small kernel its rows of partial sums in 64 chains
(at most 64 of each here) and these 64: below 256 roundings, relative to the sum of the sizes."""
import pytest
import torch

import paged_model as m
from test_norm_rope_gpu import _check, _make, _run

DEV = "cuda:0"


# a workgroup takes more heads while 512 workgroups are left: 16 heads of 128 in blocks of 32 tokens are 1008 and 1024 workgroups, then 2048 and 4096;
# last groups that are not full
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,D", [(1, 16, 3, 2016, 128), (1, 16, 3, 2048, 128), (2, 16, 5, 2048, 128), (1, 17, 9, 4100, 128), (1, 20, 9, 8200, 128),
                                        (1, 13, 2, 2100, 256), (3, 30, 7, 1700, 64)])
@pytest.mark.parametrize("weight", ["shared", "heads"])
def test_heads_per_workgroup(qfa, B, H, Hk, N, D, weight):
    _run(qfa, B, H, Hk, N, D, D, weight=weight, positions="starts", seed=N)


@pytest.mark.gpu
@pytest.mark.parametrize("weight", ["shared", "heads"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_weights_of_a_call_beyond_the_last_level_cache(qfa, weight, interleaved):
    B, H, N, D, eps = 4, 32, 2800, 128, 1e-6
    g = torch.Generator(device=DEV).manual_seed(2)
    x, dy = (torch.randn(B, H, N, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    w = torch.rand(*((D,) if weight == "shared" else (H, D)), device=DEV, generator=g) + 0.5
    cos, sin = (t.to(DEV) for t in m.table(N, D))
    leaves = [t.clone().requires_grad_(True) for t in (x, x, w, w)]
    out = qfa.norm_rope_pair(*leaves, cos, sin, eps=eps, interleaved=interleaved)
    _, dx, dw, dw2 = torch.autograd.grad(out, leaves, (dy, dy))
    assert torch.equal(dw, dw2)
    want = torch.zeros(H, D, dtype=torch.float64, device=DEV)
    size = want.clone()
    for b in range(B):
        g64, g_size = m.turn(dy[b:b + 1].double(), cos[None], sin[None], interleaved, back=True)
        xr = x[b:b + 1].double()
        xr = xr / (xr.square().mean(-1, keepdim=True) + eps).sqrt()
        want += (g64 * xr).sum((0, 2))
        size += (g_size * xr.abs()).sum((0, 2))
    if weight == "shared":
        want, size = want.sum(0), size.sum(0)
    _check("dw", dw, want.cpu(), size.cpu(), 256)


@pytest.mark.gpu
@pytest.mark.parametrize("weight", ["shared", "heads"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_by_differences(qfa, weight, interleaved):
    """As in test_norm_rope_gpu.py, where the bound is added twice: central differences along directions v with |v|^2 = the number of elements, at
    h = 1e-2, of rows of rms one.  Truncation: h^2/6 = 1.7e-5 times the third derivative, at most 1e-3 of the gradient's norm where that is
    below 60 times it.  Rounding: 2^-25 of each of at most 1536 terms of order one, as a root of a sum of squares 1.2e-6, over 2h 6e-5, far below
    1e-3 of a norm of order 10.  Bound 3e-3 of the gradient's norm."""
    q, k, w, cos, sin, pos, dy = _make(1, 2, 1, 4, 128, 128, torch.float32, weight, torch.float32, "each", 9)
    q, k = q / q.square().mean(-1, keepdim=True).sqrt(), k / k.square().mean(-1, keepdim=True).sqrt()
    args = [t.to(DEV) for t in (q, k, *w)]
    fixed = [t.to(DEV) for t in (cos, sin, pos)]
    run = lambda a: qfa.norm_rope_pair(*a, *fixed, interleaved=interleaved)   # noqa: E731
    loss = lambda a: sum((y.double() * d.to(DEV).double()).sum() for y, d in zip(run(a), dy))   # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(run(leaves), leaves, [d.to(DEV) for d in dy])
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        for _ in range(4):
            v = torch.randn(args[i].shape, generator=g).to(DEV)
            v /= v.norm() / v.numel() ** 0.5
            with torch.no_grad():
                up, down = ([a + s * v if j == i else a for j, a in enumerate(args)] for s in (1e-2, -1e-2))
                slope = (loss(up) - loss(down)) / 2e-2
            assert abs(slope - (grad.double() * v).sum()) <= 3e-3 * grad.double().norm()
