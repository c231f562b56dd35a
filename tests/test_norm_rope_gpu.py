"""norm_rope and norm_rope_pair against their formulas in 64 bits, forward and backward.

Bounds.  Everything is fp32 with one rounding at the end (half a unit of the result's type).  In fp32: the mean of squares adds 16
products in a lane and up to 4 sums over lanes, the root, the division and the products by it and the weight one rounding each -- below 32
half units, relative to the two terms that the rotation adds (`size` of paged_model).  dx: the mean of g w x likewise, two terms of
up to that: 64, relative to the sizes of both terms.  dw: at most 8 heads, 64 tokens, the partial sums in 64 chains and these 64:
256 roundings of sums of the sizes for the at most 7000 partial sums here."""
import pytest
import torch

import paged_model as m

DEV = "cuda:0"
EPS = 1e-6


def _make(B, H, Hk, N, D, R, dtype, weight, wdtype, positions, seed, layout="bhnd", T=None):
    g = torch.Generator().manual_seed(seed)
    T = T or 2 * N + 50

    def rows(h):
        x = (torch.randn(B, h, N, D, generator=g) * torch.randn(1, h, 1, D, generator=g).exp()).to(dtype)
        return x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) if layout == "bnhd" else x
    q, k = rows(H), rows(Hk)
    w = [None if weight == "none" else (1 + 0.3 * torch.randn(*((D,) if weight == "shared" else (h, D)), generator=g)).to(wdtype) for h in (H, Hk)]
    cos, sin = m.table(T, R) if R else (None, None)
    pos = {"none": None, "starts": torch.randint(0, T - N + 1, (B,), generator=g).int(), "each": torch.randint(0, T, (B, N), generator=g).int()}[positions]
    dy = [torch.randn(B, h, N, D, generator=g).to(dtype) for h in (H, Hk)]
    return q, k, w, cos, sin, pos, dy


def _check(name, got, want, size, half_units):
    bound = m.HALF[got.dtype] * want.abs() + half_units * m.U32 * size + m.TINY[got.dtype]
    excess = (got.cpu().double() - want).abs() - bound
    assert excess.max() <= 0, f"{name}: over the bound by {excess.max().item():.3e} at {want.flatten()[excess.argmax()].item():.3e}"


def _run(qfa, B, H, Hk, N, D, R, dtype=torch.bfloat16, weight="shared", wdtype=None, positions="none", interleaved=False, seed=0, layout="bhnd"):
    q, k, w, cos, sin, pos, dy = _make(B, H, Hk, N, D, R, dtype, weight, wdtype or dtype, positions, seed, layout)
    dev = lambda t: None if t is None else t.to(DEV)   # noqa: E731  (.to keeps the strides of a permuted tensor)
    leaves = [dev(t).requires_grad_(True) if t is not None else None for t in (q, k, *w)]
    out = qfa.norm_rope_pair(*leaves, dev(cos), dev(sin), dev(pos), eps=EPS, interleaved=interleaved)
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], [dev(t) for t in dy])
    gq, gk, *gw = grads
    for i, (name, x, y, gx) in enumerate((("q", q, out[0], gq), ("k", k, out[1], gk))):
        assert y.dtype == dtype and y.shape == x.shape and gx.shape == x.shape
        want, size = m.norm_rope(x, w[i], cos, sin, pos, EPS, interleaved)
        _check(name, y.detach(), want, size, 32)
        dx, dx_size, dw, dw_size = m.norm_rope_grad(x, dy[i], w[i], cos, sin, pos, EPS, interleaved)
        _check("d" + name, gx, dx, dx_size, 64)
        if dw is not None:
            assert gw[i].shape == w[i].shape and gw[i].dtype == w[i].dtype
            _check("dw of " + name, gw[i], dw, dw_size, 256)
    return out, grads


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_head_dims(qfa, D, dtype, interleaved):
    _run(qfa, 2, 3, 2, 37, D, D, dtype, interleaved=interleaved, seed=D)


@pytest.mark.gpu
@pytest.mark.parametrize("D,R", [(64, 16), (64, 48), (128, 32), (128, 112), (256, 64), (256, 240), (128, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_part_of_the_row_is_rotated(qfa, D, R, interleaved):
    _run(qfa, 1, 2, 1, 70, D, R, interleaved=interleaved, seed=R)


@pytest.mark.gpu
@pytest.mark.parametrize("weight", ["none", "shared", "heads"])
@pytest.mark.parametrize("wdtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("positions", ["none", "starts", "each"])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_weights_positions_layouts(qfa, weight, wdtype, positions, layout):
    _run(qfa, 3, 5, 2, 67, 128, 128, torch.float16, weight, wdtype, positions, seed=7, layout=layout)


# one token; tokens that fill no workgroup; several heads per workgroup (more than 2048 workgroups), a last group that is not full
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,D", [(1, 1, 1, 1, 128), (7, 32, 8, 1, 64), (1, 1, 1, 4097, 256), (2, 37, 3, 2100, 128), (1, 133, 70, 1200, 64)])
@pytest.mark.parametrize("weight", ["shared", "heads"])
def test_sizes(qfa, B, H, Hk, N, D, weight):
    _run(qfa, B, H, Hk, N, D, D, weight=weight, positions="starts", seed=N)


@pytest.mark.gpu
def test_one_tensor_is_the_pair(qfa):
    q, k, w, cos, sin, pos, dy = (x for x in _make(2, 4, 4, 50, 128, 128, torch.bfloat16, "heads", torch.bfloat16, "each", 3))
    dev = lambda t: t.to(DEV)   # noqa: E731
    a, b = qfa.norm_rope_pair(dev(q), dev(k), dev(w[0]), dev(w[1]), dev(cos), dev(sin), dev(pos))
    assert torch.equal(a, qfa.norm_rope(dev(q), dev(w[0]), dev(cos), dev(sin), dev(pos)))
    assert torch.equal(b, qfa.norm_rope(dev(k), dev(w[1]), dev(cos), dev(sin), dev(pos)))


@pytest.mark.gpu
def test_a_row_that_is_not_finite_or_has_no_angle_stays_alone(qfa):
    q, k, w, cos, sin, pos, dy = _make(1, 2, 1, 40, 64, 32, torch.bfloat16, "shared", torch.bfloat16, "each", 5)
    clean = qfa.norm_rope(q.to(DEV), w[0].to(DEV), cos.to(DEV), sin.to(DEV), pos.to(DEV))
    q[0, 1, 3, 5], q[0, 0, 9, 0] = float("nan"), float("inf")
    pos[0, 20], pos[0, 21] = -1, cos.shape[0]
    y = qfa.norm_rope(q.to(DEV), w[0].to(DEV), cos.to(DEV), sin.to(DEV), pos.to(DEV))
    assert torch.isnan(y[0, 1, 3]).all() and torch.isnan(y[0, 0, 9, 0]) and torch.isnan(y[0, :, 20:22, :32]).all()
    assert torch.equal(y[0, :, 20:22, 32:], clean[0, :, 20:22, 32:])
    keep = torch.ones(1, 2, 40, dtype=torch.bool)
    keep[0, 1, 3] = keep[0, 0, 9] = keep[0, 0, 20] = keep[0, 0, 21] = keep[0, 1, 20] = keep[0, 1, 21] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.gpu
def test_gradient_by_differences(qfa):
    """fp32, the loss summed in 64 bits: central differences along random directions.  Truncation h^2/6 times the third derivative
    (of order the gradient for rows of order one): below 1e-4 of the derivative's size at h = 1e-2; the outputs' fp32 rounding, 2^-24 of
    each of the 1536 terms of order one over 2h: 5e-6 of its root-sum-square times 100: 4e-4 at most.  Bound 3e-3 of the gradient's norm."""
    q, k, w, cos, sin, pos, dy = _make(1, 2, 1, 4, 128, 128, torch.float32, "shared", torch.float32, "each", 9)
    q, k = q / q.square().mean(-1, keepdim=True).sqrt(), k / k.square().mean(-1, keepdim=True).sqrt()
    args = [t.to(DEV) for t in (q, k, *w)]
    fixed = [t.to(DEV) for t in (cos, sin, pos)]
    loss = lambda a: sum((y.double() * d.to(DEV).double()).sum() for y, d in zip(qfa.norm_rope_pair(*a, *fixed), dy))   # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in args]
    out = qfa.norm_rope_pair(*leaves, *fixed)
    grads = torch.autograd.grad(out, leaves, [d.to(DEV) for d in dy])
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        v = torch.randn(args[i].shape, generator=g).to(DEV)
        v /= v.norm() / v.numel() ** 0.5
        with torch.no_grad():
            up, down = ([a + s * v if j == i else a for j, a in enumerate(args)] for s in (1e-2, -1e-2))
            slope = (loss(up) - loss(down)) / 2e-2
        assert abs(slope - (grad.double() * v).sum()) <= 3e-3 * grad.double().norm() * v.norm() / v.numel() ** 0.5 + 3e-3 * grad.double().norm()


@pytest.mark.gpu
def test_partial_gradients_and_fixed_bits(qfa):
    args = _make(2, 8, 2, 300, 128, 64, torch.bfloat16, "shared", torch.float32, "none", 11)
    q, k, w, cos, sin, pos, dy = args
    dev = lambda t: t.to(DEV)   # noqa: E731

    def grads(needs):
        leaves = [dev(t).requires_grad_(bool(n)) for t, n in zip((q, k, *w), needs)]
        out = qfa.norm_rope_pair(*leaves, dev(cos), dev(sin))
        return torch.autograd.grad(out, [t for t in leaves if t.requires_grad], [dev(t) for t in dy])
    every, again = grads((1, 1, 1, 1)), grads((1, 1, 1, 1))
    assert all(torch.equal(a, b) for a, b in zip(every, again))
    assert torch.equal(grads((0, 0, 0, 1))[0], every[3]) and torch.equal(grads((1, 0, 0, 0))[0], every[0])
    # only one output reaches the loss
    leaves = [dev(t).requires_grad_(True) for t in (q, k, *w)]
    out = qfa.norm_rope_pair(*leaves, dev(cos), dev(sin))
    g = torch.autograd.grad(out[0], leaves, dev(dy[0]), allow_unused=True)
    assert torch.equal(g[0], every[0]) and torch.equal(g[2], every[2])
    assert all(t is None or not t.any() for t in (g[1], g[3]))
    # a gradient that is broadcast
    leaf = dev(q).requires_grad_(True)
    y = qfa.norm_rope(leaf, dev(w[0]), dev(cos), dev(sin))
    ones = torch.ones_like(y)
    a, = torch.autograd.grad(y, leaf, ones, retain_graph=True)
    b, = torch.autograd.grad(y.sum(), leaf)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_one_large_call_is_many_small_ones(qfa, interleaved):
    """What outgrows the last-level cache is stored with other hints."""
    B, H, N, D = 4, 32, 2800, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, dq, dk = (torch.randn(B, H, N, D, device=DEV, generator=g).bfloat16() for _ in range(4))
    w = torch.rand(D, device=DEV, generator=g) + 0.5
    cos, sin = (t.to(DEV) for t in m.table(N, D))

    def step(at):
        x = [t[at].detach().requires_grad_(True) for t in (q, k)]
        y = qfa.norm_rope_pair(*x, w, w, cos, sin, interleaved=interleaved)
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, x, (dq[at], dk[at]))
    whole = step(slice(0, B))
    for b in range(B):
        assert all(torch.equal(a[b:b + 1], p) for a, p in zip(whole, step(slice(b, b + 1))))


@pytest.mark.gpu
def test_stream_and_graph(qfa):
    q, k, w, cos, sin, pos, dy = (x for x in _make(2, 4, 2, 129, 128, 128, torch.bfloat16, "shared", torch.bfloat16, "starts", 13))
    t = [x.to(DEV) for x in (q, k, *w, cos, sin, pos)]
    d = [x.to(DEV) for x in dy]
    leaves = [x.requires_grad_(True) for x in t[:4]]

    def step():
        out = qfa.norm_rope_pair(*leaves, *t[4:])
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, leaves, d)
    want = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for x in got:
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        eager = step()   # the program's own work in between
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {i}"
        assert all(torch.equal(a, b) for a, b in zip(eager, want))


@pytest.mark.gpu
def test_traced(qfa):
    q, k, w, cos, sin, pos, dy = (x for x in _make(1, 2, 2, 30, 64, 64, torch.float16, "shared", torch.float16, "none", 17))
    a, b, c, s, v0, v1 = (x.to(DEV) for x in (q, k, cos, sin, *w))
    f = lambda a, b: qfa.norm_rope_pair(a, b, v0, v1, c, s)   # noqa: E731
    traced = torch.jit.trace(f, (torch.zeros_like(a), torch.zeros_like(b)), check_trace=False)
    assert all(torch.equal(x, y) for x, y in zip(traced(a, b), f(a, b)))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(a, torch.ones_like(a))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            qfa.norm_rope(dual, v0, c, s)


@pytest.mark.gpu
def test_no_second_derivative(qfa):
    x, w = torch.randn(1, 2, 8, 64, device=DEV, requires_grad=True), torch.ones(64, device=DEV, requires_grad=True)
    y = qfa.norm_rope(x, w, None, None)
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(y, (x, w), torch.ones_like(y), create_graph=True)


def test_refusals(qfa):
    x, w, (cos, sin) = torch.randn(1, 2, 8, 64), torch.ones(64), m.table(16, 64)
    with pytest.raises(RuntimeError, match="GPU only"):
        qfa.norm_rope(x, w, cos, sin)
    with pytest.raises(ValueError):
        qfa.norm_rope(x[0], w, cos, sin)


@pytest.mark.gpu
def test_refusals_gpu(qfa):
    x, w = torch.randn(2, 2, 8, 64, device=DEV), torch.ones(64, device=DEV)
    cos, sin = (t.to(DEV) for t in m.table(16, 64))
    for bad, error, what in (((x, w[:32], cos, sin), ValueError, "weight"), ((x, w.double(), cos, sin), TypeError, "weight"),
                             ((x, w, cos, None), ValueError, "together"), ((x, w, cos.half(), sin.half()), TypeError, "float32"),
                             ((x, w, cos[:, :4], sin[:, :4]), ValueError, "rotated"), ((x, w, cos[:, :12], sin[:, :12]), ValueError, "rotated"),
                             ((x, w, cos[:0], sin[:0]), ValueError, "rotated"),
                             ((x, w, cos, sin, torch.zeros(2, 8, device=DEV, dtype=torch.int64)), TypeError, "int32"),
                             ((x, w, cos, sin, torch.zeros(3, device=DEV, dtype=torch.int32)), ValueError, "positions"),
                             ((x[..., :32].contiguous(), None, None, None), RuntimeError, "head_dim"), ((x[:, :, :0], w, cos, sin), RuntimeError, "positive"),
                             ((x, w, cos.clone().requires_grad_(True), sin), ValueError, "no gradient")):
        with pytest.raises(error, match=what):
            qfa.norm_rope(*bad)
    with pytest.raises(ValueError, match="shape"):
        qfa.norm_rope_pair(x, x[:, :, :4], w, w, cos, sin)
    with pytest.raises(TypeError, match="same dtype"):
        qfa.norm_rope_pair(x, x.half(), w, w, cos, sin)
    with pytest.raises(RuntimeError, match="eps"):
        qfa.norm_rope(x, w, cos, sin, eps=-1.0)
