"""What norm_rope keeps for its gradient: a rotation alone needs neither of its inputs."""
import ctypes
import gc

import pytest
import torch

import paged_model as m

DEV = "cuda:0"


def _inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, dq, dk = (torch.randn(2, h, 33, 128, generator=g).bfloat16().to(DEV) for h in (4, 2, 4, 2))
    return q, k, dq, dk, [t.to(DEV) for t in m.table(40, 64)], [(1 + 0.2 * torch.randn(128, generator=g)).to(DEV) for _ in range(2)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_rotated_tensor_may_change_before_the_gradient(qfa, interleaved):
    q, k, dq, dk, (cos, sin), _ = _inputs()

    def step(change):
        a, b = (t.clone().requires_grad_(True) for t in (q, k))
        x, y = a * 1, b * 1
        out = qfa.norm_rope_pair(x, y, None, None, cos, sin, interleaved=interleaved)
        if change:
            x.detach().zero_()
            y.detach().fill_(float("nan"))
        return torch.autograd.grad(out, (a, b), (dq, dk))
    assert all(torch.equal(x, y) for x, y in zip(step(True), step(False)))
    for got, dy in zip(step(True), (dq, dk)):
        want, _, _, _ = m.norm_rope_grad(dy.cpu(), dy.cpu(), None, cos.cpu(), sin.cpu(), None, 0.0, interleaved)
        assert ((got.cpu().double() - want).abs() <= m.HALF[torch.bfloat16] * want.abs() + 4 * m.U32 * dy.cpu().double().abs().amax()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("weights,needs,kept", [("", "qk", ""), ("q", "qk", "q"), ("k", "qk", "k"), ("qk", "qk", "qk"), ("qk", "q", "q"), ("qk", "k", "k"),
                                                ("q", "k", ""), ("qk", "w", "q"), ("q", "wk", "q")])
def test_inputs_are_kept_only_where_a_gradient_needs_them(qfa, weights, needs, kept):
    """needs: the tensors that want a gradient (w: q's weight).  What a step keeps is seen in the memory that is still held behind it."""
    _, _, _, _, (cos, sin), w = _inputs()
    w = [t.clone().requires_grad_(i == 0 and "w" in needs) if n in weights else None for i, (n, t) in enumerate(zip("qk", w))]
    size = {"q": 16 << 20, "k": 8 << 20}
    leaves = [torch.randn(1, h, 4096, 128, device=DEV).bfloat16().requires_grad_(n in needs) for n, h in (("q", 16), ("k", 8))]
    d = [torch.randn_like(t) for t in leaves]
    gc.collect()
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    x = [t * 1 for t in leaves]
    out = qfa.norm_rope_pair(*x, *w, cos.new_ones(4096, 64), sin.new_zeros(4096, 64))
    del x
    angles = 2 * 4096 * 64 * 4
    assert torch.cuda.memory_allocated() - held == size["q"] + size["k"] + angles + sum(size[n] for n in kept)
    wanted = [t for t in (*leaves, *w) if t is not None and t.requires_grad]
    grads = torch.autograd.grad(out, wanted, d)
    for i, n in enumerate("qk"):   # the same as each tensor's alone
        mine = [t for t in (leaves[i], w[i]) if t is not None and t.requires_grad]
        if mine:
            alone = torch.autograd.grad(qfa.norm_rope(leaves[i], w[i], cos.new_ones(4096, 64), sin.new_zeros(4096, 64)), mine, d[i])
            for t, g in zip(mine, alone):
                assert torch.equal(g, next(a for a, b in zip(grads, wanted) if b is t))


@pytest.mark.gpu
def test_inputs_that_have_to_be_copied(qfa):
    """Rows with gaps, broadcast batches and gradients: copies that a backward makes of both tensors live until its kernel has them."""
    q, k, dq, dk, (cos, sin), w = _inputs(4)
    gaps = lambda t: torch.stack([t, torch.zeros_like(t)], -1).flatten(-2)[..., ::2]   # noqa: E731
    wide = lambda t: t[:1].expand_as(t)                                            # noqa: E731

    def step(view, dense):
        leaves = [(view(t).contiguous() if dense else view(t)).requires_grad_(True) for t in (q, k)]
        out = qfa.norm_rope_pair(*leaves, *w, cos, sin)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, [view(d).contiguous() if dense else view(d) for d in (dq, dk)])]
    for view in (gaps, wide):
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(step(view, False), step(view, True)))


def test_pointers_that_the_backward_does_without_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, p = _lib.lib(), 0x1000   # never dereferenced: validation fails first

    def call(x=p, w=None, y=p, dy=p, dw=None, sx=(1024, 512, 64)):
        t = _lib.NormRopeTensor(x=x, weight=w, y=y, dy=dy, dweight=dw, H=2, sx=sx, sy=(1024, 512, 64), sdy=(1024, 512, 64))
        rc = L.qfa_norm_rope_bwd(ctypes.byref(t), None, p, p, 64, 64, 0, None, 0, 0, 1, 1e-6, 2, 2, 1, 8, 64, p, 16, None)
        return rc, L.qfa_last_error()
    for kw, what in ((dict(x=None, w=p), b"null"), (dict(y=None), b"null"), (dict(y=None, w=p), b"null"), (dict(dy=None), b"null"),
                     (dict(x=None, sx=(0, 0, 0), dw=p), b"dweight"),            # x is not looked at without a weight,
                     (dict(y=None, w=p, dw=p), b"workspace"),                   # nor dx written where dweight alone is wanted
                     (dict(w=p, sx=(0, 0, 0)), b"strides")):
        rc, said = call(**kw)
        assert rc == -1 and what in said, (kw, said)
