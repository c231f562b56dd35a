"""paged_attention_weights into a tensor of the caller's: autograd sees that it changed."""
import pytest
import torch

import long_model as lm

DEV = "cuda:0"
dev = lm.dev


@pytest.mark.gpu
def test_a_tensor_kept_for_a_gradient_may_not_change_unseen(qfa):
    p = lm.Problem(2, 4, 2, 1, 64, 16, [40, 90], seed=3)
    q, cache, (table, starts) = dev(p.q), dev(p.cache), p.places()
    _, lse = qfa.quant_flash_attn_paged(q, cache, table, starts, return_lse=True)
    add = lambda w: qfa.paged_attention_weights(q, cache, lse, table, starts, weights=w, out=w)   # noqa: E731
    total, x = torch.rand(2, 2, p.width * 16, device=DEV), torch.rand(2, 2, p.width * 16, device=DEV, requires_grad=True)
    y = (total * x).sum()
    add(total)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (total * x).sum()
    y.backward()
    assert torch.equal(x.grad, total)
    with torch.inference_mode():   # such tensors have no count of their changes
        inside = torch.rand_like(total)
        before = inside.clone()
        add(inside)
        assert bool((inside >= before).all()) and not torch.equal(inside, before)
    other = torch.rand_like(total)
    with torch.inference_mode():
        add(other)
