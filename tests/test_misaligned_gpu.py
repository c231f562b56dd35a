"""Tensors that begin anywhere: contiguous ones at an address that is no multiple of 16 bytes, and sizes of one with any stride."""
import pytest
import torch

import paged_model as m

DEV = "cuda:0"


def _off(t, by):
    """The same values, dense, `by` elements behind an aligned address."""
    room = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    out = room[by:].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 and out.is_contiguous()
    return out


def _odd(t, dim):
    """The same values with a stride of 1 where the size is one."""
    stride = [1 if d == dim else s for d, s in enumerate(t.stride())]
    return torch.as_strided(t, t.shape, stride)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("by", [1, 3])
def test_dense_tensors_anywhere(qfa, dtype, by):
    g = torch.Generator().manual_seed(0)
    q, k, v, dq, dk = (torch.randn(2, 2, 40, 128, generator=g).to(dtype).to(DEV) for _ in range(5))
    w, (cos, sin) = torch.rand(128, device=DEV), (t.to(DEV) for t in m.table(40, 128))
    table, pages = m.shared_pages(2, 3, 0, 1)
    table, zero = table.to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV)

    def run(move):
        a, b = (move(t).requires_grad_(True) for t in (q, k))
        out = qfa.norm_rope_pair(a, b, move(w), move(w), move(cos), move(sin))
        grads = torch.autograd.grad(out, (a, b), (move(dq), move(dk)))
        cache = qfa.make_paged_cache(pages, 2, 16, 128, device=DEV)
        qfa.paged_cache_append(cache, move(k), move(v), table, zero, k_weight=move(w), cos=move(cos), sin=move(sin))
        return [*out, *grads, *cache, qfa.quant_flash_attn_paged(move(q), cache, table, zero), *qfa.asymmetric_quant_per_token(move(q)),
                qfa.quant_flash_attn_qkv(move(q), move(k), move(v), True, 0.1)]
    assert all(torch.equal(x, y) for x, y in zip(run(lambda t: _off(t.detach(), by)), run(lambda t: t.detach().clone())))


@pytest.mark.gpu
def test_strides_of_sizes_of_one(qfa):
    g = torch.Generator().manual_seed(0)
    w, (cos, sin) = torch.rand(64, device=DEV), (t.to(DEV) for t in m.table(40, 64))
    for shape, dim in (((1, 3, 5, 64), 0), ((2, 1, 5, 64), 1), ((2, 3, 1, 64), 2)):
        x = torch.randn(*shape, generator=g).to(DEV).half()
        y = _odd(x, dim)
        assert torch.equal(qfa.norm_rope(y, w, cos, sin), qfa.norm_rope(x, w, cos, sin))
        assert all(torch.equal(a, b) for a, b in zip(qfa.asymmetric_quant_per_token(y), qfa.asymmetric_quant_per_token(x)))
        table = torch.arange(shape[0], dtype=torch.int32, device=DEV)[:, None]
        cache, zero = [qfa.make_paged_cache(shape[0], shape[1], 16, 64, device=DEV) for _ in range(2)], torch.zeros(shape[0], dtype=torch.int32, device=DEV)
        for c, t in zip(cache, (x, y)):
            qfa.paged_cache_append(c, t, t, table, zero)
        assert all(torch.equal(a, b) for a, b in zip(*cache))
        assert torch.equal(qfa.quant_flash_attn_paged(y, cache[0], table, zero), qfa.quant_flash_attn_paged(x, cache[0], table, zero))
