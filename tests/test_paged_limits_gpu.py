"""The largest calls of quant_flash_attn_paged: what is counted in 31 bits is the work that the call can have."""
import ctypes

import pytest
import torch

import paged_model as m

DEV = "cuda:0"


@pytest.mark.gpu
def test_a_long_piece_under_a_wide_table(qfa):
    """16384 tokens of 64 heads on 8, a table with room for 2^20 keys; only the last 101 tokens see any."""
    H, Hk, N, D, page, seen = 64, 8, 16384, 64, 64, 101
    g = torch.Generator(device=DEV).manual_seed(0)
    cache = qfa.make_paged_cache(4, Hk, page, D, device=DEV)
    k, v = (torch.randn(2, Hk, seen, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    table = torch.full((2, (1 << 20) // page), -1, dtype=torch.int32, device=DEV)
    table[:, :2] = torch.tensor([[0, 1], [3, 2]], dtype=torch.int32)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    qfa.paged_cache_append(cache, k, v, table, zero)
    q = torch.randn(2, H, N, D, device=DEV, generator=g).bfloat16()
    o = qfa.quant_flash_attn_paged(q, cache, table, zero + (seen - N))
    assert not o[:, :, :N - seen].any()
    kh, vh = (t.cpu().double() for t in qfa.paged_cache_read(cache, table, zero, seen, dtype=torch.float32))
    want, size = m.attention(m.values(*m.quantized(q[:, :, N - seen:].cpu().float())), list(kh), list(vh), torch.zeros(2, dtype=torch.int32), None, True, m.sm_of(D))
    assert ((o[:, :, N - seen:].cpu().double() - want).abs() <= m.attention_bound(want, size, q.dtype, seen, 0.05)).all()


def test_limits_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, p = _lib.lib(), 0x1000   # never dereferenced: validation fails first

    def call(B, H, Hk, N, keys, D=64, prefix=0):
        c = _lib.PagedCacheStruct(k_codes=p, k_scale=p, k_zero=p, v_codes=p, v_scale=p, v_zero=p, pages=4, H=Hk, page_size=64, D=D, scale_dtype=1)
        width = keys // 64
        rc = L.qfa_attn_paged(ctypes.byref(c), p, 2, H * N * D, N * D, D, p, width, width, 1, p, None, p, B, H, N, prefix, 0.1, 1, p, 16, None)
        return rc, L.qfa_last_error()
    for args in ((2, 64, 8, 16384, 1 << 20), (64, 32, 8, 4096, 131072), (256, 8, 8, 1, 1 << 20), (1, 128, 1, 65536, 1 << 20)):
        rc, said = call(*args)
        assert rc == -1 and b"workspace" in said, (args, said)   # everything before the workspace is in order
    for args in ((1 << 16, 8, 8, 1, 1 << 20), (1 << 14, 32, 8, 4096, 4096), (1 << 20, 1024, 1, 1, 64), (4096, 32, 8, 4096, 131072)):
        rc, said = call(*args)
        assert rc == -2 and b"too many" in said, (args, said)
    rc, said = call(1 << 14, 32, 32, 1, 1 << 17, prefix=1 << 17)
    assert rc == -2 and b"too many" in said
