"""quant_flash_attn_paged_blocks against attention in 64 bits on the listed blocks (exactly the quantized operands, the queries' codes from the C
oracle), on caches whose other rows hold any codes and scales that are NaN or infinite."""
import ctypes
import math

import pytest
import torch

import long_model as lm
import paged_model as m

DEV = "cuda:0"
dev = lm.dev


def _expect(p, blocks, sm):
    qh = m.values(*m.quantized(p.q.float()))
    o, size = torch.zeros(p.B, p.H, p.N, p.D, dtype=torch.float64), torch.zeros(p.B, p.H, p.N, p.D, dtype=torch.float64)
    for b in range(p.B):
        L = p.rows[0][b].shape[1]
        for n in range(p.tokens[b]):
            pos = int(p.starts[b]) + n
            for h in range(p.Hk):
                at = []
                for j in blocks[b, h, n].tolist():
                    if 0 <= j < p.width and 0 <= int(p.table[b, j]) < p.pages:
                        at += [i for i in range(j * p.page, (j + 1) * p.page) if i <= pos and i < L]
                if not at:
                    continue
                for g in range(h * p.G, (h + 1) * p.G):
                    o[b, g, n], size[b, g, n] = lm.attention_on(qh[b, g, n], p.rows[0][b][h, at], p.rows[1][b][h, at], torch.ones(len(at), dtype=torch.bool), sm)
    return o, size


def _check(qfa, p, keep, blocks=None, seed=0):
    blocks = p.fake_lists(keep, seed) if blocks is None else blocks
    sm = m.sm_of(p.D)
    o = qfa.quant_flash_attn_paged_blocks(dev(p.q), dev(p.cache), *p.places(), dev(blocks), dev(p.counts), sm_scale=sm)
    assert o.dtype == p.q.dtype and o.shape == p.q.shape and torch.isfinite(o).all()
    want, size = _expect(p, blocks, sm)
    excess = (o.cpu().double() - want).abs() - m.attention_bound(want, size, p.q.dtype, keep * p.page, p.v_scale)
    assert excess.max() <= 0, f"over the bound by {excess.max().item():.3e} at {want.flatten()[excess.argmax()].item():.3e}"
    return o


# ends of halves, tiles and pages; lists longer than the sequence, of one block, of an odd number
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("keep", [1, 3, 8])
def test_lengths(qfa, D, page, keep):
    _check(qfa, lm.Problem(4, 2, 2, 1, D, page, [1, 17, 64, 333], seed=D + page + keep), keep)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,N", [(8, 2, 1), (16, 1, 1), (6, 2, 3), (40, 1, 2), (33, 1, 1), (10, 2, 21), (2, 1, 70)])
def test_heads_and_tokens(qfa, H, Hk, N):
    _check(qfa, lm.Problem(2, H, Hk, N, 128, 32, [N + 400, N], seed=H + N), 5)


# lists that several workgroups share, workgroups with several lists
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,D,keep,keys", [(1, 1, 1, 1, 128, 300, 9000), (1, 4, 1, 1, 64, 90, 2000), (2, 2, 2, 3, 256, 120, 4000), (70, 2, 2, 5, 64, 3, 200),
                                                  (3, 20, 1, 1, 128, 200, 5000), (9, 8, 8, 9, 64, 2, 100), (1, 32, 1, 1, 256, 64, 3000)])
def test_dealing(qfa, B, H, Hk, N, D, keep, keys):
    _check(qfa, lm.Problem(B, H, Hk, N, D, 16, [keys - 7 * i for i in range(B)], seed=B), keep)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_types_and_layouts(qfa, dtype, scale_dtype):
    for D, layout in ((64, "bhnd"), (128, "bnhd"), (256, "bnhd")):
        _check(qfa, lm.Problem(2, 6, 3, 4, D, 64, [333, 90], dtype=dtype, scale_dtype=scale_dtype, layout=layout, seed=2), 3)


# Queries in fp32: no 16-bit rounding is left.  The score's roundings (the query's scale, that times sm_scale and log2(e), the key's scale, the multiply-add: 4 of the score's size in
# log2 units, as in weights_bound; they move a probability, and the sum that divides it, so twice) and 1 ulp of v_exp; p' in two binary16 parts (22 bits; 2^-25
# where it lies 2^21 below the largest) and its product with the scale; sums in fp32 of terms of at most 255 v_scale: those of a copy of the rows, 32 roundings inside a product and
# one for each, eight for the joining; the division and what is stored.
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,D,page,keep,keys,scale_dtype", [
    (2, 8, 2, 1, 64, 16, 12, 400, torch.float32), (2, 20, 2, 3, 128, 32, 20, 900, torch.float32), (1, 9, 1, 2, 256, 16, 40, 800, torch.float16),
    (3, 4, 1, 200, 128, 16, 33, 700, torch.float32), (2, 2, 2, 140, 64, 64, 7, 500, torch.bfloat16), (1, 4, 1, 1030, 256, 16, 20, 1100, torch.float32),
    (1, 16, 1, 1, 128, 16, 260, 4500, torch.float32)])
def test_fp32_queries(qfa, B, H, Hk, N, D, page, keep, keys, scale_dtype):
    p = lm.Problem(B, H, Hk, N, D, page, [max(N, keys - 37 * i) for i in range(B)], dtype=torch.float32, scale_dtype=scale_dtype, seed=D + N)
    blocks, sm = p.fake_lists(keep, D), m.sm_of(D)
    o = qfa.quant_flash_attn_paged_blocks(dev(p.q), dev(p.cache), *p.places(), dev(blocks), sm_scale=sm)
    want, size = _expect(p, blocks, sm)
    qh = m.values(*m.quantized(p.q.float()))
    score = max(float((p.rows[0][b][h // p.G] @ qh[b, h].T).abs().max()) for b in range(B) for h in range(H)) * sm / math.log(2)
    relative = 2 * (math.log(2) * m.U32 * (4 * score + 3) + 2 * m.U32) + 2.0 ** -22 + 8 * m.U32
    sums = (32 + keep * page / 32 + 8) * m.U32 * 255 * p.v_scale
    assert bool(((o.cpu().double() - want).abs() <= relative * size + sums + 2 * m.U32 * want.abs() + m.TINY[torch.float32]).all())
    assert float((o.cpu().double() - want).norm() / want.norm()) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-4, 1e3])
def test_rows_of_any_size(qfa, size):
    p = lm.Problem(2, 4, 2, 3, 128, 32, [700, 41], scale_dtype=torch.float32, size=size, seed=4)
    p.q = p.q / size
    _check(qfa, p, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [4, 40])
def test_padding(qfa, keep):
    _check(qfa, lm.Problem(6, 8, 2, 5, 64, 16, [8, 700, 44, 9, 5, 100], counts=[5, 3, 0, 1, 14, -3], seed=keep), keep)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [6, 60])
def test_lists_as_they_may_come(qfa, keep):
    """Blocks twice, behind the token, outside the table, without a page, holes between them and in front, a list of nothing."""
    p = lm.Problem(4, 4, 2, 2, 64, 16, [1000, 1000, 70, 1000], seed=7)
    p.table[1, 5], p.table[1, 6], p.table[3, 2] = -1, p.pages, 1 << 30
    g = torch.Generator().manual_seed(keep)
    blocks = torch.randint(-3, p.width + 5, (4, 2, 2, keep), generator=g).int()
    blocks[0, 0, 0, :4] = torch.tensor([3, 3, -1, 2147483647])
    blocks[0, 1] = -1
    blocks[1, :, :, :3] = torch.tensor([5, 6, 7])
    blocks[2, :, :, 5:] = -2147483648
    blocks[2, 1, 1, :] = -1
    blocks[2, 1, 1, -1] = 4
    _check(qfa, p, keep, blocks)


# more lists than the chip works on at once, of few query heads each; of more than 32 tiles of 64 keys; a third of the places without a block
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,D,page,keep,keys,dtype,scale_dtype", [
    (3, 8, 2, 90, 64, 16, 150, 2600, torch.float16, torch.float32), (2, 3, 1, 270, 128, 128, 19, 2500, torch.bfloat16, torch.float16),
    (1, 4, 4, 130, 128, 32, 5, 500, torch.float32, torch.bfloat16), (66, 20, 10, 1, 64, 64, 3, 700, torch.bfloat16, torch.float32),
    (300, 2, 2, 1, 128, 16, 9, 333, torch.bfloat16, torch.float16), (2, 6, 2, 260, 256, 64, 37, 2400, torch.float16, torch.float16),
    (1, 2, 1, 1030, 256, 16, 7, 1100, torch.float32, torch.float32)])
def test_many_lists(qfa, B, H, Hk, N, D, page, keep, keys, dtype, scale_dtype):
    p = lm.Problem(B, H, Hk, N, D, page, [max(N, keys - 37 * i) for i in range(B)], counts=[max(0, N - 3 * i) if N > 1 else 1 for i in range(B)], seed=H + N,
                   dtype=dtype, scale_dtype=scale_dtype)
    g = torch.Generator().manual_seed(B)
    blocks = torch.rand(B, Hk, N, p.width, generator=g).argsort(-1)[..., :keep].int()
    if blocks.shape[-1] < keep:
        blocks = torch.cat([blocks, torch.full((B, Hk, N, keep - blocks.shape[-1]), -1, dtype=torch.int32)], -1)
    blocks[torch.rand(blocks.shape, generator=g) < 1 / 3] = -1
    blocks[0, 0, 0] = -1
    _check(qfa, p, keep, blocks.contiguous())


@pytest.mark.gpu
def test_rows_that_see_nothing_are_zero(qfa):
    p = lm.Problem(3, 4, 2, 6, 128, 16, [50, 6, 20], seed=1)
    blocks = torch.zeros(3, 2, 6, 2, dtype=torch.int32)
    starts = torch.tensor([44, -3, -2147483648], dtype=torch.int32)
    o = qfa.quant_flash_attn_paged_blocks(dev(p.q), dev(p.cache), dev(p.table), dev(starts), dev(blocks)).cpu()
    assert not o[1, :, :3].any() and not o[2].any() and o[1, :, 3:].abs().amax(-1).min() > 0 and torch.isfinite(o).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,keys", [(3, 8, 2, 1, 500), (2, 4, 4, 5, 150)])
def test_all_blocks_are_all_keys(qfa, B, H, Hk, N, keys):
    """A list of every block against quant_flash_attn_paged: the same scores and probabilities, so the difference is that of roundings."""
    p = lm.Problem(B, H, Hk, N, 128, 16, [keys - 31 * i for i in range(B)], seed=3)
    blocks = torch.arange(p.width, dtype=torch.int32).expand(B, Hk, N, p.width)
    args = (dev(p.q), dev(p.cache), *p.places())
    o = qfa.quant_flash_attn_paged_blocks(*args, dev(blocks))
    full = qfa.quant_flash_attn_paged(*args)
    _, size = _expect(p, blocks, m.sm_of(128))
    assert ((o.float() - full.float()).abs().cpu() <= 2 * m.HALF[torch.bfloat16] * full.float().abs().cpu() + 2.0 ** -9 * size + 1e-5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hk,G,N,D,keys", [(50, 4, 1, 1, 64, 4800), (2, 2, 4, 40, 128, 9000), (5, 7, 20, 1, 64, 3000), (1, 3, 2, 900, 64, 2000)])
def test_workgroups_with_parts_of_several_lists(qfa, B, Hk, G, N, D, keys):
    """Enough long lists that a workgroup ends one and begins the next, and more than are under way at once: every block in any order, against
    quant_flash_attn_paged.  Both round probabilities times scales to binary16 (2^-11 each, relative to a sum of p |v|), the offsets' sums, and the result."""
    g, page = torch.Generator().manual_seed(B), 16
    width = keys // page
    table = torch.randperm(B * width, generator=g).int().view(B, width).to(DEV)
    zero = torch.zeros(B, dtype=torch.int32, device=DEV)
    q = (2 * torch.randn(B, Hk * G, N, D, generator=g)).bfloat16().to(DEV)
    k, v = (torch.randn(B, Hk, keys, D, device=DEV).bfloat16() for _ in range(2))
    starts = torch.full((B,), keys - N - 3, dtype=torch.int32, device=DEV)
    blocks = torch.rand(B, Hk, N, width, device=DEV).argsort(-1).int()
    outs = []
    for values in (v, v.abs()):
        cache = qfa.make_paged_cache(B * width, Hk, page, D, device=DEV)
        qfa.paged_cache_append(cache, k, values, table, zero)
        outs.append(qfa.quant_flash_attn_paged(q, cache, table, starts).double())
        if values is v:
            o = qfa.quant_flash_attn_paged_blocks(q, cache, table, starts, blocks).double()
    full, size = outs
    assert bool(((o - full).abs() <= 2 * m.HALF[torch.bfloat16] * full.abs() + 2.0 ** -9 * size + 2 * (32 + keys / 32) * m.U32 * 1407 * 0.05).all())


@pytest.mark.gpu
def test_a_row_that_is_not_finite_stays_alone(qfa):
    p = lm.Problem(2, 4, 2, 3, 128, 16, [40, 90], seed=9)
    blocks = p.fake_lists(3)
    call = lambda q: qfa.quant_flash_attn_paged_blocks(dev(q), dev(p.cache), *p.places(), dev(blocks)).cpu()   # noqa: E731
    clean = call(p.q)
    q = p.q.clone()
    q[1, 2, 1, 7] = float("nan")
    o = call(q)
    keep = torch.ones(2, 4, 3, dtype=torch.bool)
    keep[1, 2, 1] = False
    assert torch.equal(o[keep], clean[keep])


@pytest.mark.gpu
def test_pages_past_32_bits(qfa):
    H, page, D = 8, 64, 128
    pages = (1 << 32) // (H * page * D) + 64
    cache = [torch.empty(pages, H, page, d, dtype=t, device=DEV) for d, t in ((D, torch.int8), (1, torch.float32), (1, torch.int8)) * 2]
    bounds = qfa.make_page_bounds(cache)
    k, v, q = (torch.randn(2, H, n, D, device=DEV).bfloat16() for n in (150, 150, 1))
    near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
    far = torch.tensor([[pages - 1, pages - 2, pages - 9], [pages - 40, pages - 3, pages - 20]], dtype=torch.int32, device=DEV)
    zero, last = torch.zeros(2, dtype=torch.int32, device=DEV), torch.full((2,), 149, dtype=torch.int32, device=DEV)
    out = []
    for t in (near, far):
        qfa.paged_cache_append(cache, k, v, t, zero)
        qfa.paged_bounds_update(bounds, cache, t, zero, 150)
        blocks, scores = qfa.paged_select_blocks(q, cache, bounds, t, last, 2, return_scores=True)
        o, lse = qfa.quant_flash_attn_paged(q, cache, t, last, return_lse=True)
        out.append((blocks, scores, qfa.quant_flash_attn_paged_blocks(q, cache, t, last, blocks), lse, qfa.paged_attention_weights(q, cache, lse, t, last)))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    w = out[0][4]
    kept = qfa.paged_cache_evict(cache, near, last, w, 100, torch.tensor([[pages - 5, 7], [8, pages - 6]], dtype=torch.int32, device=DEV))
    again = qfa.paged_cache_evict(cache, far, last, w, 100, torch.tensor([[9, pages - 7], [pages - 8, 10]], dtype=torch.int32, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(kept, again))
    rows = [qfa.paged_cache_read(cache, torch.tensor(t, dtype=torch.int32, device=DEV), zero, 100, kept[2])
            for t in ([[pages - 5, 7], [8, pages - 6]], [[9, pages - 7], [pages - 8, 10]])]
    assert all(torch.equal(a, b) for a, b in zip(*rows)) and rows[0][0].abs().max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [3, 100])
def test_repeats_graphs_and_overlap(qfa, keep):
    p = lm.Problem(3, 8, 2, 2, 128, 16, [1900, 1700, 300], seed=6)
    args, blocks = (dev(p.q), dev(p.cache), *p.places()), dev(p.fake_lists(keep))
    starts, first = args[3], args[3].clone()
    call = lambda: qfa.quant_flash_attn_paged_blocks(*args, blocks)   # noqa: E731
    want = call()
    assert torch.equal(want, call())
    side, graphs = torch.cuda.Stream(), []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call()
        graphs.append((graph, o))
    for i in range(3):
        starts.copy_(first - 40 * i)
        for _, o in graphs:
            o.zero_()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            other = call()
        eager = call()
        torch.cuda.synchronize()
        assert all(torch.equal(o, eager) for o in (graphs[0][1], graphs[1][1], other)), i


@pytest.mark.gpu
def test_traced(qfa):
    p = lm.Problem(2, 4, 2, 1, 64, 16, [40, 90], seed=9)
    cache, (table, starts), blocks = dev(p.cache), p.places(), dev(p.fake_lists(3))
    f = lambda q, s: qfa.quant_flash_attn_paged_blocks(q, cache, table, s, blocks)   # noqa: E731
    traced = torch.jit.trace(f, (dev(p.q), starts), check_trace=False)
    assert torch.equal(traced(dev(p.q), starts - 20), f(dev(p.q), starts - 20))


@pytest.mark.gpu
def test_refusals(qfa):
    p = lm.Problem(2, 4, 2, 1, 64, 16, [40, 30])
    q, cache, (table, starts), blocks = dev(p.q), dev(p.cache), p.places(), dev(p.fake_lists(2))

    def refused(error, q=q, cache=cache, table=table, starts=starts, blocks=blocks, **kw):
        with pytest.raises(error):
            qfa.quant_flash_attn_paged_blocks(q, cache, table, starts, blocks, **kw)
    refused(TypeError, blocks=blocks.long())
    refused(ValueError, blocks=blocks[:, :1])
    refused(ValueError, blocks=blocks[..., :0])
    refused(ValueError, q=q[:, :3])
    refused(RuntimeError, blocks=blocks.cpu())
    refused(RuntimeError, sm_scale=0.0)
    refused(RuntimeError, q=q.float().requires_grad_(True))


def test_argument_errors_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, P = _lib.lib(), 0x1000

    def call(q=P, dt=2, sq=(1024, 512, 64), H=4, N=2, B=1, width=4, keep=2, blocks=P, o=P, sm=0.1, ws=P, wsb=1 << 30, page=16, D=64):
        c = _lib.PagedCacheStruct(k_codes=P, k_scale=P, k_zero=P, v_codes=P, v_scale=P, v_zero=P, pages=4, H=2, page_size=page, D=D, scale_dtype=1)
        return L.qfa_attn_paged_blocks(ctypes.byref(c), q, dt, *sq, P, width, width, 1, P, None, blocks, keep, o, B, H, N, sm, ws, wsb, None)
    for rc, code in ((call(q=None), -1), (call(dt=9), -1), (call(sq=(1024, 512, 60)), -1), (call(H=3), -1), (call(N=0), -1), (call(blocks=None), -1), (call(o=P + 8), -1),
                     (call(keep=0), -1), (call(keep=(1 << 30) + 1), -1), (call(sm=0.0), -1), (call(sm=float("nan")), -1), (call(page=48), -2), (call(D=96), -2),
                     (call(B=1 << 15, N=1 << 13, keep=1 << 12), -2), (call(keep=1 << 20, ws=None), -1), (call(keep=1 << 20, wsb=64), -1)):
        assert rc == code, L.qfa_last_error()
    ws = L.qfa_attn_paged_blocks_workspace_bytes
    assert ws(1, 4, 2, 1, 128, 1 << 20, 16) > 0 and ws(1, 4, 3, 1, 128, 8, 16) == 0 and ws(1, 4, 2, 1, 128, 8, 24) == 0 and ws(1, 4, 2, 1, 128, 0, 16) == 0


def test_lists_of_too_many_keys_need_no_gpu(qfa):
    """The keys of a list are counted in 31 bits."""
    from quant_flash_attn_amd import _lib
    L, P = _lib.lib(), 0x1000
    for page, keep in ((16, (1 << 26) + 1), (16, 1 << 28), (1 << 20, 1025)):
        c = _lib.PagedCacheStruct(k_codes=P, k_scale=P, k_zero=P, v_codes=P, v_scale=P, v_zero=P, pages=4, H=1, page_size=page, D=64, scale_dtype=1)
        assert L.qfa_attn_paged_blocks(ctypes.byref(c), P, 2, 64, 64, 64, P, 4, 4, 1, P, None, P, keep, P, 1, 1, 1, 0.1, P, 1 << 40, None) == -2
        assert L.qfa_attn_paged_blocks_workspace_bytes(1, 1, 1, 1, 64, keep, page) == 0
