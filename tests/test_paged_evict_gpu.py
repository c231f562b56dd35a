"""paged_cache_evict: the kept slots against a plain sort, the moved rows byte for byte; and the operators for long caches one after the other as a
serving loop runs them."""
import ctypes
import math

import pytest
import torch

import long_model as lm
import paged_model as m

DEV = "cuda:0"
dev = lm.dev


def _cache(pages, Hk, page, D, scale_dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(-128, 128, (pages, Hk, page, d), generator=g).to(torch.int8) if t is None else torch.randn(pages, Hk, page, d, generator=g).to(t)
            for d, t in ((D, None), (1, scale_dtype), (1, None)) * 2]


def _check(qfa, B, Hk, D, page, lengths, keep, first=0, last=0, scale_dtype=torch.float16, weights=None, seed=0, width=None, new_width=None, edit=None):
    g = torch.Generator().manual_seed(seed)
    width = width or max(1, -(-max(lengths) // page))
    new_width = new_width or max(1, -(-min(keep, width * page) // page))
    order = torch.randperm(B * (width + new_width) + 2, generator=g).int()
    table, new_table = order[:B * width].view(B, width).clone(), order[B * width:B * (width + new_width)].view(B, new_width).clone()
    if edit:
        edit(table, new_table)
    cache = _cache(order.numel(), Hk, page, D, scale_dtype, seed)
    if weights is None:
        weights = torch.randn(B, Hk, width * page, generator=g)
    n = torch.tensor(lengths, dtype=torch.int32)
    on = dev(cache)
    kept, new_weights, new_lengths = (t.cpu() for t in qfa.paged_cache_evict(on, dev(table), dev(n), dev(weights), keep, dev(new_table), first=first, last=last))
    want = [t.clone() for t in cache]
    pages = order.numel()
    for b in range(B):
        have = max(0, min(lengths[b], width * page))
        assert int(new_lengths[b]) == min(have, keep)
        for h in range(Hk):
            slots = lm.evict(weights[b, h], have, keep, first, last)
            assert kept[b, h].tolist() == slots + [-1] * (keep - len(slots)), (b, h)
            expect = torch.zeros(new_width * page)
            expect[:len(slots)] = weights[b, h, slots]
            assert torch.equal(new_weights[b, h].nan_to_num(7.0), expect.nan_to_num(7.0)), (b, h)
            at = torch.tensor(slots, dtype=torch.long)
            i = torch.arange(len(slots))
            src, to = table[b, at // page].long(), new_table[b, i // page].long()
            there, goes = (src >= 0) & (src < pages), (to >= 0) & (to < pages)
            for t, w in zip(cache, want):
                rows = t[src.clamp(0, pages - 1), h, at % page]
                rows[~there] = 0
                w[to[goes], h, (i % page)[goes]] = rows[goes]
    for t, w, name in zip(on, want, ("k codes", "k scale", "k zero", "v codes", "v scale", "v zero")):
        assert torch.equal(t.cpu(), w), name
    return kept


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("lengths,keep", [([1, 0, 17], 1), ([200, 64, 65], 64), ([700, 30, 333], 100), ([15, 16, 33], 500)])
def test_lengths(qfa, D, page, lengths, keep):
    _check(qfa, 3, 2, D, page, lengths, keep, seed=D + keep)


@pytest.mark.gpu
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("first,last", [(0, 0), (4, 30), (50, 0), (0, 50), (20, 30), (1, 1)])
def test_first_and_last(qfa, scale_dtype, first, last):
    _check(qfa, 2, 3, 64, 16, [300, 52], 50, first, last, scale_dtype=scale_dtype, seed=first + last)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [1, 1000, 4999, 9000])
def test_many_slots(qfa, keep):
    _check(qfa, 1, 2, 64, 128, [9001], keep, first=min(3, keep), last=min(100, keep - min(3, keep)), seed=keep)


# more slots than are brought to LDS, and more than 2^16 that are taken, that are equal, that are both
@pytest.mark.gpu
@pytest.mark.parametrize("length,keep,values", [(20011, 700, None), (140001, 70007, None), (140001, 70007, [0.0]), (140001, 3, [0.0]), (140001, 139000, [0.0, 1.0])])
def test_more_slots_than_are_held(qfa, length, keep, values):
    w = None
    if values:
        w = torch.tensor(values)[torch.randint(0, len(values), (1, 1, -(-length // 1024) * 1024), generator=torch.Generator().manual_seed(keep))]
    _check(qfa, 1, 1, 64, 1024, [length], keep, first=1, last=2, weights=w, seed=keep)


@pytest.mark.gpu
def test_ties_and_odd_weights(qfa):
    """Equal weights go to the lowest slots; -0 equals 0; infinities are the ends, NaN lies below them; subnormals are told apart."""
    g = torch.Generator().manual_seed(2)
    values = torch.tensor([0.0, -0.0, 1.0, 1.0, math.inf, -math.inf, math.nan, -math.nan, 1e-45, -1e-45, 2e-45, 3.4e38, -3.4e38, 1.0000001])
    w = values[torch.randint(0, values.numel(), (2, 2, 416), generator=g)]
    for keep in (3, 50, 200, 380, 400):
        _check(qfa, 2, 2, 64, 16, [410, 400], keep, first=1, last=1, weights=w, seed=keep)
    _check(qfa, 2, 2, 64, 16, [410, 77], 30, weights=torch.zeros(2, 2, 416))
    _check(qfa, 2, 2, 64, 16, [410, 77], 30, weights=torch.full((2, 2, 416), math.nan))


@pytest.mark.gpu
def test_lengths_outside_and_tables_with_holes(qfa):
    def edit(table, new_table):
        table[0, 2], table[1, 0], new_table[1, 1], new_table[2, 0] = -1, 1 << 30, -1, 1 << 30
    _check(qfa, 4, 2, 64, 16, [200, 90, 150, -5], 60, 2, 10, edit=edit)
    _check(qfa, 2, 2, 64, 16, [2147483647, -2147483648], 60, width=8, seed=1)


@pytest.mark.gpu
def test_more_room_than_needed_and_strided_tables(qfa):
    _check(qfa, 2, 2, 128, 16, [100, 20], 40, width=20, new_width=9)
    p = _cache(40, 2, 16, 64, torch.float16, 0)
    table = torch.arange(24, dtype=torch.int32).view(6, 4)
    one, two = dev(p), dev(p)
    w, n = torch.rand(2, 2, 96, device=DEV), torch.tensor([90, 60], dtype=torch.int32, device=DEV)
    new = torch.arange(30, 40, dtype=torch.int32, device=DEV)
    a = qfa.paged_cache_evict(one, dev(table).t()[1:3], n, w, 33, new.view(5, 2).t()[:, :3])
    b = qfa.paged_cache_evict(two, dev(table).t()[1:3].contiguous(), n, w, 33, new.view(5, 2).t()[:, :3].contiguous())
    assert all(torch.equal(x, y) for x, y in zip((*a, *one), (*b, *two)))


@pytest.mark.gpu
def test_shared_pages_stay(qfa):
    """Two sequences that share their first pages: both go to pages of their own, the shared ones are as before."""
    cache = _cache(20, 2, 16, 64, torch.float16, 3)
    on = dev(cache)
    table = torch.tensor([[0, 1, 2], [0, 1, 3]], dtype=torch.int32, device=DEV)
    w = torch.rand(2, 2, 48, device=DEV)
    qfa.paged_cache_evict(on, table, torch.tensor([48, 40], dtype=torch.int32, device=DEV), w, 20, torch.tensor([[4, 5], [6, 7]], dtype=torch.int32, device=DEV))
    assert all(torch.equal(a[:4].cpu(), b[:4]) and torch.equal(a[8:].cpu(), b[8:]) for a, b in zip(on, cache))


@pytest.mark.gpu
def test_graphs_streams_and_overlap(qfa):
    cache = dev(_cache(200, 2, 16, 64, torch.float16, 3))
    table = torch.arange(60, dtype=torch.int32, device=DEV).view(3, 20)
    news = [torch.arange(60 + 30 * i, 90 + 30 * i, dtype=torch.int32, device=DEV).view(3, 10) for i in range(4)]
    n, w = torch.tensor([300, 77, 160], dtype=torch.int32, device=DEV), torch.rand(3, 2, 320, device=DEV)
    call = lambda i: qfa.paged_cache_evict(cache, table, n, w, 150, news[i], first=2, last=20)   # noqa: E731
    rows = lambda i: [t[news[i].long()] for t in cache]   # noqa: E731
    call(0)
    side, graphs = torch.cuda.Stream(), []
    for i in (1, 2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call(i)
        graphs.append((graph, o))
    first = n.clone()
    for i in range(3):
        n.copy_(first - 30 * i)
        w.copy_(torch.rand_like(w))
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            other = call(3)
        eager = call(0)
        torch.cuda.synchronize()
        for o in (graphs[0][1], graphs[1][1], other):
            assert all(torch.equal(a, b) for a, b in zip(o, eager)), i
        for r in (1, 2, 3):
            for b in range(3):
                kept = int(eager[2][b])
                for x, y in zip(rows(r), rows(0)):
                    x, y = (t[b].transpose(1, 2).flatten(0, 1)[:kept] for t in (x, y))
                    assert torch.equal(x, y), (i, r, b)


@pytest.mark.gpu
def test_refusals(qfa):
    cache = dev(_cache(12, 2, 16, 64, torch.float16, 3))
    table, new = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4), torch.arange(8, 12, dtype=torch.int32, device=DEV).view(2, 2)
    n, w = torch.tensor([60, 30], dtype=torch.int32, device=DEV), torch.rand(2, 2, 64, device=DEV)

    def refused(error, table=table, n=n, w=w, keep=20, new=new, **kw):
        with pytest.raises(error):
            qfa.paged_cache_evict(cache, table, n, w, keep, new, **kw)
    refused(ValueError, keep=0)
    refused(ValueError, keep=33)                # two pages of 16 do not hold them
    refused(ValueError, first=15, last=6)
    refused(ValueError, last=-1)
    refused(ValueError, w=w[..., :-1])
    refused(TypeError, w=w.half())
    refused(TypeError, new=new.long())
    refused(ValueError, new=new[:1])
    refused(TypeError, n=n.long())
    refused(ValueError, n=n[:1])
    refused(RuntimeError, w=w.cpu())
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda x: qfa.paged_cache_evict(cache, table, n, x, 20, new), (w,), check_trace=False)


@pytest.mark.gpu
def test_a_serving_loop(qfa):
    """Prompt, attention with accumulated weights, eviction, decoding on what was kept, with attention on selected blocks: every step against 64 bits on the
    rows that a dictionary of slots says are there."""
    B, H, Hk, D, page, prompt, keep, steps = 2, 4, 2, 64, 16, 120, 48, 20
    g = torch.Generator().manual_seed(11)
    total = prompt + steps
    q, k, v = (torch.randn(B, h, total, D, generator=g).bfloat16() for h in (H, Hk, Hk))
    cos, sin = (t.to(DEV) for t in m.table(total, D))
    cache = qfa.make_paged_cache(40, Hk, page, D, device=DEV)
    bounds = qfa.make_page_bounds(cache)
    order = torch.randperm(40, generator=g).int().to(DEV)
    table, new_table = order[:16].view(B, 8), order[16:26].view(B, 5)
    starts = torch.zeros(B, dtype=torch.int32, device=DEV)
    sm = m.sm_of(D)
    piece = lambda t, a, b: t[:, :, a:b].to(DEV)   # noqa: E731
    turned = lambda t, a, b, at: qfa.norm_rope(piece(t, a, b), None, cos, sin, at)   # noqa: E731
    qr = turned(q, 0, prompt, starts)
    qfa.paged_cache_append(cache, piece(k, 0, prompt), piece(v, 0, prompt), table, starts, cos=cos, sin=sin)
    o, lse = qfa.quant_flash_attn_paged(qr, cache, table, starts, sm_scale=sm, return_lse=True)
    weights = qfa.paged_attention_weights(qr, cache, lse, table, starts, sm_scale=sm)
    rows = [list(t) for t in zip(*qfa.paged_cache_read(cache, table, starts, prompt, dtype=torch.float32))]   # [B] of (k, v) [Hk, n, D]
    kept, weights, lengths = qfa.paged_cache_evict(cache, table, starts + prompt, weights, keep, new_table, first=2, last=16)
    assert (lengths == keep).all() and (kept[..., -16:] == torch.arange(prompt - 16, prompt, device=DEV)).all() and (kept[..., :2] == torch.arange(2, device=DEV)).all()
    rows = [[t.gather(1, kept[b].long()[..., None].expand(-1, -1, D)) for t in rows[b]] for b in range(B)]
    qfa.paged_bounds_update(bounds, cache, new_table, torch.zeros_like(lengths), keep, lengths)
    slots = lengths.clone()
    for t in range(prompt, total):
        at = torch.full((B,), t, dtype=torch.int32, device=DEV)
        qr, kr = turned(q, t, t + 1, at), turned(k, t, t + 1, at)
        qfa.paged_cache_append(cache, kr, piece(v, t, t + 1), new_table, slots)
        qfa.paged_bounds_update(bounds, cache, new_table, slots, 1)
        blocks = qfa.paged_select_blocks(qr, cache, bounds, new_table, slots, 3)
        o = qfa.quant_flash_attn_paged_blocks(qr, cache, new_table, slots, blocks, sm_scale=sm)
        full, lse = qfa.quant_flash_attn_paged(qr, cache, new_table, slots, sm_scale=sm, return_lse=True)
        weights = qfa.paged_attention_weights(qr, cache, lse, new_table, slots, sm_scale=sm, weights=weights, out=weights)
        new = qfa.paged_cache_read(cache, new_table, slots, 1, dtype=torch.float32)
        rows = [[torch.cat([r, n[b]], 1) for r, n in zip(rows[b], new)] for b in range(B)]
        slots += 1
        qh = m.values(*m.quantized(qr.cpu().float()))
        for b in range(B):
            for h in range(H):
                keys, values = (r[h // 2].cpu().double() for r in rows[b])
                inside = torch.zeros(keys.shape[0], dtype=torch.bool)
                for j in blocks[b, h // 2, 0].tolist():
                    inside[j * page:(j + 1) * page] |= j >= 0
                for got, seen in ((full, torch.ones_like(inside)), (o, inside)):
                    want, size = lm.attention_on(qh[b, h, 0], keys, values, seen, sm)
                    assert ((got[b, h, 0].cpu().double() - want).abs() <= m.attention_bound(want, size, torch.bfloat16, keys.shape[0], 0.05)).all(), (t, b, h)
    assert ((weights.double().sum(-1)[:, :, None] > 2 * steps) & (weights.double().sum(-1)[:, :, None] < 2 * total)).all()


@pytest.mark.gpu
def test_weights_that_want_a_gradient(qfa):
    cache = dev(_cache(12, 2, 16, 64, torch.float16, 3))
    table, new = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4), torch.arange(8, 12, dtype=torch.int32, device=DEV).view(2, 2)
    n, w = torch.tensor([60, 30], dtype=torch.int32, device=DEV), torch.rand(2, 2, 64, device=DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        qfa.paged_cache_evict(cache, table, n, w, 20, new)
    with torch.no_grad():
        first = qfa.paged_cache_evict(cache, table, n, w, 20, new)
    for a, b in zip(first, qfa.paged_cache_evict(cache, table, n, w.detach(), 20, new)):
        assert torch.equal(a, b) and not a.requires_grad


def test_argument_errors_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, P = _lib.lib(), 0x1000

    def call(table=P, width=4, lengths=P, weights=P, new=P, new_width=4, kept=P, new_weights=P, new_lengths=P, B=1, keep=20, first=1, last=1, page=16, D=64, ntb=4, H=2):
        c = _lib.PagedCacheStruct(k_codes=P, k_scale=P, k_zero=P, v_codes=P, v_scale=P, v_zero=P, pages=4, H=H, page_size=page, D=D, scale_dtype=1)
        return L.qfa_paged_evict(ctypes.byref(c), table, width, width, 1, lengths, weights, new, new_width, ntb, 1, kept, new_weights, new_lengths, B, keep, first, last,
                                 None)
    for rc, code in ((call(table=None), -1), (call(lengths=None), -1), (call(weights=None), -1), (call(new=None), -1), (call(kept=None), -1),
                     (call(new_weights=None), -1), (call(new_lengths=None), -1), (call(B=0), -1), (call(keep=0), -1), (call(first=10, last=11), -1), (call(first=-1), -1),
                     (call(new_width=1), -1), (call(ntb=-1), -1), (call(page=8), -2), (call(D=32), -2), (call(width=1 << 27), -2), (call(new_width=1 << 27), -2),
                     (call(B=1 << 28, H=4), -2)):
        assert rc == code, L.qfa_last_error()
