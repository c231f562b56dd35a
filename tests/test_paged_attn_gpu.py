"""quant_flash_attn_paged against attention in 64 bits on exactly the quantized operands (the queries' codes from the C oracle), on
caches whose other rows hold any codes and scales that are NaN or infinite."""
import ctypes

import pytest
import torch

import paged_model as m

DEV = "cuda:0"


def _problem(B, H, Hk, N, D, page, keys, dtype=torch.bfloat16, scale_dtype=torch.float16, counts=None, prefix=0, seed=0, v_size=1.0, width=None, layout="bhnd"):
    """keys: of every sequence, its new tokens included.  Everything on the CPU."""
    g = torch.Generator().manual_seed(seed)
    q = (2 * torch.randn(B, H, N, D, generator=g)).to(dtype)
    if layout == "bnhd":
        q = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    width = width or max(1, -(-max(keys) // page))
    shared = prefix // page
    table, pages = m.shared_pages(B, max(width, shared), shared, seed)
    cache = m.garbage_cache(pages, Hk, page, D, scale_dtype, seed + 1)
    k_off, v_off = torch.randn(Hk, 1, D, generator=g), 0.25 * torch.randn(Hk, 1, D, generator=g)
    ks, vs, v_scale = [], [], 0.0
    first = [torch.randn(Hk, prefix, D, generator=g) for _ in range(2)]
    for b in range(B):
        n = max(keys[b], 0)
        sides = []
        for side, off, size in ((0, k_off, 1.0), (3, v_off, v_size)):
            x = torch.cat([first[side // 3][:, :min(prefix, n)], torch.randn(Hk, max(n - prefix, 0), D, generator=g)], 1)
            c, s, z = m.quantized(((x + off) * size)) if n else (torch.zeros(Hk, 0, D), torch.zeros(Hk, 0, 1), torch.zeros(Hk, 0, 1))
            m.place(cache, table, b, 0, c, s, z, side)
            sides.append(m.values(c, s.to(scale_dtype), z))
            if side and n:
                v_scale = max(v_scale, float(s.max()))
        ks.append(sides[0])
        vs.append(sides[1])
    c = torch.tensor(counts if counts is not None else [N] * B)
    starts = (torch.tensor(keys) - c.clamp(0, N)).int()
    return q, cache, table, starts, None if counts is None else c.int(), ks, vs, v_scale


def _check(qfa, *args, causal=True, **kw):
    prefix = kw.get("prefix", 0)
    q, cache, table, starts, counts, ks, vs, v_scale = _problem(*args, **kw)
    D, sm = q.shape[-1], m.sm_of(q.shape[-1])
    dev = lambda t: None if t is None else t.to(DEV)   # noqa: E731
    call = (dev(q), [dev(t) for t in cache], dev(table), dev(starts), dev(counts))
    out = [qfa.quant_flash_attn_paged(*call, causal=causal, sm_scale=sm, prefix_len=prefix)]
    if prefix:
        out.append(_with_prefix_pass(*call, causal, sm, prefix))
    assert out[0].dtype == q.dtype and out[0].shape == q.shape
    qh = m.values(*m.quantized(q.float()))
    want, size = m.attention(qh, ks, vs, starts, counts, causal, sm)
    keys = max([t.shape[1] for t in ks] + [1])
    bound = m.attention_bound(want, size, q.dtype, keys, v_scale)
    for o in out:
        excess = (o.cpu().double() - want).abs() - bound
        assert torch.isfinite(o).all()
        assert excess.max() <= 0, f"over the bound by {excess.max().item():.3e} at {want.flatten()[excess.argmax()].item():.3e}"
    return out[0]


def _with_prefix_pass(q, cache, table, starts, counts, causal, sm, prefix):
    """The C entry, which gives a prefix a pass of its own whether it pays or not."""
    from quant_flash_attn_amd import _lib
    L, (B, H, N, D), (pages, Hk, page, _) = _lib.lib(), q.shape, cache[0].shape
    c = _lib.PagedCacheStruct(*[t.data_ptr() for t in cache], pages, Hk, page, D, _lib.DTYPE_CODE[cache[1].dtype])
    need = L.qfa_attn_paged_workspace_bytes(B, H, Hk, N, D, prefix)
    ws, o = torch.empty(need, dtype=torch.uint8, device=q.device), torch.full((B, H, N, D), float("nan"), dtype=q.dtype, device=q.device)
    rc = L.qfa_attn_paged(ctypes.byref(c), q.data_ptr(), _lib.DTYPE_CODE[q.dtype], *q.stride()[:3], table.data_ptr(), table.shape[1], *table.stride(),
                          starts.data_ptr(), None if counts is None else counts.data_ptr(), o.data_ptr(), B, H, N, prefix, sm, int(causal), ws.data_ptr(), need,
                          _lib.stream_of(q))
    assert rc == 0, L.qfa_last_error()
    return o


# ends of halves, tiles and pages; one key; a sequence without keys beside others
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("keys", [[1, 2, 15, 16], [17, 31, 32, 33], [0, 63, 64, 65], [127, 129, 300, 1]])
def test_lengths(qfa, D, page, keys):
    _check(qfa, 4, 2, 2, 1, D, page, keys, seed=D + page)


# shared key heads: rows of a block from several queries, several blocks of rows, blocks that are not full
@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,N", [(8, 2, 1), (16, 1, 1), (6, 2, 3), (32, 1, 2), (40, 2, 1), (4, 4, 16), (3, 1, 17), (10, 2, 50), (2, 1, 130)])
@pytest.mark.parametrize("causal", [True, False])
def test_heads_and_queries(qfa, H, Hk, N, causal):
    _check(qfa, 3, H, Hk, N, 128, 32, [N, N + 40, 500], causal=causal, seed=H + N)


# keys of a sequence over several workgroups, and several sequences in one
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,D,keys", [(1, 1, 1, 1, 128, [9000]), (1, 4, 1, 1, 64, [20001]), (2, 2, 2, 3, 256, [4000, 5]), (40, 8, 8, 1, 128, None),
                                             (70, 2, 1, 1, 64, None), (130, 4, 4, 1, 128, None), (3, 8, 2, 20, 128, [2500, 70, 1031])])
def test_dealing(qfa, B, H, Hk, N, D, keys):
    keys = keys or [(37 * i * i) % 700 for i in range(B)]
    _check(qfa, B, H, Hk, N, D, 16, [max(k, N) for k in keys], seed=B)


# every size of a block of rows, for every row size: 16 (one and two blocks), 64, 128 and more
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,H,Hk,N", [(2, 8, 1, 2), (3, 8, 2, 5), (65, 4, 2, 9), (2, 4, 1, 10), (2, 3, 1, 41), (1, 2, 1, 161)])
def test_blocks_of_rows(qfa, D, B, H, Hk, N):
    _check(qfa, B, H, Hk, N, D, 32, [N + (211 * i) % 600 for i in range(B)], seed=D + N)
    _check(qfa, B, H, Hk, N, D, 16, [161 + N + (97 * i) % 300 for i in range(B)], prefix=161, seed=D + N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_types_and_layouts(qfa, dtype, scale_dtype, layout):
    for D in (64, 128, 256):
        _check(qfa, 2, 6, 3, 4, D, 64, [333, 90], dtype=dtype, scale_dtype=scale_dtype, layout=layout, seed=2)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-4, 1e3])
def test_values_of_any_size(qfa, size):
    _check(qfa, 2, 4, 2, 3, 128, 32, [700, 41], dtype=torch.bfloat16, scale_dtype=torch.float32, v_size=size, seed=4)


# fewer tokens than the call has room for, none at all, more; and a start before the first key
@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,N", [(4, 5), (8, 33)])
def test_padding(qfa, causal, H, N):
    _check(qfa, 6, H, 2, N, 128, 16, [N + 3, 70, 44, 9, N, 100], counts=[N, 3, 0, 1, N + 9, -3], causal=causal, seed=N)


@pytest.mark.gpu
def test_rows_that_see_nothing_are_zero(qfa):
    q, cache, table, starts, counts, ks, vs, _ = _problem(3, 4, 2, 6, 128, 16, [50, 6, 20], seed=1)
    starts = torch.tensor([44, -3, -2147483648], dtype=torch.int32)
    o = qfa.quant_flash_attn_paged(q.to(DEV), [t.to(DEV) for t in cache], table.to(DEV), starts.to(DEV)).cpu()
    assert not o[1, :, :3].any() and not o[2].any() and o[1, :, 3:].abs().amax(-1).min() > 0 and torch.isfinite(o).all()
    want, _ = m.attention(m.values(*m.quantized(q.float())), ks, vs, starts, None, True, m.sm_of(128))
    assert (o.double() - want).abs().max() < 2e-2


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 1 << 30])
def test_pages_that_are_not_there_are_hidden(qfa, bad):
    """The keys of a page that is none of the cache's are left out, wherever it stands; the table's width ends the keys."""
    q, cache, table, starts, counts, ks, vs, v_scale = _problem(3, 2, 1, 2, 64, 16, [200, 200, 100], seed=3)
    for b, at in ((0, 0), (1, 3), (1, 12), (2, 6)):
        table[b, at] = bad
    drop = [[i for i in range(k.shape[1]) if 0 <= int(table[b, i // 16]) < cache[0].shape[0]] for b, k in enumerate(ks)]
    o = qfa.quant_flash_attn_paged(q.to(DEV), [t.to(DEV) for t in cache], table.to(DEV), starts.to(DEV), causal=False).cpu()
    qh = m.values(*m.quantized(q.float()))
    want, size = m.attention(qh, [k[:, i] for k, i in zip(ks, drop)], [v[:, i] for v, i in zip(vs, drop)], starts, None, False, m.sm_of(64))
    assert ((o.double() - want).abs() <= m.attention_bound(want, size, q.dtype, 200, v_scale)).all()
    narrow = qfa.quant_flash_attn_paged(q.to(DEV), [t.to(DEV) for t in cache], table[:, :4].contiguous().to(DEV), starts.to(DEV), causal=False).cpu()
    first = [[i for i in d if i < 64] for d in drop]
    want, size = m.attention(qh, [k[:, i] for k, i in zip(ks, first)], [v[:, i] for v, i in zip(vs, first)], starts, None, False, m.sm_of(64))
    assert ((narrow.double() - want).abs() <= m.attention_bound(want, size, q.dtype, 64, v_scale)).all()


# a prefix of whole pages, one that ends inside a page or a tile, one of a single key, rows of all sequences in several blocks
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,D,prefix,page", [(5, 4, 2, 1, 128, 64, 16), (3, 8, 2, 2, 64, 100, 32), (9, 4, 1, 3, 256, 48, 16), (4, 2, 2, 1, 128, 1, 16),
                                                    (33, 4, 4, 1, 128, 2048, 64), (6, 8, 1, 9, 128, 515, 16), (70, 8, 2, 1, 64, 777, 64), (2, 2, 1, 70, 128, 333, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_shared_prefix(qfa, B, H, Hk, N, D, prefix, page, causal):
    _check(qfa, B, H, Hk, N, D, page, [prefix + N + (29 * i) % 150 for i in range(B)], prefix=prefix, causal=causal, seed=B)


@pytest.mark.gpu
def test_prefix_with_padding_and_short_sequences(qfa):
    """Sequences that bring nothing, end inside the prefix (the mask hides the rest of it), or have nothing behind it."""
    prefix = 96
    q, cache, table, starts, counts, ks, vs, v_scale = _problem(5, 4, 2, 3, 128, 16, [99, 130, 120, 99, 300], counts=[3, 2, 0, 3, 1], prefix=prefix, seed=8)
    starts = torch.tensor([96, 128, 120, 50, 299], dtype=torch.int32)
    for causal in (True, False):
        dev = lambda t: t.to(DEV)   # noqa: E731
        o = _with_prefix_pass(dev(q), [dev(t) for t in cache], dev(table), dev(starts), dev(counts), causal, m.sm_of(128), prefix).cpu()
        want, size = m.attention(m.values(*m.quantized(q.float())), ks, vs, starts, counts, causal, m.sm_of(128))
        # (not causal, a sequence that ends inside the prefix sees starts + counts keys all the same)
        assert ((o.double() - want).abs() <= m.attention_bound(want, size, q.dtype, 300, v_scale)).all(), causal


@pytest.mark.gpu
def test_same_as_a_cache_in_one_piece(qfa):
    """The same rows through quant_flash_attn_quantized_kv: the same codes of queries, keys and values, so the difference is that of the
    probabilities' and the outputs' roundings."""
    B, H, N, D, L = 2, 4, 3, 128, 700
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(B, H, n, D, generator=g).bfloat16().to(DEV) for n in (N, L, L))
    cache = qfa.make_paged_cache(2 * 11 + 1, H, 64, D, device=DEV)
    table = torch.randperm(23)[:22].int().view(2, 11).to(DEV)
    qfa.paged_cache_append(cache, k, v, table, torch.zeros(B, dtype=torch.int32, device=DEV))
    starts = torch.full((B,), L - N, dtype=torch.int32, device=DEV)
    o = qfa.quant_flash_attn_paged(q, cache, table, starts)
    want = qfa.quant_flash_attn_quantized_kv(q, k, v, qfa.asymmetric_quant_per_token(k), qfa.asymmetric_quant_per_token(v), True, m.sm_of(D))
    size = qfa.quant_flash_attn_quantized_kv(q, k, v, qfa.asymmetric_quant_per_token(k), qfa.asymmetric_quant_per_token(v.abs()), True, m.sm_of(D)).float()
    assert ((o.float() - want.float()).abs() <= 2 * m.HALF[torch.bfloat16] * want.float().abs() + 2.0 ** -9 * size + 1e-5).all()


@pytest.mark.gpu
def test_a_decoding_loop_follows_the_dense_path(qfa):
    """Norm, rotation, append and attention together, token by token from an empty cache, against the same steps on dense tensors."""
    B, H, Hk, D, page, steps = 3, 4, 2, 64, 16, 40
    g = torch.Generator().manual_seed(5)
    rows = lambda h: torch.randn(B, h, steps, D, generator=g).bfloat16()   # noqa: E731
    q, k, v, (wq, wk) = rows(H), rows(Hk), rows(Hk), (1 + 0.1 * torch.randn(2, D, generator=g)).bfloat16()
    cos, sin = m.table(64, D)
    table, pages = m.shared_pages(B, 4, 0, 3)
    cache, table = qfa.make_paged_cache(pages, Hk, page, D, device=DEV), table.to(DEV)
    dev = lambda t: t.to(DEV)   # noqa: E731
    starts = torch.zeros(B, dtype=torch.int32, device=DEV)
    outs, qs = [], []
    for t in range(steps):
        one = slice(t, t + 1)
        qr = qfa.norm_rope(dev(q[:, :, one]), dev(wq), dev(cos), dev(sin), starts)
        qfa.paged_cache_append(cache, dev(k[:, :, one]), dev(v[:, :, one]), table, starts, k_weight=dev(wk), cos=dev(cos), sin=dev(sin))
        outs.append(qfa.quant_flash_attn_paged(qr, cache, table, starts))
        qs.append(qr)
        starts += 1
    o = torch.cat(outs, 2).cpu().double()
    kh, vh = (t.cpu().double() for t in qfa.paged_cache_read(cache, table, torch.zeros_like(starts), steps, dtype=torch.float32))
    qr = torch.cat(qs, 2)
    assert torch.equal(qr, qfa.norm_rope(dev(q), dev(wq), dev(cos), dev(sin)))
    qh = m.values(*m.quantized(qr.cpu().float()))
    want, size = m.attention(qh, list(kh), list(vh), torch.zeros(B, dtype=torch.int32), None, True, m.sm_of(D))
    assert ((o - want).abs() <= m.attention_bound(want, size, torch.bfloat16, steps, 0.05)).all()
    # the whole prompt in one call gives the same cache, and attention of all its tokens the same rows
    again = qfa.make_paged_cache(pages, Hk, page, D, device=DEV)
    qfa.paged_cache_append(again, dev(k), dev(v), table, torch.zeros_like(starts), k_weight=dev(wk), cos=dev(cos), sin=dev(sin))
    assert all(torch.equal(a, b) for a, b in zip(cache, again))
    full = qfa.quant_flash_attn_paged(qfa.norm_rope(dev(q), dev(wq), dev(cos), dev(sin)), again, table,
                                      torch.zeros_like(starts)).cpu().double()
    assert ((full - o).abs() <= 2 * m.HALF[torch.bfloat16] * o.abs() + 2.0 ** -9 * size + 1e-5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [0, 64])
def test_repeats_and_graphs(qfa, prefix):
    """The same bits every time; a captured call follows the lengths, two captured calls do not share their scratch, another stream."""
    B, H, Hk, N, D, page = 5, 8, 2, 2, 128, 16
    q, cache, table, starts, _, ks, vs, _ = _problem(B, H, Hk, N, D, page, [500, 80, 300, 66, 120], prefix=prefix, seed=6)
    q, table, starts, cache = q.to(DEV), table.to(DEV), starts.to(DEV), [t.to(DEV) for t in cache]
    call = lambda: (_with_prefix_pass(q, cache, table, starts, None, True, m.sm_of(D), prefix) if prefix else   # noqa: E731
                    qfa.quant_flash_attn_paged(q, cache, table, starts))
    want = call()
    assert torch.equal(want, call())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.synchronize()
    assert torch.equal(want, other)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call()
        graphs.append((graph, o))
    first = starts.clone()
    for i in range(4):
        starts.copy_(first - 7 * i if i != 2 else first)
        (g0, o0), (g1, o1) = graphs
        o0.zero_()
        o1.zero_()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        g0.replay()
        with torch.cuda.stream(side):
            g1.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(o0, eager) and torch.equal(o1, eager), f"replay {i}"


@pytest.mark.gpu
def test_two_calls_at_once(qfa):
    """Calls on two streams that overlap, and two captured ones whose replays do, give what each gives alone."""
    made = []
    for B, H, Hk, N, D, keys, prefix in ((40, 8, 2, 1, 128, 700, 300), (2, 4, 4, 150, 64, 1200, 0)):
        q, cache, table, starts, *_ = _problem(B, H, Hk, N, D, 32, [keys - i for i in range(B)], prefix=prefix, seed=B)
        args = (q.to(DEV), [t.to(DEV) for t in cache], table.to(DEV), starts.to(DEV))
        made.append(lambda args=args, prefix=prefix: _with_prefix_pass(*args, None, True, 0.1, prefix))
    want = [f().clone() for f in made]
    streams = [torch.cuda.Stream() for _ in made]
    graphs = [torch.cuda.CUDAGraph() for _ in made]
    torch.cuda.synchronize()
    for i in range(3):
        got = []
        for f, st in zip(made, streams):
            with torch.cuda.stream(st):
                got.append([f() for _ in range(5)])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for os, w in zip(got, want) for o in os), i
    outs = []
    for f, g in zip(made, graphs):
        with torch.cuda.graph(g):
            outs.append(f())
    for i in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), f"replay {i}"


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_call_that_may_reach_a_large_cache(qfa, D):
    """... reads it with other hints: the same bits whatever room the page table has."""
    B, H, page = 8, 16, 64
    pages = (400 << 20) // (2 * H * page * D)
    q, small, table, starts, *_ = _problem(B, H, H, 1, D, page, [700 - 60 * i for i in range(B)], seed=D)
    cache = [torch.zeros(pages, *t.shape[1:], dtype=t.dtype, device=DEV) for t in small]
    for c, t in zip(cache, small):
        c[:t.shape[0]] = t.to(DEV)
    wide = torch.zeros(B, -(-pages // B), dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table.to(DEV)
    q, table, starts = q.to(DEV), table.to(DEV), starts.to(DEV)
    assert torch.equal(qfa.quant_flash_attn_paged(q, cache, wide, starts), qfa.quant_flash_attn_paged(q, [t.to(DEV) for t in small], table, starts))


@pytest.mark.gpu
def test_pages_past_32_bits(qfa):
    H, page, D = 8, 64, 128
    pages = (1 << 32) // (H * page * D) + 64
    cache = [torch.empty(pages, H, page, d, dtype=t, device=DEV) for d, t in ((D, torch.int8), (1, torch.float32), (1, torch.int8)) * 2]
    k, v, q = (torch.randn(2, H, n, D, device=DEV).bfloat16() for n in (150, 150, 1))
    near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
    far = torch.tensor([[pages - 1, pages - 2, pages - 9], [pages - 40, pages - 3, pages - 20]], dtype=torch.int32, device=DEV)
    zero, last = torch.zeros(2, dtype=torch.int32, device=DEV), torch.full((2,), 149, dtype=torch.int32, device=DEV)
    out = []
    for t in (near, far):
        qfa.paged_cache_append(cache, k, v, t, zero)
        out.append(qfa.quant_flash_attn_paged(q, cache, t, last))
    assert torch.equal(*out)


@pytest.mark.gpu
def test_a_row_that_is_not_finite_stays_alone(qfa):
    q, cache, table, starts, *_ = _problem(2, 4, 2, 3, 128, 16, [40, 90], seed=9)
    call = lambda x: qfa.quant_flash_attn_paged(x.to(DEV), [t.to(DEV) for t in cache], table.to(DEV), starts.to(DEV)).cpu()   # noqa: E731
    clean = call(q)
    q[1, 2, 1, 7] = float("nan")
    o = call(q)
    keep = torch.ones(2, 4, 3, dtype=torch.bool)
    keep[1, 2, 1] = False
    assert torch.equal(o[keep], clean[keep])


@pytest.mark.gpu
def test_traced(qfa):
    q, cache, table, starts, *_ = _problem(2, 4, 2, 1, 64, 16, [40, 90], seed=9)
    cache, table = [t.to(DEV) for t in cache], table.to(DEV)
    f = lambda q, s: qfa.quant_flash_attn_paged(q, cache, table, s)   # noqa: E731
    traced = torch.jit.trace(f, (q.to(DEV), starts.to(DEV)), check_trace=False)
    shorter = (starts - 20).to(DEV)
    assert torch.equal(traced(q.to(DEV), shorter), f(q.to(DEV), shorter))


def test_argument_errors_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, p = _lib.lib(), 0x1000

    def call(q=p, dt=2, sq=(1024, 512, 64), H=4, N=2, B=1, width=4, prefix=0, sm=0.1, ws=p, wsb=1 << 30, page=16, D=64):
        c = _lib.PagedCacheStruct(k_codes=p, k_scale=p, k_zero=p, v_codes=p, v_scale=p, v_zero=p, pages=4, H=2, page_size=page, D=D, scale_dtype=1)
        return L.qfa_attn_paged(ctypes.byref(c), q, dt, *sq, p, width, width, 1, p, None, p, B, H, N, prefix, sm, 1, ws, wsb, None)
    for rc, code, what in ((call(q=None), -1, b"null"), (call(dt=9), -1, b"q_dtype"), (call(sq=(1024, 512, 60)), -1, b"strides"), (call(H=3), -1, b"multiple"),
                           (call(N=0), -1, b"positive"), (call(sm=0.0), -1, b"sm_scale"), (call(sm=float("inf")), -1, b"sm_scale"),
                           (call(prefix=65), -1, b"prefix"), (call(prefix=-1), -1, b"prefix"), (call(ws=None), -1, b"workspace"), (call(wsb=64), -1, b"workspace"),
                           (call(page=48), -2, b"page size"), (call(D=96), -2, b"head_dim"), (call(B=1 << 20, width=1 << 20), -2, b"too many")):
        assert rc == code, (rc, code, what)
    assert call(q=None) == -1 and b"null" in L.qfa_last_error()
    ws = L.qfa_attn_paged_workspace_bytes
    share = L.qfa_attn_paged_shared_prefix
    assert share(64, 32, 8, 1, 128, 16384) == 16384 and share(64, 32, 8, 1, 128, 100) == 0 and share(1, 32, 8, 1, 128, 16384) == 0
    assert share(64, 32, 8, 1, 96, 16384) == 0 and share(64, 32, 7, 1, 128, 16384) == 0 and share(64, 32, 8, 300, 128, 400) == 0
    assert ws(1, 4, 2, 1, 128, 0) > 0 and ws(1, 4, 2, 1, 96, 0) == 0 and ws(1, 4, 3, 1, 128, 0) == 0 and ws(8, 4, 2, 1, 128, 5) > 2 * ws(8, 4, 2, 1, 128, 0)


@pytest.mark.gpu
def test_refusals(qfa):
    q, cache, table, starts, *_ = _problem(1, 4, 2, 1, 64, 16, [40], seed=9)
    q, cache, table, starts = q.to(DEV), [t.to(DEV) for t in cache], table.to(DEV), starts.to(DEV)
    with pytest.raises(RuntimeError, match="no gradient"):
        qfa.quant_flash_attn_paged(q.clone().requires_grad_(True), cache, table, starts)
    with pytest.raises(ValueError, match="shape"):
        qfa.quant_flash_attn_paged(q[:, :3], cache, table, starts)
    with pytest.raises(ValueError, match="prefix_len"):
        qfa.quant_flash_attn_paged(q, cache, table, starts, prefix_len=1000)
    with pytest.raises(RuntimeError, match="sm_scale"):
        qfa.quant_flash_attn_paged(q, cache, table, starts, sm_scale=-1.0)
    with pytest.raises(TypeError, match="starts"):
        qfa.quant_flash_attn_paged(q, cache, table, starts.long())
