"""The log-sum-exp of quant_flash_attn_paged and the attention weights that keys get (paged_attention_weights), against the sums in 64 bits on exactly
the quantized operands, on caches whose other rows hold any codes and scales that are NaN or infinite."""
import ctypes
import math

import pytest
import torch

import long_model as lm
import paged_model as m

DEV = "cuda:0"
dev = lm.dev


def _check(qfa, p, causal=True, prefix=0):
    sm, slots = m.sm_of(p.D), p.width * p.page
    args = (dev(p.q), dev(p.cache), *p.places())
    o, lse = qfa.quant_flash_attn_paged(*args, dev(p.counts), causal=causal, sm_scale=sm, prefix_len=prefix, return_lse=True)
    assert torch.equal(o, qfa.quant_flash_attn_paged(*args, dev(p.counts), causal=causal, sm_scale=sm, prefix_len=prefix))
    lse = lse.cpu()
    want, size = lm.log_sums(p, causal, sm)
    none = want == -math.inf
    assert lse.shape == want.shape and lse.dtype == torch.float32 and torch.equal(lse == -math.inf, none)
    # the scores' roundings (as in weights_bound), the sum of the keys' exponentials (one rounding for each key of a lane and each joined piece, which the
    # logarithm leaves as they are), v_exp and v_log good for 1 ulp, and the result rounded
    log2 = size / math.log(2)
    keys = max([k.shape[1] for k in p.rows[0]] + [1])
    bound = math.log(2) * m.U32 * (4 * log2 + 3 * (log2 + 20)) + (keys / 4 + 20) * m.U32 + 4 * m.U32 * (size + math.log(keys + 1))
    assert ((lse.double() - want)[~none].abs() <= bound).all(), ((lse.double() - want)[~none].abs().max(), bound)
    new = lm.weights_of(p, lse, causal, sm, slots)
    tol = lm.weights_bound(new, size, p.N * p.G + 3)
    w = qfa.paged_attention_weights(*args[:2], dev(lse), *args[2:], dev(p.counts), causal=causal, sm_scale=sm)
    assert w.shape == (p.B, p.Hk, slots) and w.dtype == torch.float32
    excess = (w.cpu().double() - new).abs() - tol
    assert excess.max() <= 0, (excess.max().item(), new.flatten()[excess.argmax()].item())
    # on top of what was there: one multiply-add rounded
    g = torch.Generator().manual_seed(1)
    before = torch.rand(p.B, p.Hk, slots, generator=g)
    for decay in (1.0, 0.5, 0.0):
        out = dev(before)
        same = qfa.paged_attention_weights(*args[:2], dev(lse), *args[2:], dev(p.counts), causal=causal, sm_scale=sm, weights=out, decay=decay, out=out)
        assert same.data_ptr() == out.data_ptr()
        expect = decay * before.double() + new
        assert ((out.cpu().double() - expect).abs() <= tol + m.U32 * expect).all(), decay
        other = qfa.paged_attention_weights(*args[:2], dev(lse), *args[2:], dev(p.counts), causal=causal, sm_scale=sm, weights=dev(before), decay=decay)
        assert torch.equal(out, other)
    assert torch.equal(w, qfa.paged_attention_weights(*args[:2], dev(lse), *args[2:], dev(p.counts), causal=causal, sm_scale=sm, weights=dev(before), decay=0.0,
                                                      out=torch.full_like(w, math.nan)))
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("keys", [[1, 2, 15, 16], [17, 31, 64, 65], [0, 255, 256, 257], [300, 1, 600, 129]])
def test_lengths(qfa, D, page, keys):
    _check(qfa, lm.Problem(4, 2, 2, 1, D, page, keys, seed=D + page))


# a table so wide that keys are not to stay in the caches; pages of all sizes, rows that a block holds and does not
@pytest.mark.gpu
@pytest.mark.parametrize("D,page,H,N,scale_dtype", [(64, 16, 2, 1, torch.float16), (128, 128, 8, 4, torch.float32), (128, 16, 6, 2, torch.bfloat16), (256, 32, 4, 3, torch.float16)])
def test_wide_tables(qfa, D, page, H, N, scale_dtype):
    p = lm.Problem(4, H, 2, N, D, page, [max(N, 1), 700, 257, 530], counts=[N, N, 0, 1], seed=D + page, scale_dtype=scale_dtype)
    width = 330 * 2 ** 20 // (8 * D * page)
    p.table = torch.cat([p.table, torch.full((4, width - p.width), -1, dtype=torch.int32)], 1)
    p.width = width
    _check(qfa, p)


# rows that fill a block, do not, several blocks, several panels of 64
@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,N", [(8, 2, 1), (16, 1, 1), (6, 2, 3), (17, 1, 1), (40, 2, 1), (4, 4, 16), (3, 1, 17), (10, 2, 13), (2, 1, 65)])
@pytest.mark.parametrize("causal", [True, False])
def test_heads_and_tokens(qfa, H, Hk, N, causal):
    _check(qfa, lm.Problem(2, H, Hk, N, 128, 32, [N + 330, N], seed=H + N), causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_types_and_layouts(qfa, dtype, scale_dtype):
    for D, N, layout in ((64, 4, "bhnd"), (128, 9, "bnhd"), (256, 9, "bhnd"), (256, 2, "bnhd")):
        _check(qfa, lm.Problem(2, 6, 3, N, D, 64, [333, 90], dtype=dtype, scale_dtype=scale_dtype, layout=layout, seed=2))


# several steps of a workgroup, and several workgroups; room behind the last key
@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,N,keys,width", [(1, 4, 1, 1, 3000, 400), (70, 8, 8, 1, 120, 40), (300, 4, 4, 1, 40, 130), (2, 4, 1, 6, 1500, 300)])
def test_dealing(qfa, B, H, Hk, N, keys, width):
    _check(qfa, lm.Problem(B, H, Hk, N, 64, 16, [max(N, keys - 17 * (i % 50)) for i in range(B)], width=width, seed=B))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,N", [(4, 5), (8, 33)])
def test_padding(qfa, causal, H, N):
    _check(qfa, lm.Problem(6, H, 2, N, 64, 16, [N + 3, 70, 44, 9, N, 100], counts=[N, 3, 0, 1, N + 9, -3], seed=N), causal)


# rows in blocks of 16, 64 and 128, in one piece and in several; with a prefix pass or without
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,H,Hk,N,keys", [(2, 4, 2, 1, 3000), (1, 8, 1, 5, 700), (2, 4, 1, 40, 500), (1, 2, 2, 150, 400)])
def test_log_sums_of_every_kernel(qfa, D, B, H, Hk, N, keys):
    _check(qfa, lm.Problem(B, H, Hk, N, D, 16, [keys - 31 * i for i in range(B)], seed=N))


@pytest.mark.gpu
def test_log_sums_behind_a_prefix(qfa):
    """With a pass of its own and without: the same rows, so the same sums but for roundings."""
    B, H, Hk, N, D, page, prefix = 64, 32, 8, 1, 128, 16, 6400
    g = torch.Generator().manual_seed(3)
    shared, own = prefix // page, 5
    cache = [t.to(DEV) for t in m.garbage_cache(shared + B * own, Hk, page, D, torch.float16, 1)]
    table = torch.cat([torch.arange(shared).expand(B, shared), shared + torch.arange(B * own).view(B, own)], 1).int().contiguous().to(DEV)
    k, v = (torch.randn(1, Hk, prefix, D, generator=g).bfloat16().to(DEV) for _ in range(2))
    qfa.paged_cache_append(cache, k, v, table[:1].contiguous(), torch.zeros(1, dtype=torch.int32, device=DEV))
    k, v = (torch.randn(B, Hk, own * page, D, generator=g).bfloat16().to(DEV) for _ in range(2))
    starts = torch.full((B,), prefix, dtype=torch.int32, device=DEV)
    qfa.paged_cache_append(cache, k, v, table, starts)
    q = (2 * torch.randn(B, H, N, D, generator=g)).bfloat16().to(DEV)
    at = starts + torch.arange(B, dtype=torch.int32, device=DEV)
    from quant_flash_attn_amd import _lib
    assert _lib.lib().qfa_attn_paged_shared_prefix(B, H, Hk, N, D, prefix) == prefix
    (o0, l0), (o1, l1) = (qfa.quant_flash_attn_paged(q, cache, table, at, prefix_len=n, return_lse=True) for n in (prefix, 0))
    assert torch.equal(o0, qfa.quant_flash_attn_paged(q, cache, table, at, prefix_len=prefix))
    assert (l0 - l1).abs().max() < 1e-4 and l0.abs().max() < 100


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2, 40])
def test_missing_pages(qfa, N):
    """Keys of a page that is none of the cache's get nothing, and the table's width ends them."""
    p = lm.Problem(2, 2, 1, N, 64, 16, [200, 150], seed=3)
    for b, at, bad in ((0, 0, -1), (1, 3, 1 << 30), (0, 12, p.pages)):
        p.table[b, at] = bad
    sm = m.sm_of(64)
    args = (dev(p.q), dev(p.cache), *p.places())
    _, lse = qfa.quant_flash_attn_paged(*args, causal=False, return_lse=True)
    w = qfa.paged_attention_weights(*args[:2], lse, *args[2:], causal=False).cpu().double()
    want = lm.weights_of(p, lse.cpu(), False, sm, p.width * p.page)
    for b, at in ((0, 0), (1, 3), (0, 12)):
        want[b, :, at * 16:at * 16 + 16] = 0
    assert torch.equal(w == 0, want == 0)
    assert ((w - want).abs() <= lm.weights_bound(want, 40.0, 2 * N)).all()
    assert ((w.sum(-1) - p.G * N).abs() < 1e-3 * p.G * N).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 30])
def test_sums_are_the_number_of_rows(qfa, N):
    """Every row's probabilities add up to one."""
    p = lm.Problem(3, 8, 2, N, 128, 16, [900, 333, N], seed=8)
    args = (dev(p.q), dev(p.cache), *p.places())
    _, lse = qfa.quant_flash_attn_paged(*args, return_lse=True)
    w = qfa.paged_attention_weights(*args[:2], lse, *args[2:])
    assert ((w.double().sum(-1) - p.G * N).abs() <= 1e-4 * p.G * N).all() and (w >= 0).all()


@pytest.mark.gpu
def test_positions_outside(qfa):
    p = lm.Problem(3, 4, 2, 6, 64, 16, [50, 6, 20], seed=1)
    starts = torch.tensor([44, -3, -2147483648], dtype=torch.int32)
    args = (dev(p.q), dev(p.cache), dev(p.table), dev(starts))
    o, lse = qfa.quant_flash_attn_paged(*args, return_lse=True)
    assert (lse[1, :, :3] == -math.inf).all() and (lse[2] == -math.inf).all() and torch.isfinite(lse[1, :, 3:]).all()
    w = qfa.paged_attention_weights(*args[:2], lse, *args[2:])
    assert torch.isfinite(w).all() and not w[2].any() and not w[1, :, 3:].any() and ((w[1].sum(-1) - 6).abs() < 1e-4).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 20])
def test_graphs_streams_and_overlap(qfa, N):
    p = lm.Problem(5, 8, 2, N, 128, 16, [500, 80, 300, 66, 120], seed=6)
    args = (dev(p.q), dev(p.cache), *p.places())
    starts, first = args[3], args[3].clone()

    def call():
        _, lse = qfa.quant_flash_attn_paged(*args, return_lse=True)
        return qfa.paged_attention_weights(*args[:2], lse, *args[2:])
    want = call()
    assert torch.equal(want, call())
    side, graphs = torch.cuda.Stream(), []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call()
        graphs.append((graph, o))
    for i in range(3):
        starts.copy_(first - 13 * i)
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
def test_in_place_in_a_graph(qfa):
    """A captured step that adds to the same tensor adds once for every replay, and leaves slots behind the last key."""
    p = lm.Problem(2, 4, 2, 1, 64, 16, [100, 40], seed=6)
    args = (dev(p.q), dev(p.cache), *p.places())
    _, lse = qfa.quant_flash_attn_paged(*args, return_lse=True)
    one = qfa.paged_attention_weights(*args[:2], lse, *args[2:])
    total = torch.full_like(one, 0.25)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qfa.paged_attention_weights(*args[:2], lse, *args[2:], weights=total, out=total)
    expect = torch.full_like(one, 0.25)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        expect = expect + one
        assert ((total - expect).abs() <= 8 * m.U32 * expect).all()
    assert (total[1, :, 48:] == 0.25).all()


@pytest.mark.gpu
def test_traced_with_log_sums(qfa):
    p = lm.Problem(2, 4, 2, 1, 64, 16, [40, 90], seed=9)
    cache, (table, starts) = dev(p.cache), p.places()
    f = lambda q, s: qfa.quant_flash_attn_paged(q, cache, table, s, return_lse=True)   # noqa: E731
    traced = torch.jit.trace(f, (dev(p.q), starts), check_trace=False)
    assert all(torch.equal(a, b) for a, b in zip(traced(dev(p.q), starts - 20), f(dev(p.q), starts - 20)))


@pytest.mark.gpu
def test_refusals(qfa):
    p = lm.Problem(2, 4, 2, 1, 64, 16, [40, 30])
    q, cache, (table, starts) = dev(p.q), dev(p.cache), p.places()
    _, lse = qfa.quant_flash_attn_paged(q, cache, table, starts, return_lse=True)
    w = torch.zeros(2, 2, p.width * 16, device=DEV)
    wide = torch.zeros(2 * 2 * p.width * 16 + 16, device=DEV)

    def refused(error, q=q, lse=lse, **kw):
        with pytest.raises(error):
            qfa.paged_attention_weights(q, cache, lse, table, starts, **kw)
    refused(TypeError, lse=lse.half())
    refused(ValueError, lse=lse[:, :2])
    refused(ValueError, weights=w[..., :-1])
    refused(TypeError, weights=w.double())
    refused(ValueError, out=w[..., 1:])
    refused(ValueError, out=torch.zeros(2, p.width * 16, 2, device=DEV).transpose(1, 2))
    refused(RuntimeError, weights=wide[:w.numel()].view_as(w), out=wide[4:4 + w.numel()].view_as(w))
    refused(ValueError, weights=w, decay=math.inf)
    refused(RuntimeError, sm_scale=-1.0)
    refused(RuntimeError, q=q.float().requires_grad_(True))
    refused(RuntimeError, lse=lse.cpu())
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda x: qfa.paged_attention_weights(x, cache, lse, table, starts), (q,), check_trace=False)


def test_argument_errors_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, P = _lib.lib(), 0x1000

    def struct(page=16, D=64):
        return ctypes.byref(_lib.PagedCacheStruct(k_codes=P, k_scale=P, k_zero=P, v_codes=P, v_scale=P, v_zero=P, pages=4, H=2, page_size=page, D=D, scale_dtype=1))

    def weights(q=P, dt=2, sq=(1024, 512, 64), lse=P, H=4, N=2, B=1, width=4, before=None, decay=1.0, out=P, sm=0.1, ws=None, wsb=0, page=16, D=64):
        return L.qfa_paged_weights(struct(page, D), q, dt, *sq, lse, P, width, width, 1, P, None, before, decay, out, B, H, N, sm, 1, ws, wsb, None)

    def attn(lse=P, o=P, ws=P, wsb=1 << 30, sm=0.1, prefix=0):
        return L.qfa_attn_paged_lse(struct(), P, 2, 1024, 512, 64, P, 4, 4, 1, P, None, o, lse, 1, 4, 2, prefix, sm, 1, ws, wsb, None)
    for rc, code in ((weights(q=None), -1), (weights(dt=9), -1), (weights(sq=(1024, 512, 60)), -1), (weights(lse=None), -1), (weights(H=3), -1), (weights(N=0), -1),
                     (weights(before=P, decay=math.nan), -1), (weights(before=P, decay=math.inf), -1), (weights(out=None), -1), (weights(sm=0.0), -1),
                     (weights(N=40), -1), (weights(N=40, ws=P, wsb=64), -1), (weights(page=40), -2), (weights(D=80), -2), (weights(width=1 << 27), -2),
                     (weights(B=1 << 16, N=1 << 14), -2),
                     (attn(lse=None), -1), (attn(o=None), -1), (attn(ws=None), -1), (attn(wsb=64), -1), (attn(sm=math.inf), -1), (attn(prefix=65), -1)):
        assert rc == code, L.qfa_last_error()
    assert L.qfa_paged_weights_workspace_bytes(2, 8, 2, 4, 64) == 0 and L.qfa_paged_weights_workspace_bytes(2, 8, 2, 5, 64) >= 2 * 8 * 5 * 64
    assert L.qfa_paged_weights_workspace_bytes(2, 8, 3, 5, 64) == 0
    assert L.qfa_attn_paged_lse_workspace_bytes(1, 4, 2, 1, 128, 0) > L.qfa_attn_paged_workspace_bytes(1, 4, 2, 1, 128, 0)
    assert L.qfa_attn_paged_lse_workspace_bytes(1, 4, 3, 1, 128, 0) == 0
