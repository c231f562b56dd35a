"""quant_flash_attn_paged where a call has more than 32 rows (queries times the heads that share a key head): tiles that a workgroup expands once, in
blocks of 64 rows (N = 20 of two heads) and of 128 (N = 70).  The oracle and the bounds are those of the blocks of 16."""
import pytest
import torch

import paged_model as m
from test_paged_attn_gpu import _check, _problem, _with_prefix_pass

DEV = "cuda:0"
ROWS = pytest.mark.parametrize("N", [20, 70])


def _dev(*ts):
    return [None if t is None else [x.to(DEV) for x in t] if isinstance(t, list) else t.to(DEV) for t in ts]


def _within(o, want, size, dtype, keys, v_scale, keep=None):
    excess = (o.cpu().double() - want).abs() - m.attention_bound(want, size, dtype, keys, v_scale)
    if keep is not None:
        o, excess = o[keep.to(o.device)], excess[keep]
    assert torch.isfinite(o).all() and excess.max() <= 0, f"over the bound by {excess.max().item():.3e}"


@pytest.mark.gpu
@ROWS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_types(qfa, N, dtype, scale_dtype, D):
    _check(qfa, 2, 4, 2, N, D, 64, [333, 90], dtype=dtype, scale_dtype=scale_dtype, layout="bnhd" if N == 70 else "bhnd", seed=D)


@pytest.mark.gpu
@ROWS
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_and_pages(qfa, N, page, causal):
    """Ends of quarters, tiles and pages, pages larger than a tile, the shortest sequences that hold their tokens."""
    for keys in ([N, N + 1, 79, 80], [81, 127, 128, 129], [255, 257, 1000, N]):
        _check(qfa, 4, 2, 1, N, 128, page, keys, causal=causal, seed=page)


@pytest.mark.gpu
@ROWS
@pytest.mark.parametrize("size", [1e-4, 1e3])
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float32])
def test_values_of_any_size(qfa, N, size, scale_dtype):
    _check(qfa, 2, 4, 2, N, 128, 32, [700, 141], dtype=torch.float32, scale_dtype=scale_dtype, v_size=size, seed=4)


# one token: the quantizer takes the heads for tokens
@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk", [(48, 1), (160, 2)])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_many_heads_of_one_token(qfa, H, Hk, layout):
    for D in (64, 128, 256):
        _check(qfa, 3, H, Hk, 1, D, 16, [400, 1, 77], dtype=torch.float16, layout=layout, seed=H)


@pytest.mark.gpu
@ROWS
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_padding(qfa, N, causal, D):
    """Fewer tokens than the call has room for, none at all, more."""
    _check(qfa, 6, 4, 2, N, D, 16, [N + 3, 170, 44, 9, N, 100], counts=[N, 3, 0, 1, N + 9, -3], causal=causal, seed=N)


@pytest.mark.gpu
@ROWS
def test_rows_that_see_nothing_are_zero(qfa, N):
    q, cache, table, starts, _, ks, vs, v_scale = _problem(3, 4, 2, N, 128, 16, [N + 44, N, N + 14], seed=1)
    starts = torch.tensor([44, -7, -2147483648], dtype=torch.int32)
    o = qfa.quant_flash_attn_paged(*_dev(q, cache, table, starts))
    assert not o[1, :, :7].any() and not o[2].any() and o[1, :, 7:].abs().amax(-1).min() > 0
    want, size = m.attention(m.values(*m.quantized(q.float())), ks, vs, starts, None, True, m.sm_of(128))
    _within(o, want, size, q.dtype, N + 44, v_scale)


@pytest.mark.gpu
@ROWS
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("bad", [-1, 1 << 30])
def test_pages_that_are_not_there_are_hidden(qfa, N, page, bad):
    """Quarters of a tile and whole tiles; the first, the last, all of a sequence; and the table's width ends the keys."""
    q, cache, table, starts, _, ks, vs, v_scale = _problem(4, 4, 2, N, 64, page, [400, 400, 300, 200], seed=3)
    for b, at in ((0, 0), (1, 3), (1, 399 // page), (2, 2), *((3, i) for i in range(table.shape[1]))):
        table[b, at] = bad
    qh = m.values(*m.quantized(q.float()))
    for width in (table.shape[1], 128 // page):
        there = [[i for i in range(k.shape[1]) if i < width * page and 0 <= int(table[b, i // page]) < cache[0].shape[0]] for b, k in enumerate(ks)]
        o = qfa.quant_flash_attn_paged(*_dev(q, cache, table[:, :width].contiguous(), starts), causal=False)
        want, size = m.attention(qh, [k[:, i] for k, i in zip(ks, there)], [v[:, i] for v, i in zip(vs, there)], starts, None, False, m.sm_of(64))
        assert not o[3].any()
        _within(o, want, size, q.dtype, 400, v_scale)


@pytest.mark.gpu
@ROWS
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_row_that_is_not_finite_stays_alone(qfa, N, value):
    """... over many tiles: it makes the reference of its wave's rows move at every one."""
    q, cache, table, starts, _, ks, vs, v_scale = _problem(2, 4, 2, N, 128, 16, [700, 390], seed=9)
    want, size = m.attention(m.values(*m.quantized(q.float())), ks, vs, starts, None, True, m.sm_of(128))
    q[1, 2, 11, 7] = value
    keep = torch.ones(2, 4, N, dtype=torch.bool)
    keep[1, 2, 11] = False
    _within(qfa.quant_flash_attn_paged(*_dev(q, cache, table, starts)), want, size, q.dtype, 700, v_scale, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_row_that_is_not_finite_stays_alone_among_few(qfa, value):
    """The same in a block of 16, with several tiles for each wave."""
    q, cache, table, starts, _, ks, vs, v_scale = _problem(2, 4, 2, 3, 128, 16, [1500, 390], seed=9)
    want, size = m.attention(m.values(*m.quantized(q.float())), ks, vs, starts, None, True, m.sm_of(128))
    q[1, 2, 1, 7] = q[0, 0, 2, 100] = value
    keep = torch.ones(2, 4, 3, dtype=torch.bool)
    keep[1, 2, 1] = keep[0, 0, 2] = False
    _within(qfa.quant_flash_attn_paged(*_dev(q, cache, table, starts)), want, size, q.dtype, 1500, v_scale, keep)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3, 20, 70])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefix_with_padding_and_short_sequences(qfa, N, causal, D):
    """A pass over the prefix with the rows of all sequences in tiles: sequences that bring nothing, end inside the prefix or have nothing
    behind it, a prefix that ends inside a page and a tile; 72 rows at least."""
    prefix, B = 333, 6
    keys = [prefix + N, prefix + N + 31, prefix + 200, prefix + N, prefix + 300, prefix + 2 * N]
    q, cache, table, _, counts, ks, vs, v_scale = _problem(B, 8, 2, N, D, 32, keys, counts=[N, 2, 0, N, 1, -5], prefix=prefix, seed=8)
    starts = torch.tensor([prefix, prefix + 29, prefix + 200, 50, prefix + 299, -4], dtype=torch.int32)
    o = _with_prefix_pass(*_dev(q, cache, table, starts, counts), causal, m.sm_of(D), prefix)
    want, size = m.attention(m.values(*m.quantized(q.float())), ks, vs, starts, counts, causal, m.sm_of(D))
    _within(o, want, size, q.dtype, max(keys), v_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float32])
def test_prefix_types(qfa, dtype, scale_dtype):
    for D in (64, 128, 256):
        _check(qfa, 9, 4, 1, 3, D, 64, [130 + 3 + 40 * i for i in range(9)], prefix=130, dtype=dtype, scale_dtype=scale_dtype, layout="bnhd", seed=D)


@pytest.mark.gpu
def test_prefix_pages_that_are_not_there(qfa):
    """A page that is missing in the row that the pass reads, sequence 0's, is hidden from all sequences."""
    prefix, N = 192, 3
    q, cache, table, starts, _, ks, vs, v_scale = _problem(6, 8, 2, N, 128, 32, [prefix + N + 20 * i for i in range(6)], prefix=prefix, seed=2)
    table[0, 1] = -1
    there = [i for i in range(prefix) if i // 32 != 1]
    own = [list(range(prefix, k.shape[1])) for k in ks]
    o = _with_prefix_pass(*_dev(q, cache, table, starts), None, False, m.sm_of(128), prefix)
    want, size = m.attention(m.values(*m.quantized(q.float())), [k[:, there + i] for k, i in zip(ks, own)], [v[:, there + i] for v, i in zip(vs, own)], starts, None,
                             False, m.sm_of(128))
    _within(o, want, size, q.dtype, 300, v_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [40, 130])
def test_pages_past_32_bits(qfa, N):
    H, page, D = 8, 64, 128
    pages = (1 << 32) // (H * page * D) + 64
    cache = [torch.empty(pages, H, page, d, dtype=t, device=DEV) for d, t in ((D, torch.int8), (1, torch.float32), (1, torch.int8)) * 2]
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v, q = (torch.randn(2, h, n, D, device=DEV, generator=g).bfloat16() for h, n in ((H, 150), (H, 150), (2 * H, N)))
    near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
    far = torch.tensor([[pages - 1, pages - 2, pages - 9], [pages - 40, pages - 3, pages - 20]], dtype=torch.int32, device=DEV)
    zero, start = torch.zeros(2, dtype=torch.int32, device=DEV), torch.full((2,), 150 - N, dtype=torch.int32, device=DEV)
    out = []
    for t in (near, far):
        qfa.paged_cache_append(cache, k, v, t, zero)
        out.append(qfa.quant_flash_attn_paged(q, cache, t, start))
    assert torch.isfinite(out[0]).all() and torch.equal(*out)


@pytest.mark.gpu
@ROWS
def test_repeats_graphs_and_streams(qfa, N):
    """The same bits every time, from a captured call that follows the lengths and the page table, and on another stream."""
    q, cache, table, starts, *_ = _problem(3, 4, 2, N, 128, 16, [500, N, 300], width=33, seed=6)
    q, cache, table, starts = _dev(q, cache, table, starts)
    first, pages = starts.clone(), table.clone()
    graph = torch.cuda.CUDAGraph()
    qfa.quant_flash_attn_paged(q, cache, table, starts)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o = qfa.quant_flash_attn_paged(q, cache, table, starts)
    side = torch.cuda.Stream()
    for i in range(4):
        starts.copy_(first - 11 * i)
        table.copy_(pages.roll(i, 0))
        o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        eager = qfa.quant_flash_attn_paged(q, cache, table, starts)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = qfa.quant_flash_attn_paged(q, cache, table, starts)
        torch.cuda.synchronize()
        assert torch.equal(o.nan_to_num(7.0), eager.nan_to_num(7.0)) and torch.equal(other.nan_to_num(7.0), eager.nan_to_num(7.0)), f"replay {i}"
