"""paged_bounds_update and paged_select_blocks: bounds, scores and lists bit for bit as the same arithmetic in 64 bits gives them (the queries'
and the bounds' codes from the C oracle), on caches whose other rows hold any codes and scales that are NaN or infinite."""
import ctypes

import pytest
import torch

import long_model as lm
import paged_model as m

DEV = "cuda:0"
dev = lm.dev


def _end(p, b):
    return int(p.starts[b]) + p.tokens[b]


def _expected_bounds(p):
    """Of the pages of every sequence: codes, scale, zero point [blocks, Hk, 2, ...] (nothing for a sequence without keys)."""
    out = []
    for b in range(p.B):
        n = max(0, min(_end(p, b), p.rows[0][b].shape[1]))
        out.append([[lm.bounds_of_page(p.rows[0][b][h, j * p.page:min(n, (j + 1) * p.page)]) for h in range(p.Hk)] for j in range(-(-n // p.page))])
    return out


def _bounds(qfa, p):
    """As a user makes them: whole prompts."""
    cache = dev(p.cache)
    bounds = qfa.make_page_bounds(cache)
    for t in bounds:
        t.fill_(77)
    ends = torch.tensor([max(0, _end(p, b)) for b in range(p.B)], dtype=torch.int32)
    if int(ends.max()) > 0:
        qfa.paged_bounds_update(bounds, cache, dev(p.table), torch.zeros_like(dev(ends)), max(1, int(ends.max())), dev(ends))
    return cache, bounds


def _check_bounds(p, bounds, want):
    written = set()
    for b in range(p.B):
        for j, heads in enumerate(want[b]):
            page = int(p.table[b, j])
            if not 0 <= page < p.pages:
                continue
            written.add(page)
            for h, (c, s, z) in enumerate(heads):
                for got, w, name in zip(bounds, (c, s, z), ("codes", "scale", "zero point")):
                    assert torch.equal(got[page, h].cpu().double(), w.double()), (b, j, h, name)
    rest = [i for i in range(p.pages) if i not in written]
    assert all(bool((t[rest].cpu() == 77).all()) for t in bounds), "a page of nobody's was written"


def _check(qfa, p, keep, first=1, last=1):
    cache, bounds = _bounds(qfa, p)
    want = _expected_bounds(p)
    _check_bounds(p, bounds, want)
    args = (dev(p.q), cache, bounds, *p.places(), keep, dev(p.counts))
    blocks, scores = qfa.paged_select_blocks(*args, first=first, last=last, return_scores=True)
    assert torch.equal(blocks, qfa.paged_select_blocks(*args, first=first, last=last))
    blocks, scores = blocks.cpu(), scores.cpu()
    assert blocks.shape == (p.B, p.Hk, p.N, keep) and scores.shape == (p.B, p.Hk, p.N, p.width)
    for b in range(p.B):
        for h in range(p.Hk):
            there = [j for j in range(len(want[b])) if 0 <= int(p.table[b, j]) < p.pages]
            stack = [torch.stack([want[b][j][h][i] for j in there]) for i in range(3)] if there else None
            for n in range(p.N):
                mine = (int(p.starts[b]) + n) // p.page if n < p.tokens[b] and int(p.starts[b]) + n >= 0 else -1
                candidates = [j for j in there if j <= mine]
                s = torch.full((p.width,), -float("inf"))
                if candidates:
                    s[candidates] = lm.scores_of(p.q[b, h * p.G:(h + 1) * p.G, n], [t[:len(candidates)] for t in stack])
                assert torch.equal(scores[b, h, n], s), (b, h, n)
                assert blocks[b, h, n].tolist() == lm.select(s, candidates, mine, keep, first, last), (b, h, n)


# ends inside a page and a wave's 16 blocks, one key, a sequence without keys
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("keys", [[1, 16, 17], [255, 256, 0], [257, 1025, 900]])
def test_lengths(qfa, D, page, keys):
    _check(qfa, lm.Problem(3, 4, 2, 1, D, page, keys, seed=D + page), keep=5, last=2)


# groups of heads that fill a block of rows, do not, or need several; one token and many
@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,N", [(1, 1, 1), (8, 1, 3), (6, 2, 7), (5, 1, 4), (16, 1, 2), (17, 1, 1), (40, 1, 3), (3, 3, 33), (2, 1, 21)])
def test_heads_and_tokens(qfa, H, Hk, N):
    _check(qfa, lm.Problem(2, H, Hk, N, 64, 16, [N + 150, N + 3], seed=H + N), keep=6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_types(qfa, dtype, scale_dtype):
    for D, layout in ((64, "bhnd"), (128, "bnhd"), (256, "bnhd")):
        _check(qfa, lm.Problem(2, 4, 2, 3, D, 32, [300, 70], dtype=dtype, scale_dtype=scale_dtype, seed=3, layout=layout), keep=4)


# more than there are, all, one; everything forced
@pytest.mark.gpu
@pytest.mark.parametrize("keep,first,last", [(1, 0, 1), (1, 1, 0), (3, 0, 0), (12, 4, 8), (64, 1, 1), (20, 20, 0)])
def test_how_many(qfa, keep, first, last):
    _check(qfa, lm.Problem(3, 4, 2, 2, 64, 16, [700, 40, 330], seed=keep), keep, first, last)


@pytest.mark.gpu
def test_padding_and_missing_pages(qfa):
    p = lm.Problem(5, 4, 2, 4, 64, 16, [300, 90, 44, 200, 120], counts=[4, 2, 0, 9, -1], seed=4)
    p.table[0, 3], p.table[0, 18], p.table[3, 0], p.table[1, 2] = -1, 1 << 30, -7, p.pages
    _check(qfa, p, keep=7, first=2, last=2)


@pytest.mark.gpu
def test_positions_outside(qfa):
    """Before the first key nothing is selected; past the table's end its blocks are all that there is."""
    p = lm.Problem(3, 2, 1, 3, 64, 16, [64, 64, 64], seed=5)
    cache, bounds = _bounds(qfa, p)
    starts = torch.tensor([-2, -2147483648, 2147483645], dtype=torch.int32, device=DEV)
    blocks, scores = qfa.paged_select_blocks(dev(p.q), cache, bounds, dev(p.table), starts, 4, last=2, first=0, return_scores=True)
    blocks, scores = blocks.cpu(), scores.cpu()
    assert (blocks[0, 0, :2] == -1).all() and blocks[0, 0, 2].tolist() == [0, -1, -1, -1] and (blocks[1] == -1).all()
    assert (blocks[2] == torch.arange(4)).all() and torch.isfinite(scores[2]).all() and (scores[1] == -float("inf")).all()
    before = [t.clone() for t in bounds]
    qfa.paged_bounds_update(bounds, cache, dev(p.table), torch.tensor([-40, -2147483648, 2147483645], dtype=torch.int32, device=DEV), 3)
    assert all(torch.equal(a, b) for a, b in zip(before, bounds))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [600, 5000])
def test_long_tables(qfa, width):
    """Ties between equal blocks and the order of thousands of them, several workgroups and steps for a token; room for more than there is."""
    B, Hk, page, D = 2, 1, 16, 64
    g = torch.Generator().manual_seed(width)
    q = torch.randn(B, 2, 1, D, generator=g).bfloat16()
    few = torch.randn(40, Hk, page, D, generator=g)   # 40 different pages, each many times
    pick = torch.randint(0, 40, (width,), generator=g)
    cache = qfa.make_paged_cache(40, Hk, page, D, device=DEV)
    qfa.paged_cache_append(cache, *[few.transpose(0, 1).reshape(1, Hk, -1, D).to(DEV)] * 2, torch.arange(40, dtype=torch.int32, device=DEV)[None],
                           torch.zeros(1, dtype=torch.int32, device=DEV))
    bounds = qfa.make_page_bounds(cache)
    qfa.paged_bounds_update(bounds, cache, torch.arange(40, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV), 40 * page)
    table = pick.int().expand(B, width).contiguous().to(DEV)
    starts = torch.tensor([width * page - 1, (width - 17) * page + 3], dtype=torch.int32, device=DEV)
    keep = 333
    blocks, scores = qfa.paged_select_blocks(q.to(DEV), cache, bounds, table, starts, keep, return_scores=True)
    c, s, z = (t.cpu() for t in bounds)
    for b in range(B):
        mine = int(starts[b]) // page
        one = lm.scores_of(q[b, :, 0], (c[:, 0], s[:, 0], z[:, 0]))[pick]
        one[mine + 1:] = -float("inf")
        assert torch.equal(scores[b, 0, 0].cpu(), one)
        assert blocks[b, 0, 0].tolist() == lm.select(one, list(range(mine + 1)), mine, keep, 1, 1)


# more blocks than are brought to LDS, most of them equal to many others, and more than 2^16 of them taken
@pytest.mark.gpu
@pytest.mark.parametrize("width,keep,pages", [(17001, 64, 40), (140003, 70001, 40), (140003, 5, 2), (140003, 139999, 2)])
def test_more_blocks_than_are_held(qfa, width, keep, pages):
    g = torch.Generator().manual_seed(width + keep)
    page, D = 16, 64
    q = torch.randn(1, 2, 1, D, generator=g).bfloat16()
    cache = qfa.make_paged_cache(pages, 1, page, D, device=DEV)
    rows = torch.randn(1, 1, pages * page, D, generator=g).to(DEV)
    own = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    qfa.paged_cache_append(cache, rows, rows, own, zero)
    bounds = qfa.make_page_bounds(cache)
    qfa.paged_bounds_update(bounds, cache, own, zero, pages * page)
    pick = torch.randint(0, pages, (width,), generator=g)
    starts = torch.tensor([width * page - 9], dtype=torch.int32, device=DEV)
    blocks, scores = qfa.paged_select_blocks(q.to(DEV), cache, bounds, pick.int()[None].to(DEV), starts, keep, last=2, return_scores=True)
    c, s, z = (t.cpu() for t in bounds)
    one = lm.scores_of(q[0, :, 0], (c[:, 0], s[:, 0], z[:, 0]))[pick]
    assert torch.equal(scores[0, 0, 0].cpu(), one)
    rank = one.clone()
    rank[0] = rank[-2:] = float("inf")
    assert torch.equal(blocks[0, 0, 0].cpu(), rank.argsort(descending=True, stable=True)[:keep].sort().values.int())


@pytest.mark.gpu
def test_token_by_token(qfa):
    """Bounds kept up to date behind every append are those of the whole prompt; pages that a call does not touch stay."""
    B, Hk, D, page, steps = 2, 2, 64, 16, 50
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(B, Hk, steps, D, generator=g).bfloat16().to(DEV) for _ in range(2))
    table = torch.randperm(9, generator=g)[:8].int().view(B, 4).to(DEV)
    cache, starts = qfa.make_paged_cache(9, Hk, page, D, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    bounds, whole = qfa.make_page_bounds(cache), qfa.make_page_bounds(cache)
    at = 0
    for n in (1, 1, 14, 1, 20, 5, 1, 7):
        qfa.paged_cache_append(cache, k[:, :, at:at + n], v[:, :, at:at + n], table, starts)
        qfa.paged_bounds_update(bounds, cache, table, starts, n)
        starts += n
        at += n
    qfa.paged_bounds_update(whole, cache, table, torch.zeros_like(starts), steps)
    assert all(torch.equal(a, b) for a, b in zip(bounds, whole)) and bounds[1].abs().max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_queries_that_are_not_finite(qfa, bad):
    """An infinite element makes a row's scale infinite, and its scores (whole numbers times that: zero, or of one sign here) no numbers, which count as the
    least, or infinite: equal either way, and the lowest blocks are taken.  (Over a NaN the quantizer's minimum and maximum pass, so the rest of its
    row still has scores.)  Other rows keep theirs."""
    p = lm.Problem(2, 4, 2, 2, 64, 16, [200, 120], seed=9)
    cache, bounds = _bounds(qfa, p)
    call = lambda q: [t.cpu() for t in qfa.paged_select_blocks(dev(q), cache, bounds, *p.places(), 4, last=1, return_scores=True)]   # noqa: E731
    clean = call(p.q)
    q = p.q.clone()
    q[1, 2:, 1, 3] = bad
    blocks, scores = call(q)
    taken = blocks[1, 1, 1].tolist()
    assert taken[0] == 0 and taken[3] == 7 and taken == sorted(set(taken))
    if bad == bad:
        assert taken == [0, 1, 2, 7]
        assert (scores[1, 1, 1, :8] == (torch.finfo(torch.float32).min if bad > 0 else -bad)).all()
    keep = torch.ones(2, 2, 2, dtype=torch.bool)
    keep[1, 1, 1] = False
    assert torch.equal(blocks[keep], clean[0][keep]) and torch.equal(scores[keep], clean[1][keep])


@pytest.mark.gpu
def test_graphs_streams_and_overlap(qfa):
    p = lm.Problem(6, 8, 2, 2, 128, 16, [500, 80, 300, 66, 120, 900], seed=6)
    cache, bounds = _bounds(qfa, p)
    table, starts = p.places()
    q = dev(p.q)

    def call():
        qfa.paged_bounds_update(bounds, cache, table, starts, 2)
        return qfa.paged_select_blocks(q, cache, bounds, table, starts, 9)
    want = call()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call()
        graphs.append((graph, o))
    first = starts.clone()
    for i in range(3):
        starts.copy_(first - 16 * i)
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
        assert i > 0 or torch.equal(eager, want)


@pytest.mark.gpu
def test_refusals(qfa):
    p = lm.Problem(2, 4, 2, 1, 64, 16, [40, 30])
    cache, bounds = _bounds(qfa, p)
    q, (table, starts) = dev(p.q), p.places()

    def refused(error, q=q, cache=cache, bounds=bounds, table=table, starts=starts, keep=2, **kw):
        with pytest.raises(error):
            qfa.paged_select_blocks(q, cache, bounds, table, starts, keep, **kw)
    refused(ValueError, keep=0)
    refused(ValueError, first=2, last=1)
    refused(ValueError, first=-1)
    refused(ValueError, bounds=[bounds[0][:1], *bounds[1:]])
    refused(TypeError, bounds=[bounds[0], bounds[1].half(), bounds[2]])
    refused(ValueError, bounds=[bounds[0], bounds[1][:1], bounds[2]])
    refused(ValueError, q=q[:, :3])
    refused(TypeError, starts=starts.long())
    refused(TypeError, table=table.long())
    refused(RuntimeError, q=q.cpu())
    refused(RuntimeError, q=q.float().requires_grad_(True))
    with pytest.raises(ValueError):
        qfa.paged_bounds_update(bounds, cache, table, starts, 0)
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda s: qfa.paged_bounds_update(bounds, cache, table, s, 1), (starts,), check_trace=False)


def test_argument_errors_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, P = _lib.lib(), 0x1000
    cache = lambda **kw: ctypes.byref(_lib.PagedCacheStruct(**{**dict(k_codes=P, k_scale=P, k_zero=P, v_codes=P, v_scale=P, v_zero=P, pages=4, H=2,   # noqa: E731
                                                                      page_size=16, D=64, scale_dtype=1), **kw}))
    bounds = lambda c=P, s=P, z=P: ctypes.byref(_lib.PageBoundsStruct(c, s, z))   # noqa: E731

    def update(cache=cache(), bounds=bounds(), table=P, width=4, B=1, N=1):
        return L.qfa_paged_bounds(cache, bounds, table, width, width, 1, P, None, B, N, None)

    def choose(cache=cache(), bounds=bounds(), q=P, dt=2, sq=(1024, 512, 64), width=4, blocks=P, scores=None, B=1, H=4, N=2, keep=2, first=1, last=1, ws=P, wsb=1 << 20):
        return L.qfa_paged_select(cache, bounds, q, dt, *sq, P, width, width, 1, P, None, blocks, scores, B, H, N, keep, first, last, ws, wsb, None)
    for rc, code in ((update(bounds=None), -1), (update(bounds=bounds(c=P + 8)), -1), (update(bounds=bounds(s=P + 4)), -1), (update(bounds=bounds(z=P + 1)), -1),
                     (update(table=None), -1), (update(N=0), -1), (update(cache=cache(page_size=24)), -2), (update(width=1 << 28), -2),
                     (update(B=1 << 28, N=1 << 28), -2),
                     (choose(q=None), -1), (choose(dt=7), -1), (choose(sq=(1024, 512, 60)), -1), (choose(H=3), -1), (choose(blocks=None), -1),
                     (choose(keep=0), -1), (choose(keep=1), -1), (choose(first=-1), -1), (choose(ws=None), -1), (choose(wsb=16), -1), (choose(ws=P + 8), -1),
                     (choose(bounds=bounds(c=None)), -1), (choose(cache=cache(D=96)), -2), (choose(B=1 << 20, N=1 << 20), -2)):
        assert rc == code, L.qfa_last_error()
    size = L.qfa_paged_select_workspace_bytes
    assert size(2, 3, 5, 7) == (2 * 3 * 5 * 7 * 4 + 15) // 16 * 16 and size(0, 1, 1, 1) == 0 and size(1, 1, 1, -1) == 0
