"""Bounds of pages hold what lies in the page: rows of one sign too, which the least and the largest keys of a page often are."""
import ctypes

import pytest
import torch

import bounds_model as bm
import long_model as lm
import paged_model as m

DEV = "cuda:0"
dev = lm.dev

# ranges of codes and of zero points of the keys, with what their rows become
KEYS = {
    "zero mean": (-128, 128, -20, 21),         # many rows, so that least ones are all negative and largest ones all positive
    "positive": (-100, 128, -128, -127),
    "negative": (-128, 100, 127, 128),
    "far positive": (60, 128, -128, -127),     # less than a quarter of the largest apart
    "far negative": (-128, -60, 127, 128),
    "constant": (90, 91, -128, -127),
    "zeros": (5, 6, 5, 6),
}


def _cache(kind, pages, Hk, page, D, scale_dtype, seed, size=0.02):
    """Keys of that kind; scales differ by a factor of two at most.  Values: anything."""
    g = torch.Generator().manual_seed(seed)
    c0, c1, z0, z1 = KEYS[kind]
    out = []
    for _ in range(2):
        codes = torch.randint(c0, c1, (pages, Hk, page, D), generator=g).to(torch.int8)
        if kind == "zero mean":   # spread like a bell
            codes = (30 * torch.randn(pages, Hk, page, D, generator=g)).round().clamp(-128, 127).to(torch.int8)
        out += [codes, (size * (1 + torch.rand(pages, Hk, page, 1, generator=g))).to(scale_dtype),
                torch.randint(z0, z1, (pages, Hk, page, 1), generator=g).to(torch.int8)]
    return out


def _keys(cache):
    """As the kernels see them: the product with the scale rounded to 32 bits."""
    c, s, z = cache[:3]
    return (c.float() - z.float()) * s.float()


# No GPU: the arithmetic itself.  What the rows stand for, against the least and the largest keys
@pytest.mark.parametrize("kind", list(KEYS))
@pytest.mark.parametrize("page", [1, 16, 64, 256])
def test_rows_stand_for_the_extremes(kind, page):
    rows = bm.extremes(_keys(_cache(kind, 6, 3, page, 64, torch.float32, page)))
    codes, scale, zero = bm.bound_rows(rows)
    assert ((bm.values(codes, scale, zero) - rows.double()).abs() <= bm.HALF_STEP * scale.double()).all()
    both = ((rows.amin(-1) <= 0) & (rows.amax(-1) >= 0)).unsqueeze(-1)
    token = m.quantized(rows)
    for a, b in zip((codes, scale, zero), token):   # rows with both signs: a token's arithmetic
        assert torch.equal(a.double()[both.expand_as(a)], b.double()[both.expand_as(b)])
    if page > 16 and kind not in ("zeros", "constant"):   # the others are why it is not a token's (which gives a constant row a step of 1)
        assert not both.all() and ((m.values(*token) - rows.double()).abs() > 2 * token[1].double()).any()


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_rows_of_any_size(scale):
    rows = bm.extremes(_keys(_cache("zero mean", 6, 3, 128, 64, torch.float32, 1)).double() * scale)
    assert ((bm.values(*bm.bound_rows(rows)) - rows.double()).abs() <= bm.HALF_STEP * bm.bound_rows(rows)[1].double()).all()


def _problem(kind, D, page, Hk, G, N, scale_dtype, dtype, query, seed, blocks=24):
    g = torch.Generator().manual_seed(seed)
    cache = _cache(kind, blocks + 2, Hk, page, D, scale_dtype, seed)
    table = torch.randperm(blocks + 2, generator=g)[:blocks].int()[None]
    q = torch.randn(1, Hk * G, N, D, generator=g)
    if query == "one channel":
        q[..., 5] *= 200
    return cache, table, q.to(dtype), torch.tensor([blocks * page - N - 3], dtype=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KEYS))
@pytest.mark.parametrize("D,page,scale_dtype,G,N,query", [(64, 64, torch.float16, 2, 1, "spread"), (128, 128, torch.float32, 4, 3, "one channel"),
                                                          (256, 16, torch.bfloat16, 8, 9, "spread"), (64, 256, torch.float32, 1, 20, "one channel")])
def test_bounds_and_scores(qfa, kind, D, page, scale_dtype, G, N, query):
    """Bit for bit the model's rows, and scores of those; no key of a block has a larger product than its score, but for half a step of the codes."""
    Hk, dtype = 2, torch.float32 if G == 1 else torch.bfloat16
    cache, table, q, starts = _problem(kind, D, page, Hk, G, N, scale_dtype, dtype, query, D + page)
    end, blocks = int(starts[0]) + N, table.shape[1]
    on = dev(cache)
    bounds = qfa.make_page_bounds(on)
    qfa.paged_bounds_update(bounds, on, dev(table), torch.zeros(1, dtype=torch.int32, device=DEV), end)
    keep = 5
    lists, scores = (t.cpu() for t in qfa.paged_select_blocks(dev(q), on, bounds, dev(table), dev(starts), keep, return_scores=True))
    got = [t.cpu() for t in bounds]
    keys = _keys(cache)[table[0].long()]   # [blocks, Hk, page, D]
    qc, qs, qz = m.quantized(q.float())
    e = qc.double() - qz.double()
    for h in range(Hk):
        rows, products = [], []
        for j in range(blocks):
            k = keys[j, h, :min(page, end - j * page)]
            want = bm.bound_rows(bm.extremes(k))
            at = int(table[0, j])
            assert all(torch.equal(t[at, h].double(), w.double()) for t, w in zip(got, want)), (j, h)
            rows.append(want)
            products.append(torch.einsum("gnd,kd->gnk", e[0, h * G:(h + 1) * G], k.double()).amax(-1) * qs.double()[0, h * G:(h + 1) * G, :, 0])
        stack = [torch.stack([r[i] for r in rows]) for i in range(3)]
        for n in range(N):
            mine = (int(starts[0]) + n) // page
            s = lm.scores_of(q[0, h * G:(h + 1) * G, n], stack)
            s[mine + 1:] = -float("inf")
            assert torch.equal(scores[0, h, n], s)
            assert lists[0, h, n].tolist() == lm.select(s, list(range(mine + 1)), mine, keep, 1, 1)
            slack = torch.stack([(e[0, h * G:(h + 1) * G, n].clamp_min(0) * stack[1][j, 1].double() - e[0, h * G:(h + 1) * G, n].clamp_max(0) * stack[1][j, 0].double()).sum(-1)
                                 * qs.double()[0, h * G:(h + 1) * G, n, 0] for j in range(mine + 1)]).amax(-1) * bm.HALF_STEP
            most = torch.stack([p[:, n].amax(0) for p in products[:mine + 1]])
            assert (s[:mine + 1].double() >= most - slack - 2 * m.U32 * most.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["zero mean", "far negative"])
@pytest.mark.parametrize("G,N,width", [(1, 1, 20), (4, 1, 1100), (8, 3, 20), (3, 7, 300)])
def test_zero_points_of_8_bits(qfa, kind, G, N, width):
    """Bounds that a caller holds with int8 zero points: rows as the token quantizer makes them, and scores of what they stand for."""
    D, page, Hk, pages = 64, 64, 2, 20
    g = torch.Generator().manual_seed(G)
    cache = _cache(kind, pages, Hk, page, D, torch.float32, G)
    on = dev(cache)
    made = qfa.make_page_bounds(on)
    bounds = (made.codes, made.scale, made.zero_point.to(torch.int8))
    own = torch.arange(pages, dtype=torch.int32)[None]
    qfa.paged_bounds_update(bounds, on, dev(own), torch.zeros(1, dtype=torch.int32, device=DEV), pages * page)
    want = m.quantized(bm.extremes(_keys(cache)))
    assert all(torch.equal(t.cpu().double(), w.double()) for t, w in zip(bounds, want))
    q = torch.randn(1, Hk * G, N, D, generator=g).bfloat16()
    pick = torch.randint(0, pages, (width,), generator=g)
    starts = torch.tensor([width * page - N], dtype=torch.int32)
    _, scores = qfa.paged_select_blocks(dev(q), on, bounds, dev(pick.int()[None]), dev(starts), 4, return_scores=True)
    for h in range(Hk):
        for n in range(N):
            assert torch.equal(scores[0, h, n].cpu(), lm.scores_of(q[0, h * G:(h + 1) * G, n], [t[:, h] for t in want])[pick])


@pytest.mark.gpu
def test_refusals(qfa):
    cache = dev(_cache("zero mean", 4, 2, 16, 64, torch.float16, 0))
    bounds = qfa.make_page_bounds(cache)
    assert bounds.zero_point.dtype == torch.int16
    table, zero = torch.arange(4, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError):
        qfa.paged_bounds_update((bounds.codes, bounds.scale, bounds.zero_point.int()), cache, table, zero, 5)


def test_argument_errors_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, P = _lib.lib(), 0x1000
    cache = _lib.PagedCacheStruct(k_codes=P, k_scale=P, k_zero=P, v_codes=P, v_scale=P, v_zero=P, pages=4, H=2, page_size=16, D=64, scale_dtype=1)
    for codes, scale, zero, eight in ((P, P, P + 2, False), (P, P, P + 1, True), (P, P + 4, P, False), (P + 8, P, P, False), (P, P, None, False), (None, P, P, True)):
        for update, select in ((L.qfa_paged_bounds, L.qfa_paged_select), (L.qfa_paged_bounds16, L.qfa_paged_select16))[not eight:]:
            bounds = ctypes.byref(_lib.PageBoundsStruct(codes, scale, zero))
            assert update(ctypes.byref(cache), bounds, P, 4, 4, 1, P, None, 1, 1, None) == -1, (codes, scale, zero)
            assert select(ctypes.byref(cache), bounds, P, 2, 1024, 512, 64, P, 4, 4, 1, P, None, P, None, 1, 4, 2, 2, 1, 1, P, 1 << 20, None) == -1
    assert L.qfa_paged_bounds16(ctypes.byref(cache), None, P, 4, 4, 1, P, None, 1, 1, None) == -1
