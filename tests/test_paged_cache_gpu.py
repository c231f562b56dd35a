"""paged_cache_append and paged_cache_read: what is written, where, and that nothing else is."""
import ctypes

import pytest
import torch

import paged_model as m

DEV = "cuda:0"
EPS = 1e-6


def _gpu(ts):
    return [t.to(DEV) for t in ts]


def _filled(pages, H, page, D, scale_dtype, seed):
    """A cache whose every byte is known (finite, so that it can be compared)."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        out += [torch.randint(-128, 128, (pages, H, page, D), generator=g).to(torch.int8), torch.rand(pages, H, page, 1, generator=g).to(scale_dtype),
                torch.randint(-128, 128, (pages, H, page, 1), generator=g).to(torch.int8)]
    return out


def _case(qfa, B, H, N, D, page, starts, counts=None, dtype=torch.bfloat16, scale_dtype=torch.float16, R=None, interleaved=False, weight=None, seed=0,
          layout="bhnd", width=None, hole=None, rope_rows=None):
    g = torch.Generator().manual_seed(seed)
    R = D if R is None else R

    def rows():
        x = (torch.randn(B, H, N, D, generator=g) * 2 + torch.randn(1, H, 1, D, generator=g)).to(dtype)
        return x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) if layout == "bnhd" else x
    k, v = rows(), rows()
    w = {"shared": (1 + 0.2 * torch.randn(D, generator=g)).to(dtype), "heads": 1 + 0.2 * torch.randn(H, D, generator=g)}.get(weight)
    width = width or max(1, -(-(max(starts) + N) // page))
    table, pages = m.shared_pages(B, width, 0, seed)
    if hole:
        table[hole[0], hole[1]] = hole[2]
    rope_rows = rope_rows or width * page
    cos, sin = m.table(rope_rows, R) if R else (None, None)
    before = _filled(pages, H, page, D, scale_dtype, seed + 1)
    cache = _gpu(before)
    s, c = torch.tensor(starts, dtype=torch.int32), None if counts is None else torch.tensor(counts, dtype=torch.int32)
    dev = lambda t: None if t is None else t.to(DEV)   # noqa: E731
    qfa.paged_cache_append(cache, dev(k), dev(v), dev(table), dev(s), dev(c), k_weight=dev(w), cos=dev(cos), sin=dev(sin), interleaved=interleaved, eps=EPS)
    back = qfa.paged_cache_read(cache, dev(table), dev(s), N, dev(c), dtype=dtype)
    got = [t.cpu() for t in cache]
    # ---- what has to be there
    want = [t.clone() for t in before]
    exact = w is None   # norms in fp32 may round otherwise: those rows are compared as values
    place = [(b, n, starts[b] + n) for b in range(B) for n in range(N if counts is None else min(N, counts[b]))]
    place = [(b, n, p) for b, n, p in place if 0 <= p < width * page and 0 <= int(table[b, p // page]) < pages]
    mask = torch.zeros(pages, page, dtype=torch.bool)
    written = [(b, n, p) for b, n, p in place if not R or p < rope_rows]
    sides = [(0, k), (3, v)]
    for side, x in sides:
        y = x.float()
        if side == 0:
            if w is not None:
                ww = w.float()
                y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * (ww[:, None] if ww.dim() == 2 else ww)
            if R:
                at = (s[:, None].long() + torch.arange(N)).clamp(0, rope_rows - 1)
                y, _ = m.turn(y, cos[at], sin[at], interleaved)   # fp32, each operation rounded by itself
        codes, scale, zero = m.quantized(y)
        for b, n, p in written:
            pg, row = int(table[b, p // page]), p % page
            mask[pg, row] = True
            if side == 3 or exact:
                want[side][pg, :, row], want[side + 1][pg, :, row], want[side + 2][pg, :, row] = codes[b, :, n], scale[b, :, n].to(scale_dtype), zero[b, :, n]
            else:
                # one code more or less where the norm rounds otherwise, with the scale's own rounding; half a unit of the range at its ends
                a = m.values(got[0][pg, :, row], got[1][pg, :, row], got[2][pg, :, row])
                assert ((a - y[b, :, n].double()).abs() <= 1.2 * scale[b, :, n].double()).all()
                for i in range(3):
                    want[i][pg, :, row] = got[i][pg, :, row]
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), f"tensor {i}: {int((a != b).sum())} values differ"
    # ---- read back
    for side, x in zip((0, 3), back):
        y = torch.zeros(B, H, N, D, dtype=torch.float64)
        for b, n, p in place:
            pg, row = int(table[b, p // page]), p % page
            y[b, :, n] = m.values(got[side][pg, :, row], got[side + 1][pg, :, row], got[side + 2][pg, :, row])
        assert x.dtype == dtype and ((x.cpu().double() - y).abs() <= (m.HALF[dtype] + 2 * m.U32) * y.abs() + m.TINY[dtype]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_types(qfa, D, dtype, scale_dtype):
    _case(qfa, 2, 3, 21, D, 16, [0, 13], dtype=dtype, scale_dtype=scale_dtype, interleaved=D == 128, seed=D)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("N,starts", [(1, [0, 15, 16, 63, 500]), (5, [14, 0, 60, 255, 254]), (300, [1, 0, 200, 16, 31])])
def test_pages_and_positions(qfa, page, N, starts):
    _case(qfa, 5, 2, N, 128, page, starts, seed=page + N)


@pytest.mark.gpu
@pytest.mark.parametrize("weight", ["shared", "heads"])
@pytest.mark.parametrize("R,interleaved", [(0, False), (64, False), (64, True), (128, False)])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_norm_and_partial_rotation(qfa, weight, R, interleaved, layout):
    _case(qfa, 3, 4, 33, 128, 32, [0, 7, 90], R=R, interleaved=interleaved, weight=weight, layout=layout, seed=R)


@pytest.mark.gpu
def test_many_heads_and_tokens(qfa):
    _case(qfa, 2, 37, 700, 64, 64, [5, 130], seed=3)


# padding behind a sequence, none of it, too many; positions before the first and past the last page; a page that is not there; past the angles
@pytest.mark.gpu
@pytest.mark.parametrize("counts,starts,width,hole,rope_rows", [([3, 0, 40, -2], [1, 2, 3, 4], None, None, None), (None, [-5, 0, 40, 47], 3, None, None),
                                                               (None, [0, 1, 2, 3], None, (1, 0, -1), None), (None, [0, 1, 2, 3], None, (2, 1, 1 << 30), None),
                                                               (None, [-2147483648, 2147483647, 0, 1], 4, None, None)])
def test_tokens_without_a_place(qfa, counts, starts, width, hole, rope_rows):
    _case(qfa, 4, 2, 30, 64, 16, starts, counts, width=width or 4, hole=hole, rope_rows=rope_rows, seed=5)


@pytest.mark.gpu
def test_tokens_past_the_angles_are_not_written(qfa):
    """... neither their keys nor their values."""
    _case(qfa, 2, 2, 30, 64, 16, [0, 10], width=4, rope_rows=20, seed=6)


@pytest.mark.gpu
def test_rows_past_32_bits(qfa):
    """Codes and scales beyond 2^31 bytes and elements."""
    H, page, D = 8, 64, 128
    pages = (1 << 32) // (H * page * D) + 64
    cache = [torch.empty(pages, H, page, d, dtype=t, device=DEV) for d, t in ((D, torch.int8), (1, torch.float32), (1, torch.int8)) * 2]
    x = torch.randn(2, H, 20, D, device=DEV).half()
    table = torch.tensor([[pages - 1, 0], [pages - 2, pages - 40]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([50, 60], dtype=torch.int32, device=DEV)
    qfa.paged_cache_append(cache, x, -x, table, starts)
    codes, scale, zero = qfa.asymmetric_quant_per_token(x, torch.float32)
    for b in range(2):
        for n in range(20):
            p = int(starts[b]) + n
            pg = int(table[b, p // page])
            assert torch.equal(cache[0][pg, :, p % page], codes[b, :, n]) and torch.equal(cache[1][pg, :, p % page], scale[b, :, n])
    k, v = qfa.paged_cache_read(cache, table, starts, 20, dtype=torch.float32)
    assert torch.equal(k, qfa.dequantize_per_token(codes, scale, zero))


@pytest.mark.gpu
def test_one_large_call_is_many_small_ones(qfa):
    """What outgrows the last-level cache is loaded with other hints."""
    B, H, N, D, page = 4, 32, 2800, 128, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(B, H, N, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    cos, sin = (t.to(DEV) for t in m.table(N, D))
    width = -(-N // page)
    table, zero = torch.arange(B * width, device=DEV, dtype=torch.int32).reshape(B, width), torch.zeros(B, dtype=torch.int32, device=DEV)
    for interleaved in (False, True):
        whole, parts = (qfa.make_paged_cache(B * width, H, page, D) for _ in range(2))
        qfa.paged_cache_append(whole, k, v, table, zero, cos=cos, sin=sin, interleaved=interleaved)
        for b in range(B):
            qfa.paged_cache_append(parts, k[b:b + 1], v[b:b + 1], table[b:b + 1], zero[:1], cos=cos, sin=sin, interleaved=interleaved)
        assert all(torch.equal(a, b) for a, b in zip(whole, parts))
    rows = qfa.paged_cache_read(whole, table, zero, N)
    for b in range(B):
        assert all(torch.equal(r[b:b + 1], x) for r, x in zip(rows, qfa.paged_cache_read(whole, table[b:b + 1], zero[:1], N)))


@pytest.mark.gpu
def test_graph_follows_the_lengths(qfa):
    B, H, N, D, page = 3, 2, 2, 64, 16
    table, pages = m.shared_pages(B, 4, 0, 1)
    cache, again = qfa.make_paged_cache(pages, H, page, D, device=DEV), qfa.make_paged_cache(pages, H, page, D, device=DEV)
    table = table.to(DEV)
    k, v = (torch.zeros(B, H, N, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    starts = torch.zeros(B, dtype=torch.int32, device=DEV)
    cos, sin = _gpu(m.table(64, D))
    for c in (cache, again):
        qfa.paged_cache_append(c, k, v, table, starts, cos=cos, sin=sin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qfa.paged_cache_append(cache, k, v, table, starts, cos=cos, sin=sin)
    for i in range(6):
        k.normal_()
        v.normal_()
        starts.copy_(torch.tensor([2 * i, 3 * i, 30 + i], dtype=torch.int32))
        graph.replay()
        qfa.paged_cache_append(again, k, v, table, starts, cos=cos, sin=sin)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cache, again)), f"replay {i}"


@pytest.mark.gpu
def test_another_stream(qfa):
    B, H, N, D, page = 2, 2, 40, 128, 32
    table, pages = m.shared_pages(B, 2, 0, 1)
    x = torch.randn(B, H, N, D, device=DEV).bfloat16()
    starts = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    a, b = (qfa.make_paged_cache(pages, H, page, D, device=DEV) for _ in range(2))
    qfa.paged_cache_append(a, x, x, table.to(DEV), starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qfa.paged_cache_append(b, x, x, table.to(DEV), starts)
        read = qfa.paged_cache_read(b, table.to(DEV), starts, N)
    torch.cuda.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(a, b)) and torch.equal(read[0], qfa.paged_cache_read(a, table.to(DEV), starts, N)[0])


def _abi_cache(_lib, **change):
    f = dict(k_codes=0x1000, k_scale=0x1000, k_zero=0x1000, v_codes=0x1000, v_scale=0x1000, v_zero=0x1000, pages=4, H=2, page_size=16, D=64, scale_dtype=1)
    return _lib.PagedCacheStruct(**{**f, **change})


def test_argument_errors_need_no_gpu(qfa):
    from quant_flash_attn_amd import _lib
    L, p = _lib.lib(), 0x1000   # never dereferenced: validation fails first

    def append(cache=None, k=p, dtype=2, sk=(1024, 512, 64), table=p, width=4, starts=p, w=None, wd=0, eps=1e-6, cos=p, sin=p, rows=64, rot=64, B=1, N=8, stb=4):
        c = _abi_cache(_lib) if cache is None else cache
        return L.qfa_paged_append(ctypes.byref(c), k, p, dtype, *sk, 1024, 512, 64, table, width, stb, 1, starts, None, w, wd, 0, eps, cos, sin, rows, rot, 0, B, N, None)

    def read(cache=None, k=p, dtype=2, starts=p):
        c = _abi_cache(_lib) if cache is None else cache
        return L.qfa_paged_read(ctypes.byref(c), p, 4, 4, 1, starts, None, k, p, dtype, 1, 8, None)

    def said(rc, code, what):
        assert rc == code and what in L.qfa_last_error(), (rc, L.qfa_last_error())
    for call in (append, read):
        said(call(_abi_cache(_lib, k_scale=None)), -1, b"null")
        said(call(_abi_cache(_lib, page_size=24)), -2, b"page size")
        said(call(_abi_cache(_lib, page_size=8)), -2, b"page size")
        said(call(_abi_cache(_lib, D=96)), -2, b"head_dim")
        said(call(_abi_cache(_lib, pages=0)), -1, b"positive")
        said(call(_abi_cache(_lib, scale_dtype=7)), -1, b"scale_dtype")
        said(call(_abi_cache(_lib, v_codes=0x1008)), -1, b"aligned")
        said(call(k=None), -1, b"null")
        said(call(k=0x1008), -1, b"aligned")
        said(call(dtype=5), -1, b"dtype")
        said(call(starts=None), -1, b"starts")
    said(append(sk=(1024, 512, 60)), -1, b"strides")
    said(append(width=0), -1, b"width")
    said(append(stb=-4), -1, b"strides")
    said(append(width=1 << 28), -2, b"2^31")
    said(append(N=0), -1, b"positive")
    said(append(w=p, wd=1), -1, b"weights")
    said(append(w=p, eps=float("nan")), -1, b"eps")
    said(append(sin=None), -1, b"together")
    said(append(rot=8), -2, b"rotated")
    said(append(rot=80), -2, b"rotated")
    said(append(rows=0), -1, b"empty")

    def norm(D=64, H=2, x=p, dy=p, w=None, dw=None, ws=p, wsb=1 << 20, step=1, dtype=2):
        t = _lib.NormRopeTensor(x=x, weight=w, y=p, dy=dy, dweight=dw, H=H, sx=(1024, 512, 64), sy=(1024, 512, 64), sdy=(1024, 512, 64))
        return L.qfa_norm_rope_bwd(ctypes.byref(t), None, p, p, 64, 64, 0, None, 0, 0, step, 1e-6, dtype, 2, 1, 8, D, ws, wsb, None)
    said(norm(D=80), -2, b"head_dim")
    said(norm(H=0), -1, b"H must")
    said(norm(dy=None), -1, b"null")
    said(norm(step=2), -1, b"step")
    said(norm(dw=p), -1, b"dweight")
    said(norm(w=p, dw=p, wsb=16), -1, b"workspace")
    assert L.qfa_norm_rope_bwd_workspace_bytes(1, 8, 2, 0, 64, 0) == 2 * 64 * 4 and L.qfa_norm_rope_bwd_workspace_bytes(1, 8, 2, 0, 96, 0) == 0


def test_cpu_tensors_are_refused(qfa):
    cache = qfa.make_paged_cache(2, 2, 16, 64, device="cpu")
    x, table, starts = torch.randn(1, 2, 4, 64), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: qfa.paged_cache_append(cache, x, x, table, starts), lambda: qfa.paged_cache_read(cache, table, starts, 4),
                 lambda: qfa.quant_flash_attn_paged(x, cache, table, starts)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.mark.gpu
def test_refusals(qfa):
    cache = qfa.make_paged_cache(4, 2, 16, 64, device=DEV)
    x = torch.randn(1, 2, 4, 64, device=DEV).half()
    table, starts = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    bad = lambda i, t: [t if i == j else c for j, c in enumerate(cache)]   # noqa: E731
    for args, error, what in (((bad(0, cache[0][..., :32]), x, x, table, starts), ValueError, "differ in shape"),
                              ((bad(1, cache[1].float()), x, x, table, starts), TypeError, "scales"),
                              ((bad(2, cache[2].int()), x, x, table, starts), TypeError, "zero points"),
                              ((bad(1, cache[1][:2]), x, x, table, starts), ValueError, "one value per row"),
                              (([t.transpose(0, 1) if t.dim() == 4 else t for t in cache], x, x, table, starts), ValueError, "contiguous"),
                              ((cache, x, x, table.long(), starts), TypeError, "page_table"), ((cache, x, x, table, starts.long()), TypeError, "starts"),
                              ((cache, x, x, table[0], starts), ValueError, "page_table"), ((cache, x, x, table, starts.repeat(2)), ValueError, "starts"),
                              ((cache, x, x, table, starts, starts.float()), TypeError, "counts"), ((cache, x, x.float(), table, starts), TypeError, "dtype"),
                              ((cache, x[:, :1], x[:, :1], table, starts), ValueError, "shape"), ((cache, x, x.cpu(), table, starts), RuntimeError, "GPU only"),
                              ((cache, x, x, table, starts, None, torch.ones(32, device=DEV)), ValueError, "k_weight"),
                              ((cache, x[:, :, :0], x[:, :, :0], table, starts), RuntimeError, "positive"),
                              ((cache, x, x, table[:, :0], starts), RuntimeError, "width")):
        with pytest.raises(error, match=what):
            qfa.paged_cache_append(*args)
    with pytest.raises(TypeError):
        qfa.paged_cache_read(cache, table, starts, 4, dtype=torch.int8)
    with pytest.raises(ValueError):
        qfa.paged_cache_read(cache, table, starts, 0)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: qfa.paged_cache_read(cache, table, t, 4), (starts,), check_trace=False)
