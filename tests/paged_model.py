"""Plain 64-bit implementations of the operators around a paged cache, and helpers that build one (not collected by pytest)."""
import math

import torch

from oracle import oracle

U32 = 2.0 ** -24   # half a unit in the last place of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}   # half a step among subnormals


def table(T, rotated, base=10000.0):
    angle = torch.arange(T, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    return angle.cos().float(), angle.sin().float()


def positions_of(positions, B, N):
    n = torch.arange(N).expand(B, N)
    if positions is None:
        return n
    return positions.long() if positions.dim() == 2 else positions.long()[:, None] + n


def turn(x, cos, sin, interleaved, back=False):
    """Rotation of [B,H,N,D]; cos, sin [B,N,R/2].  Also what bounds the error of each element: the sizes of its two terms."""
    half = cos.shape[-1]
    a_at = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b_at = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    c, s = cos[:, None].to(x.dtype), (-sin if back else sin)[:, None].to(x.dtype)
    y, size = x.clone(), x.abs()
    a, b = x[..., a_at], x[..., b_at]
    y[..., a_at], y[..., b_at] = a * c - b * s, b * c + a * s
    size[..., a_at], size[..., b_at] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def wide(w, x):
    return None if w is None else (w.double()[:, None] if w.dim() == 2 else w.double())


def norm_rope(x, w, cos, sin, positions, eps, interleaved):
    """y and the size that its fp32 error is relative to."""
    x, w = x.double(), wide(w, x)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    if cos is None:
        return x, x.abs()
    at = positions_of(positions, x.shape[0], x.shape[2])
    return turn(x, cos.double()[at], sin.double()[at], interleaved)


def norm_rope_grad(x, dy, w, cos, sin, positions, eps, interleaved):
    """dx, its size, dw (None without a weight), its size."""
    x, dy, per_head = x.double(), dy.double(), w is not None and w.dim() == 2
    w = wide(w, x)
    g, g_size = dy, dy.abs()
    if cos is not None:
        at = positions_of(positions, x.shape[0], x.shape[2])
        g, g_size = turn(dy, cos.double()[at], sin.double()[at], interleaved, back=True)
    if w is None:
        return g, g_size, None, None
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    dx = r * g * w - x * r ** 3 * (g * w * x).mean(-1, keepdim=True)
    size = r * g_size * w.abs() + x.abs() * r ** 3 * (g_size * w.abs() * x.abs()).mean(-1, keepdim=True)
    over = (0, 2) if per_head else (0, 1, 2)
    return dx, size, (g * x * r).sum(over), (g_size * x.abs() * r).sum(over)


def quantized(x):
    """(codes, scale fp32, zero point) of [..., D] by the C oracle."""
    shape = x.shape
    c, s, z, _ = oracle.quantize_per_token_c(x.reshape(1, 1, -1, shape[-1]).contiguous())
    return c.reshape(shape), s.reshape(*shape[:-1], 1), z.reshape(*shape[:-1], 1)


def values(c, s, z):
    return (c.double() - z.double()) * s.double()


def shared_pages(B, width, shared, seed, spare=3):
    """A page table [B, width] in no order, its first `shared` columns the same for all, and the number of pages."""
    g = torch.Generator().manual_seed(seed)
    n = shared + B * (width - shared) + spare
    order = torch.randperm(n, generator=g).int()
    t = torch.cat([order[:shared].expand(B, shared), order[shared:shared + B * (width - shared)].view(B, width - shared)], 1)
    return t.contiguous(), n


def garbage_cache(pages, H, page, D, scale_dtype, seed):
    """A cache of rows that nobody wrote: any codes, scales that are NaN, infinite or the largest finite number."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        s = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(scale_dtype).max])[torch.randint(0, 4, (pages, H, page, 1), generator=g)]
        out += [torch.randint(-128, 128, (pages, H, page, D), generator=g).to(torch.int8), s.to(scale_dtype),
                torch.randint(-128, 128, (pages, H, page, 1), generator=g).to(torch.int8)]
    return out


def place(cache, page_table, b, first, c, s, z, side):
    """Rows [H, n, ...] of sequence b to positions first .. in a CPU cache; side 0: keys, 3: values."""
    page = cache[0].shape[2]
    for i in range(c.shape[1]):
        p = first + i
        at = int(page_table[b, p // page]), slice(None), p % page
        cache[side][at], cache[side + 1][at], cache[side + 2][at] = c[:, i], s[:, i].to(cache[side + 1].dtype), z[:, i]


def attention(q, k, v, starts, counts, causal, sm):
    """O and, per element, sum_j p_j |v_j|, in 64 bits.  q [B,H,N,D] (its codes' values); k, v: lists of [Hk, keys, D], one per sequence."""
    B, H, N, D = q.shape
    o, size = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        n = N if counts is None else max(0, min(int(counts[b]), N))
        Hk, L = k[b].shape[0], k[b].shape[1]
        kk, vv = (t.repeat_interleave(H // Hk, 0) for t in (k[b], v[b]))
        for i in range(n):
            end = max(0, min(int(starts[b]) + (i + 1 if causal else n), L))
            if end == 0:
                continue
            p = torch.softmax((kk[:, :end] @ q[b, :, i, :, None])[..., 0] * sm, -1)
            o[b, :, i] = (p[:, None] @ vv[:, :end])[:, 0]
            size[b, :, i] = (p[:, None] @ vv[:, :end].abs())[:, 0]
    return o, size


def attention_bound(want, size, dtype, keys, v_scale):
    """As for the kernel on a cache in one piece: the output rounded once; probability times scale rounded to binary16 (2^-11; a factor 2
    covers the fp32 exponentials and the joining of pieces); the codes' offset of at most 1152 + 255 in fp32 sums, 32 roundings inside
    a tile and one per tile of 32 keys."""
    return HALF[dtype] * want.abs() + 2.0 ** -10 * size + (32 + keys / 32) * U32 * (1152 + 255) * v_scale + TINY[dtype]


def sm_of(D):
    return 1.0 / math.sqrt(D)
