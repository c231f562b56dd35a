"""Operators around a paged INT8 cache of keys and values, as timed cases, with their plain forms.

Three kinds, each over the range of sizes that it is used at:

  rotate   norm_rope_pair: RMSNorm of every head's queries and keys and the position rotation (training: with its gradient)
  append   paged_cache_append: keys (normed and rotated on the way) and values quantized per token into the pages of a cache;
           paged_cache_read gives the rows back as the values that they stand for
  attend   quant_flash_attn_paged: the queries at the end of every sequence on its pages; a prefix that all sequences of the
           batch share is read once for all of them

Heads: H of queries, Hk of keys and values (H is a multiple of Hk).  A cache is six tensors: codes [pages, Hk, page, D] int8,
scale and zero point [pages, Hk, page, 1], of keys and of values.  Position p of sequence b is row p % page of page
page_table[b, p // page].
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6

# Bounds of a drawn case: what the largest listed ones cost.
_MAX_BYTES = {"rotate": 1.35e9, "append": 9.5e8, "attend": 6.5e8}
_MAX_FLOPS = 7.0e10


def listed():
    return [
        # One decoding step of eight sequences: latency, launches and host time.
        dict(name="rotate_decode", kind="rotate", B=8, H=32, Hk=8, N=1, D=128, R=128, dtype="bf16", weight="shared",
             interleaved=False, positions="starts", grad=False),
        # Training on four 4096-token sequences with 32 heads of 128.
        dict(name="rotate_train_d128", kind="rotate", B=4, H=32, Hk=32, N=4096, D=128, R=128, dtype="bf16", weight="shared",
             interleaved=False, positions="none", grad=True),
        # Packed pieces of odd length: positions of their own, weights for each head, half of a small head rotated.
        dict(name="rotate_train_odd", kind="rotate", B=3, H=20, Hk=5, N=1003, D=64, R=32, dtype="fp16", weight="heads",
             interleaved=True, positions="each", grad=True),
        # fp32 tensors of wide heads, shared key heads.
        dict(name="rotate_train_fp32", kind="rotate", B=2, H=16, Hk=4, N=2048, D=256, R=256, dtype="fp32", weight="shared",
             interleaved=False, positions="none", grad=True),
        # One token each of 64 sequences into pages of 16.
        dict(name="append_decode", kind="append", B=64, Hk=8, N=1, D=128, R=128, page=16, start_low=100, start_high=2000, ragged=False,
             dtype="bf16", scale="fp16", norm=True, interleaved=False),
        # The prompts of four sequences of 4096 tokens, 32 heads.
        dict(name="append_prompt", kind="append", B=4, Hk=32, N=4096, D=128, R=128, page=64, start_low=0, start_high=0, ragged=False,
             dtype="bf16", scale="fp16", norm=False, interleaved=False),
        # Pieces of up to 517 tokens of sixteen prompts; every sequence brings another number, behind what it has.
        dict(name="append_pieces", kind="append", B=16, Hk=16, N=517, D=64, R=64, page=32, start_low=3, start_high=1500, ragged=True,
             dtype="fp16", scale="fp32", norm=True, interleaved=True),
        # One token of one sequence of 16384: few rows on a long axis.
        dict(name="attend_long", kind="attend", B=1, H=16, Hk=16, N=1, D=128, page=64, keys_low=16384, keys_high=16384, prefix=0,
             ragged=False, dtype="bf16", scale="fp16"),
        # A decoding step of 64 sequences of very different length, four query heads to a key head.
        dict(name="attend_batch", kind="attend", B=64, H=32, Hk=8, N=1, D=128, page=16, keys_low=65, keys_high=8192, prefix=0,
             ragged=False, dtype="bf16", scale="fp16"),
        # The same behind a prefix of 16384 tokens that all 64 share.
        dict(name="attend_prefix", kind="attend", B=64, H=32, Hk=8, N=1, D=128, page=64, keys_low=16400, keys_high=16895, prefix=16384,
             ragged=False, dtype="bf16", scale="fp16"),
        # Up to five drafted tokens of eight sequences at once, the widest heads, odd lengths.
        dict(name="attend_draft", kind="attend", B=8, H=16, Hk=4, N=5, D=256, page=32, keys_low=801, keys_high=3001, prefix=0,
             ragged=True, dtype="fp16", scale="fp32"),
        # A piece of a prompt on a cache of several thousand tokens; no length is a multiple of a tile.
        dict(name="attend_piece", kind="attend", B=2, H=32, Hk=32, N=333, D=128, page=64, keys_low=6001, keys_high=7001, prefix=0,
             ragged=False, dtype="bf16", scale="fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["rotate", "append", "attend", "attend"])
        Hk = _log(rng, 1, 32)
        D = rng.choice([64, 128, 128, 256])
        c = dict(kind=kind, B=_log(rng, 1, 64), Hk=Hk, D=D, dtype=rng.choice(["bf16", "bf16", "fp16"]))
        if kind != "append":
            c["H"] = Hk * rng.choice([1, 1, 2, 3, 4, 8])
        if kind != "attend":
            c.update(N=1 if rng.random() < 0.25 else _log(rng, 2, 8192), R=rng.choice([D, D, D // 2]),
                     interleaved=rng.random() < 0.3)
        if kind == "rotate":
            c.update(weight=rng.choice(["shared", "shared", "heads", "none"]), positions=rng.choice(["none", "starts", "each"]),
                     grad=c["N"] > 1 and rng.random() < 0.6)
            if rng.random() < 0.2:
                c["dtype"] = "fp32"
        else:
            c.update(page=rng.choice([16, 32, 64, 128]), scale=rng.choice(["fp16", "fp16", "fp32"]), ragged=rng.random() < 0.3)
        if kind == "append":
            low = rng.choice([0, _log(rng, 1, 2000)])
            c.update(start_low=low, start_high=low if rng.random() < 0.3 else low + _log(rng, 1, 2000), norm=rng.random() < 0.5)
        if kind == "attend":
            c["N"] = 1 if rng.random() < 0.6 else _log(rng, 2, 400)
            high = _log(rng, max(64, 2 * c["N"]), 32768)
            c["prefix"] = rng.randint(1, high - 1 - c["N"]) if c["B"] > 1 and high > 600 and rng.random() < 0.4 else 0
            c.update(keys_low=rng.randint(max(c["prefix"] + c["N"], high // 8), high), keys_high=high)
        w = work(c)
        held = 4 * c["B"] * max(c.get("keys_high", 0), 1) * Hk * D * 2   # keys and values of the plain form, in bytes
        if w["bytes"] <= _MAX_BYTES[kind] and w["flops"] <= _MAX_FLOPS and (kind != "attend" or held < 6e9):
            return c


# ---------------------------------------------------------------------------------------------------------------- inputs
def _spread(low, high, n):
    """n whole numbers from low to high, evenly."""
    return [low + (high - low) * (2 * i + 1) // (2 * n) if n > 1 else high for i in range(n)]


def _tokens(case):
    """Tokens of its own that every sequence brings: N, or of ragged ones from one to N."""
    return _spread(1, case["N"], case["B"]) if case["ragged"] else [case["N"]] * case["B"]


def _table(T, R, device):
    """cos and sin of position times 10000^(-2i/R), fp32 [T, R/2]."""
    rate = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=device) / R)
    angle = torch.arange(T, dtype=torch.float64, device=device)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _quantize(x):
    """Codes, scale and zero point of every row (last axis), as the framework's quantizer has them."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = (high - low) / 255
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    zero = _round(-128 - low / scale).clamp(-128, 127)
    return _round(x / scale + zero).clamp(-128, 127), scale, zero


def _round(x):
    """To the nearest whole number, halves away from zero."""
    t = x.trunc()
    return t + ((x - t).abs() >= 0.5) * x.sign()


def _cache(g, pages, Hk, page, D, scale_dtype, device, fill):
    """A cache of that many pages; filled: keys with an offset for each channel, values of order one."""
    out = []
    for offset in (1.0, 0.25):
        if fill:
            x = torch.randn(pages, Hk, page, D, generator=g, device=device)
            x += offset * torch.randn(1, Hk, 1, D, generator=g, device=device)
            codes, scale, zero = _quantize(x)
            out += [codes.to(torch.int8), scale.to(scale_dtype), zero.to(torch.int8)]
        else:
            out += [torch.zeros(pages, Hk, page, D, dtype=torch.int8, device=device),
                    torch.zeros(pages, Hk, page, 1, dtype=scale_dtype, device=device),
                    torch.zeros(pages, Hk, page, 1, dtype=torch.int8, device=device)]
    return tuple(out)


def _inputs(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)
    B, Hk, N, D, dtype = case["B"], case["Hk"], case["N"], case["D"], _DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=device)   # noqa: E731
    mixed = lambda values: torch.tensor(values, dtype=torch.int32, device=device)[   # noqa: E731
        torch.randperm(len(values), generator=g, device=device)]
    s = {}
    if case["kind"] == "rotate":
        H = case["H"]
        s["q"], s["k"] = ((normal(B, N, h, D) * normal(1, 1, h, D).exp()).to(dtype).permute(0, 2, 1, 3) for h in (H, Hk))
        for name, h in (("q_weight", H), ("k_weight", Hk)):
            shape = {"shared": (D,), "heads": (h, D)}.get(case["weight"])
            s[name] = (1 + 0.2 * normal(*shape)).to(dtype) if shape else None
        T = 2 * N + 4096
        s["cos"], s["sin"] = _table(T, case["R"], device)
        s["positions"] = (None if case["positions"] == "none" else
                          torch.randint(0, T - N, (B,), generator=g, device=device, dtype=torch.int32) if case["positions"] == "starts" else
                          torch.randint(0, T, (B, N), generator=g, device=device, dtype=torch.int32))
        if case["grad"]:
            s["dq"], s["dk"] = normal(B, H, N, D).to(dtype), normal(B, Hk, N, D).to(dtype)
            for name in ("q", "k", "q_weight", "k_weight"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    page, tokens = case["page"], _tokens(case)
    if case["kind"] == "append":
        s["starts"] = mixed(_spread(case["start_low"], case["start_high"], B))
        width = -(-(case["start_high"] + N) // page)
        s["k"], s["v"] = (normal(B, N, Hk, D).to(dtype).permute(0, 2, 1, 3) for _ in range(2))
        s["k_weight"] = (1 + 0.2 * normal(D)).to(dtype) if case["norm"] else None
        s["cos"], s["sin"] = _table(width * page, case["R"], device)
        prefix = 0
    else:
        keys = mixed(_spread(case["keys_low"], case["keys_high"], B))
        s["q"] = (2 * normal(B, N, case["H"], D)).to(dtype).permute(0, 2, 1, 3)
        width = -(-case["keys_high"] // page)
        prefix = case["prefix"]
    s["counts"] = mixed(tokens) if case["ragged"] else None
    if case["kind"] == "attend":   # the last token of a sequence is its last key
        s["starts"] = keys - (s["counts"] if case["ragged"] else N)
        s["starts"] = s["starts"].clamp_min(prefix)
    # pages in no order; the whole pages of the prefix are the same for all
    shared = prefix // page
    order = torch.randperm(shared + B * (width - shared) + 1, generator=g, device=device, dtype=torch.int32)
    table = order[shared:-1].view(B, width - shared)
    s["page_table"] = torch.cat([order[:shared].expand(B, shared), table], 1).contiguous()
    s["spare"] = order[-1:]   # a page that nothing is mapped to
    s["cache"] = _cache(g, order.numel(), Hk, page, D, _DTYPES[case["scale"]], device, fill=case["kind"] == "attend")
    if prefix % page:   # the prefix ends inside a page: every sequence has a copy of that part
        part = s["page_table"][:, shared].long()
        for t in s["cache"]:
            t[part, :, :prefix % page] = t[part[0], :, :prefix % page].clone()
    return s


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# ----------------------------------------------------------------------------------------------------------- plain forms
def _where(positions, B, N, device):
    """The position of every token, [B, N] or [1, N]."""
    n = torch.arange(N, device=device)
    if positions is None:
        return n[None]
    return positions.long() if positions.dim() == 2 else positions.long()[:, None] + n


def _norm_rope(x, weight, cos, sin, at, interleaved):
    """[B, H, N, D] in 32 bits: x / rms(x) * weight, then the first 2 * cos.shape[1] elements of each row rotated."""
    x = x.float()
    if weight is not None:
        w = weight.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * (w[:, None] if w.dim() == 2 else w)
    c, s, half = cos[at][:, None], sin[at][:, None], cos.shape[1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _rotate_plain(s):
    case, out = s["case"], []
    at = _where(s["positions"], case["B"], case["N"], s["cos"].device)
    out = [_norm_rope(s[n], s[n + "_weight"], s["cos"], s["sin"], at, case["interleaved"]).to(s[n].dtype) for n in "qk"]
    return tuple(out)


def _rows(s, N):
    """Page and row of tokens 0 .. N - 1 behind each sequence's start, and whether it brings them: [B, N] each."""
    n = torch.arange(N, device=s["starts"].device)
    at = s["starts"].long()[:, None] + n
    there = n < (s["counts"][:, None] if s["counts"] is not None else N)
    page = s["cache"][0].shape[2]
    return torch.where(there, s["page_table"].long().gather(1, at.clamp_max(page * s["page_table"].shape[1] - 1) // page), s["spare"].long()), at % page, there


def _append_plain(s):
    case, cache = s["case"], s["cache"]
    page, row, there = _rows(s, case["N"])
    at = (s["starts"].long()[:, None] + torch.arange(case["N"], device=row.device)).clamp_max(s["cos"].shape[0] - 1)
    k = _norm_rope(s["k"], s["k_weight"], s["cos"], s["sin"], at, case["interleaved"])
    whole = torch.cat([k, s["v"].float()], 1)
    codes, scale, zero = _quantize(whole)
    Hk, back = case["Hk"], []
    for i, rows in ((0, slice(0, Hk)), (3, slice(Hk, None))):   # keys, values
        for t, new in zip(cache[i:i + 3], (codes, scale, zero)):
            t[page, :, row] = new[:, rows].permute(0, 2, 1, 3).to(t.dtype)
        c, f, z = (t[page, :, row].float() for t in cache[i:i + 3])   # [B, N, Hk, D or 1]
        x = torch.where(there[..., None, None], (c - z) * f, 0)
        back.append(x.permute(0, 2, 1, 3).to(s["k"].dtype).contiguous())
    return tuple(back)


def _values(cache, table):
    """Keys and values of the pages of a table [B, width], in 32 bits: [B, Hk, width * page, D]."""
    out = []
    for codes, scale, zero in (cache[:3], cache[3:]):
        x = (codes[table].float() - zero[table].float()) * scale[table].float()   # [B, width, Hk, page, D]
        out.append(x.transpose(1, 2).flatten(2, 3).contiguous())
    return out


def _attend_plain(s):
    case = s["case"]
    B, H, N, D, Hk, prefix = case["B"], case["H"], case["N"], case["D"], case["Hk"], case["prefix"]
    page, table = case["page"], s["page_table"].long()
    G = H // Hk
    codes, scale, zero = _quantize(s["q"].float())
    q = ((codes - zero) * scale / math.sqrt(D)).reshape(B, Hk, G * N, D)
    skip = prefix // page   # the rows of a page in which the prefix ends are masked out below
    k, v = _values(s["cache"], table[:, skip:])
    n = torch.arange(N, device=q.device)
    last = s["starts"].long()[:, None] + n   # the last key that a query sees
    if s["counts"] is not None:
        last = torch.where(n < s["counts"][:, None], last, -1)
    last = last[:, None, None, :].expand(B, 1, G, N).reshape(B, 1, G * N, 1)
    at = skip * page + torch.arange(k.shape[2], device=q.device)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous())
    scores = scores.masked_fill((at > last) | (at < prefix), -math.inf)
    if prefix:   # all sequences' queries on the one copy
        kp, vp = (x[0, :, :prefix] for x in _values(s["cache"], table[:1, :-(-prefix // page)]))
        qp = q.transpose(0, 1).reshape(Hk, B * G * N, D)
        sp = torch.matmul(qp, kp.transpose(1, 2).contiguous()).reshape(Hk, B, G * N, prefix).transpose(0, 1)
        sp = sp.masked_fill(torch.arange(prefix, device=q.device) > last, -math.inf)
        scores = torch.cat([sp, scores], -1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., prefix:], v)
    if prefix:
        pp = p[..., :prefix].transpose(0, 1).reshape(Hk, B * G * N, prefix)
        o = o + torch.matmul(pp, vp).reshape(Hk, B, G * N, D).transpose(0, 1)
    o = torch.where(total == 0, 0, o / total)
    return o.reshape(B, H, N, D).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------------------------- run
def _rotate_own(s):
    import quant_flash_attn_amd as qfa
    return qfa.norm_rope_pair(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"],
                              interleaved=s["case"]["interleaved"], eps=_EPS)


def _append_own(s):
    import quant_flash_attn_amd as qfa
    case = s["case"]
    qfa.paged_cache_append(s["cache"], s["k"], s["v"], s["page_table"], s["starts"], s["counts"], k_weight=s["k_weight"],
                           cos=s["cos"], sin=s["sin"], interleaved=case["interleaved"], eps=_EPS)
    return qfa.paged_cache_read(s["cache"], s["page_table"], s["starts"], case["N"], s["counts"], dtype=s["k"].dtype)


def _attend_own(s):
    import quant_flash_attn_amd as qfa
    case = s["case"]
    return qfa.quant_flash_attn_paged(s["q"], s["cache"], s["page_table"], s["starts"], s["counts"],
                                      sm_scale=1 / math.sqrt(case["D"]), prefix_len=case["prefix"])


def run(state):
    case = state["case"]
    if case["kind"] == "append":
        return _append_own(state) if own else _append_plain(state)
    if case["kind"] == "attend":
        return _attend_own(state) if own else _attend_plain(state)
    with torch.set_grad_enabled(case["grad"]):
        out = _rotate_own(state) if own else _rotate_plain(state)
    if not case["grad"]:
        return out
    leaves = [state[n] for n in ("q", "k", "q_weight", "k_weight") if state[n] is not None]
    grads = torch.autograd.grad(out, leaves, [state["dq"], state["dk"]])
    return tuple(t.detach() for t in out) + grads


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    B, Hk, N, D, es = case["B"], case["Hk"], case["N"], case["D"], _ES[case["dtype"]]
    if case["kind"] == "rotate":
        rows = B * N * (case["H"] + Hk)
        # in and out; the gradient: input and gradient in, gradient out
        return {"bytes": rows * D * es * (2 + (3 if case["grad"] else 0)), "flops": rows * D * (7 + (14 if case["grad"] else 0))}
    cached = D + 1 + _ES[case["scale"]]   # bytes of a row in the cache
    tokens = _tokens(case)
    if case["kind"] == "append":
        rows = 2 * Hk * sum(tokens)
        # in, into the cache, out of the cache, and all rows of the answer
        return {"bytes": rows * (D * es + 2 * cached) + 2 * B * Hk * N * D * es, "flops": rows * D * 12}
    G, prefix = case["H"] // Hk, case["prefix"]
    own_keys = [max(k - prefix, 0) for k in _spread(case["keys_low"], case["keys_high"], B)]
    read = 2 * Hk * (sum(own_keys) + prefix) * cached
    pairs = case["H"] * sum(t * (k + prefix - (t - 1) / 2) for t, k in zip(tokens, own_keys))
    return {"bytes": read + 2 * B * case["H"] * N * D * es, "flops": 4 * D * pairs}


# ----------------------------------------------------------------------------------------------------------------- exact
def _turn64(x, cos, sin, interleaved, back=False):
    """Rotation of rows in 64 bits; back: by the opposite angle."""
    y = x.clone()
    half = cos.shape[-1]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos, -sin if back else sin)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _quantize64(x):
    """The values that a row's codes stand for before its scale, and the scale, in 64 bits."""
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    scale = torch.where(high > low, (high - low) / 255.0, 1.0)
    away = lambda y: torch.sign(y) * torch.floor(torch.abs(y) + 0.5)   # noqa: E731
    zero = away(-128.0 - low / scale).clip(-128, 127)
    return away(x / scale + zero).clip(-128, 127) - zero, scale


def _exact_rotate(case, s):
    out, grads, weight_grads = [], [], []
    positions = s["positions"]
    for b_name, d_name in (("q", "dq"), ("k", "dk")):
        x = s[b_name].detach().double()
        B, H, N, D = x.shape
        p = torch.arange(N, device=x.device).expand(B, N)
        if positions is not None:
            p = positions.long() if positions.dim() == 2 else p + positions.long()[:, None]
        cos, sin = (s[t].double()[p].unsqueeze(1) for t in ("cos", "sin"))
        w = s[b_name + "_weight"]
        if w is not None:
            w = w.detach().double()
            wide = w.unsqueeze(1) if w.dim() == 2 else w
            r = 1 / (x.square().mean(-1, keepdim=True) + _EPS).sqrt()
            y = x * r * wide
        else:
            y = x
        out.append(_turn64(y, cos, sin, case["interleaved"]))
        if case["grad"]:
            g = _turn64(s[d_name].double(), cos, sin, case["interleaved"], back=True)
            if w is None:
                grads.append(g)
                continue
            weight_grads.append((g * x * r).sum((0, 2) if w.dim() == 2 else (0, 1, 2)))
            h = g * wide
            grads.append(r * h - x * r ** 3 * (h * x).mean(-1, keepdim=True))
    return tuple(out + grads + weight_grads)


def _exact_append(case, s):
    B, Hk, N, D = case["B"], case["Hk"], case["N"], case["D"]
    count = s["counts"].tolist() if s["counts"] is not None else [N] * B
    start = s["starts"].tolist()
    back = []
    for name in "kv":
        y = torch.zeros(B, Hk, N, D, dtype=torch.float64, device=s["k"].device)
        for b in range(B):
            x = s[name][b, :, :count[b]].double()
            if name == "k":
                if s["k_weight"] is not None:
                    x = x / (x.square().mean(-1, keepdim=True) + _EPS).sqrt() * s["k_weight"].double()
                cos, sin = (s[t].double()[start[b]:start[b] + count[b]] for t in ("cos", "sin"))
                x = _turn64(x, cos, sin, case["interleaved"])
            whole, scale = _quantize64(x)
            y[b, :, :count[b]] = whole * scale.to(_DTYPES[case["scale"]]).double()
        back.append(y)
    return tuple(back)


def _exact_attend(case, s):
    B, H, N, D, Hk, page = case["B"], case["H"], case["N"], case["D"], case["Hk"], case["page"]
    o = torch.zeros(B, H, N, D, dtype=torch.float64, device=s["q"].device)
    start = s["starts"].tolist()
    count = s["counts"].tolist() if s["counts"] is not None else [N] * B
    for b in range(B):
        n, end = count[b], start[b] + count[b]
        if n == 0:
            continue
        pages = s["page_table"][b, :-(-end // page)].long()
        whole, scale = _quantize64(s["q"][b, :, :n].double())
        q = whole * scale
        hidden = torch.arange(end, device=q.device) > start[b] + torch.arange(n, device=q.device)[:, None]
        for h in range(Hk):   # (one key head at a time: the scores of a long piece in 64 bits)
            k, v = ((s["cache"][i][pages, h].double() - s["cache"][i + 2][pages, h].double()).mul(s["cache"][i + 1][pages, h].double())
                    .reshape(-1, D)[:end] for i in (0, 3))
            heads = slice(h * (H // Hk), (h + 1) * (H // Hk))
            score = (q[heads] @ k.T) / math.sqrt(D)
            o[b, heads, :n] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    return o


def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend}[case["kind"]](case, s)
