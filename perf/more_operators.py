"""Operators for paged INT8 caches that have grown long, as timed cases, with their plain forms.

Four kinds, each over the range of sizes that it is used at:

  select   paged_bounds_update and paged_select_blocks: the smallest and largest keys of the pages that a call's tokens lie in,
           and for every token the blocks (pages) whose bounds promise the largest scores
  attend   quant_flash_attn_paged_blocks: attention of every token on its own list of blocks
  weigh    paged_attention_weights: the attention weight that every key of the cache gets from the call's queries, added to what it had
  evict    paged_cache_evict: the heaviest rows of every key head, in order, to new pages; paged_cache_read gives them back as values

Heads: H of queries, Hk of keys and values (H is a multiple of Hk).  A cache is six tensors: codes [pages, Hk, page, D] int8,
scale and zero point [pages, Hk, page, 1], of keys and of values.  Position p of sequence b is row p % page of page
page_table[b, p // page].  The bounds of the pages are three tensors: codes [pages, Hk, 2, D] int8 (low, high), scale fp32 and zero
point [pages, Hk, 2, 1].
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4}

# Bounds of a drawn case: what the largest listed ones cost.
_MAX_BYTES = {"select": 3.8e7, "attend": 1.4e8, "weigh": 3.2e8, "evict": 1.35e9}
_MAX_FLOPS = {"select": 7.0e8, "attend": 2.2e10, "weigh": 6.3e9, "evict": 1.0e9}


def listed():
    return [
        # One token each of 64 sequences of very different length, four query heads to a key head, pages of 16: 1024 keys of each are wanted.
        dict(name="select_batch", kind="select", B=64, H=32, Hk=8, N=1, D=128, page=16, keys_low=65, keys_high=8192, keep=64, first=1, last=2,
             ragged=False, dtype="bf16", scale="fp16"),
        # One token of one sequence of 131072: few rows on a long axis.
        dict(name="select_long", kind="select", B=1, H=32, Hk=8, N=1, D=128, page=64, keys_low=131072, keys_high=131072, keep=64, first=1, last=1,
             ragged=False, dtype="bf16", scale="fp16"),
        # A piece of two prompts, every token with a list of its own; no length is a multiple of a tile.
        dict(name="select_piece", kind="select", B=2, H=20, Hk=5, N=333, D=64, page=32, keys_low=6001, keys_high=7001, keep=48, first=1, last=4,
             ragged=False, dtype="fp16", scale="fp32"),
        # One token of one sequence, a short list: latency, launches and host time.
        dict(name="attend_one", kind="attend", B=1, H=8, Hk=2, N=1, D=64, page=16, keys_low=1000, keys_high=1000, keep=16, ragged=False,
             dtype="bf16", scale="fp16"),
        # A decoding step of 64 sequences of very different length, 1024 keys of each.
        dict(name="attend_batch", kind="attend", B=64, H=32, Hk=8, N=1, D=128, page=16, keys_low=65, keys_high=8192, keep=64, ragged=False,
             dtype="bf16", scale="fp16"),
        # Up to five drafted tokens of eight sequences at once, the widest heads, odd lengths.
        dict(name="attend_draft", kind="attend", B=8, H=16, Hk=4, N=5, D=256, page=32, keys_low=801, keys_high=3001, keep=20, ragged=True,
             dtype="fp16", scale="fp32"),
        # A piece of two prompts, 2048 keys for every token.
        dict(name="attend_piece", kind="attend", B=2, H=32, Hk=8, N=333, D=128, page=64, keys_low=6001, keys_high=7001, keep=32, ragged=False,
             dtype="bf16", scale="fp16"),
        # A decoding step of 64 sequences of very different length: every key's weight grows by what the token gave it.
        dict(name="weigh_batch", kind="weigh", B=64, H=32, Hk=8, N=1, D=128, page=16, keys_low=65, keys_high=8192, ragged=False,
             dtype="bf16", scale="fp16", before=True),
        # The last 32 tokens of four prompts say which keys of them are worth keeping.
        dict(name="weigh_window", kind="weigh", B=4, H=32, Hk=8, N=32, D=128, page=64, keys_low=4001, keys_high=8000, ragged=False,
             dtype="bf16", scale="fp16", before=False),
        # A few tokens of three sequences, three query heads to a key head, small heads, an odd length.
        dict(name="weigh_odd", kind="weigh", B=3, H=15, Hk=5, N=7, D=64, page=32, keys_low=333, keys_high=1501, ragged=True,
             dtype="fp16", scale="fp32", before=True),
        # One sequence of 5120 goes back to 4096.
        dict(name="evict_one", kind="evict", B=1, Hk=8, D=128, page=16, keys_low=5120, keys_high=5120, keep=4096, first=4, last=256, scale="fp16"),
        # Sixteen sequences at once, all heads of a model with as many key heads as query heads, odd lengths.
        dict(name="evict_batch", kind="evict", B=16, Hk=32, D=128, page=64, keys_low=1500, keys_high=3001, keep=2000, first=1, last=333, scale="fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["select", "attend", "weigh", "evict"])
        Hk = _log(rng, 1, 32)
        c = dict(kind=kind, B=_log(rng, 1, 64), Hk=Hk, D=rng.choice([64, 128, 128, 256]), page=rng.choice([16, 32, 64, 128]),
                 scale=rng.choice(["fp16", "fp16", "fp32"]))
        high = _log(rng, 64, 131072 if kind == "select" else 32768)
        c.update(keys_low=rng.randint(max(1, high // 8), high), keys_high=high)
        blocks = -(-high // c["page"])
        if kind == "evict":
            c["keep"] = _log(rng, max(2, high // 4), high)
            c.update(first=rng.randint(0, min(16, c["keep"] // 2)), last=rng.randint(0, c["keep"] // 2))
        else:
            most = 64 if kind == "weigh" else 400
            c.update(H=Hk * rng.choice([1, 1, 2, 3, 4, 8]), N=1 if rng.random() < 0.6 else _log(rng, 2, max(2, min(most, c["keys_low"]))),
                     ragged=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        if kind in ("select", "attend"):
            c["keep"] = _log(rng, 1, min(blocks, 4096 // c["page"]))
        if kind == "select":
            c.update(first=rng.randint(0, c["keep"] // 2), last=rng.randint(1, max(1, c["keep"] // 2)))
        if kind == "weigh":
            c["before"] = rng.random() < 0.7
        w = work(c)
        cache = 2 * c["B"] * high * Hk * c["D"]
        rows = c["B"] * (c.get("H", 0) * c.get("N", 0))
        # the largest tensors of the plain form, in bytes: scores, or the rows of all lists
        held = {"select": 8 * rows * blocks, "weigh": 4 * rows * high, "evict": 0}.get(kind, 4 * c["B"] * Hk * c.get("N", 0) * c.get("keep", 0) * c["page"] * c["D"])
        if w["bytes"] <= _MAX_BYTES[kind] and w["flops"] <= _MAX_FLOPS[kind] and cache < 1.2e9 and held < 6e9 and c["keys_low"] >= c.get("N", 1):
            return c


# ---------------------------------------------------------------------------------------------------------------- inputs
def _spread(low, high, n):
    """n whole numbers from low to high, evenly."""
    return [low + (high - low) * (2 * i + 1) // (2 * n) if n > 1 else high for i in range(n)]


def _tokens(case):
    """Tokens of its own that every sequence brings: N, or of ragged ones from one to N."""
    return _spread(1, case["N"], case["B"]) if case["ragged"] else [case["N"]] * case["B"]


def _round(x):
    """To the nearest whole number, halves away from zero."""
    t = x.trunc()
    return t + ((x - t).abs() >= 0.5) * x.sign()


def _over(a, b):
    """The quotient rounded to 32 bits (the one in 64 bits has more than twice as many)."""
    return (a.double() / b.double()).float()


def _quantize(x):
    """Codes, scale and zero point of every row (last axis) of 32-bit values, bit for bit as the framework's quantizer has them."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = _over(high - low, torch.full_like(low, 255))
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    zero = _round(-128 - _over(low, scale)).clamp(-128, 127)
    return _round(_over(x, scale) + zero).clamp(-128, 127), scale, zero


def _cache(g, pages, Hk, page, D, scale_dtype, device):
    """A filled cache: keys with an offset for each channel and one for each page (what it is about), values of order one."""
    out = []
    for offset, about in ((1.0, 0.5), (0.25, 0.0)):
        x = torch.randn(pages, Hk, page, D, generator=g, device=device)
        x += offset * torch.randn(1, Hk, 1, D, generator=g, device=device)
        x += about * torch.randn(pages, Hk, 1, D, generator=g, device=device)
        low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        scale = ((high - low) / 255).to(scale_dtype)
        zero = (-128 - low / scale).round().clamp(-128, 127)
        x = x.div_(scale).add_(zero).round_().clamp_(-128, 127)
        out += [x.to(torch.int8), scale, zero.to(torch.int8)]
    return tuple(out)


def _inputs(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)
    kind, B, Hk, D, page = case["kind"], case["B"], case["Hk"], case["D"], case["page"]
    mixed = lambda values: torch.tensor(values, dtype=torch.int32, device=device)[   # noqa: E731
        torch.randperm(len(values), generator=g, device=device)]
    s = {}
    keys = mixed(_spread(case["keys_low"], case["keys_high"], B))
    width = -(-case["keys_high"] // page)
    more = -(-min(case["keep"], case["keys_high"]) // page) if kind == "evict" else 0   # new pages of a sequence
    order = torch.randperm(B * (width + more) + 1, generator=g, device=device, dtype=torch.int32)   # pages in no order
    s["page_table"] = order[:B * width].view(B, width)
    s["spare"] = order[-1:]   # a page that nothing is mapped to
    s["cache"] = _cache(g, order.numel(), Hk, page, D, _DTYPES[case["scale"]], device)
    if kind == "evict":
        s["new_page_table"] = order[B * width:-1].view(B, more)
        s["lengths"] = keys
        # a few keys have most of the weight
        s["weights"] = torch.randn(B, Hk, width * page, generator=g, device=device).mul_(2).exp_()
        return s
    H, N = case["H"], case["N"]
    s["counts"] = mixed(_tokens(case)) if case["ragged"] else None
    s["starts"] = keys - (s["counts"] if case["ragged"] else N)   # the last token of a sequence is its last key
    s["q"] = (2 * torch.randn(B, N, H, D, generator=g, device=device)).to(_DTYPES[case["dtype"]]).permute(0, 2, 1, 3)
    if kind == "select":
        low, high = (f(_values(s["cache"][:3], None), 2) for f in (torch.amin, torch.amax))   # of whole pages: the last one is the call's
        codes, scale, zero = _quantize(torch.stack([low, high], 2))
        s["bounds"] = (codes.to(torch.int8), scale, zero.to(torch.int8))
    elif kind == "attend":
        at = s["starts"][:, None] + torch.arange(N, device=device)
        if s["counts"] is not None:
            at = torch.where(torch.arange(N, device=device) < s["counts"][:, None], at, -1)
        s["blocks"] = _some_blocks(g, case, at, width)
    else:
        s["lse"] = _log_sums(s, case)
        # of the order of what a few calls give a key
        s["weights"] = torch.rand(B, Hk, width * page, generator=g, device=device).mul_(8 * H / Hk / case["keys_high"]) if case["before"] else None
    return s


def _some_blocks(g, case, at, width):
    """For every token and key head `keep` of the blocks that it sees, its own among them, ascending, -1 behind: [B, Hk, N, keep]."""
    B, Hk, N, page, keep = case["B"], case["Hk"], case["N"], case["page"], case["keep"]
    mine = (at // page)[:, None, :, None]
    j = torch.arange(width, device=at.device)
    rank = torch.rand(B, Hk, N, width, generator=g, device=at.device)
    rank = torch.where(j == mine, 2.0, rank).masked_fill(j > mine, -1.0)
    best = rank.topk(keep, -1)
    return torch.where(best.values < 0, width, best.indices).sort(-1).values.masked_fill_(torch.arange(keep, device=at.device) > mine, -1).int()


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# ----------------------------------------------------------------------------------------------------------- plain forms
def _values(side, pages):
    """What the rows of those pages (all: None) stand for, in 32 bits; side: codes, scale, zero point."""
    codes, scale, zero = side if pages is None else (t[pages] for t in side)
    return (codes.float() - zero.float()) * scale.float()


def _in_order(s, side):
    """Keys or values of every sequence, [B, Hk, width * page, D] in 32 bits."""
    return _values(side, s["page_table"].long()).transpose(1, 2).flatten(2, 3)


def _positions(s, N):
    """The position of every token, [B, N]; -1: padding."""
    n = torch.arange(N, device=s["starts"].device)
    at = s["starts"].long()[:, None] + n
    return at if s["counts"] is None else torch.where(n < s["counts"][:, None], at, -1)


def _scores(s, case):
    """Scores of all rows of a sequence and key head, query by query and in it head by head, on all its keys, and whether a row sees the key."""
    B, H, N, D, Hk = case["B"], case["H"], case["N"], case["D"], case["Hk"]
    codes, scale, zero = _quantize(s["q"].float())
    q = ((codes - zero) * scale / math.sqrt(D)).reshape(B, Hk, H // Hk, N, D).transpose(2, 3).reshape(B, Hk, -1, D)
    k = _in_order(s, s["cache"][:3])
    seen = torch.arange(k.shape[2], device=k.device) <= _positions(s, N).repeat_interleave(H // Hk, 1)[:, None, :, None]
    return torch.matmul(q, k.transpose(2, 3).contiguous()), seen


def _log_sums(s, case):
    """What quant_flash_attn_paged hands out beside its output: [B, H, N] fp32."""
    scores, seen = _scores(s, case)
    lse = torch.logsumexp(scores.masked_fill_(~seen, -math.inf), -1)
    return lse.reshape(case["B"], case["Hk"], case["N"], -1).transpose(2, 3).reshape(case["B"], case["H"], case["N"]).contiguous()


def _select_plain(s):
    case = s["case"]
    B, H, N, D, Hk, page, keep = (case[n] for n in ("B", "H", "N", "D", "Hk", "page", "keep"))
    table, at = s["page_table"].long(), _positions(s, N)
    width = table.shape[1]
    # the pages that the call's tokens lie in
    end = at.amax(1)[:, None] + 1
    touched = s["starts"].long()[:, None] // page + torch.arange((N + page - 2) // page + 1, device=at.device)
    pages = torch.where(touched * page < end, table.gather(1, touched.clamp_max(width - 1)), s["spare"].long())
    k = _values(s["cache"][:3], pages)   # [B, pages, Hk, page, D]
    there = (touched[..., None] * page + torch.arange(page, device=at.device) < end[..., None])[:, :, None, :, None]
    low, high = k.masked_fill(~there, math.inf).amin(3), k.masked_fill(~there, -math.inf).amax(3)
    for t, new in zip(s["bounds"], _quantize(torch.stack([low, high], 3))):
        t[pages] = new.to(t.dtype)
    # whole numbers, and beside them 64 bits: the last block that is taken borders on the first one that is not
    codes, scale, zero = _quantize(s["q"].float())
    e = (codes - zero).double().reshape(B, Hk, -1, D)
    bc, bs, bz = (t[table].transpose(1, 2).double() for t in s["bounds"])   # [B, Hk, width, 2, D or 1]
    whole = (bc - bz).permute(0, 1, 3, 4, 2).contiguous()
    score = torch.matmul(e.clamp_min(0), whole[:, :, 1]) * bs[:, :, None, :, 1, 0] + torch.matmul(e.clamp_max(0), whole[:, :, 0]) * bs[:, :, None, :, 0, 0]
    score = (score * scale.double().reshape(B, Hk, -1, 1)).float().reshape(B, Hk, H // Hk, N, width).amax(2)
    mine = (torch.where(at < 0, -1, at // page))[:, None, :, None]
    j = torch.arange(width, device=at.device)
    score = score.masked_fill(j > mine, -math.inf)
    always = (j < case["first"]) | (j > mine - case["last"])
    rank = torch.where(always & (j <= mine), math.inf, score)
    best = rank.sort(dim=-1, descending=True, stable=True)
    taken = torch.where(best.values[..., :keep] == -math.inf, width, best.indices[..., :keep]).sort(-1).values
    return taken.masked_fill(taken == width, -1).int(), score


def _attend_plain(s):
    case, cache = s["case"], s["cache"]
    B, H, N, D, Hk, page = (case[n] for n in ("B", "H", "N", "D", "Hk", "page"))
    blocks = s["blocks"].long()
    b, h = torch.arange(B, device=blocks.device)[:, None, None, None], torch.arange(Hk, device=blocks.device)[:, None, None]
    places = (s["page_table"].long()[b, blocks.clamp_min(0)], h)
    k, v = (_values(side, places).flatten(3, 4) for side in (cache[:3], cache[3:]))   # [B, Hk, N, keep * page, D]
    codes, scale, zero = _quantize(s["q"].float())
    q = ((codes - zero) * scale / math.sqrt(D)).reshape(B, Hk, H // Hk, N, D).transpose(2, 3).contiguous()
    at = (blocks[..., None] * page + torch.arange(page, device=blocks.device)).flatten(3)
    seen = (at >= 0) & (at <= _positions(s, N)[:, None, :, None])
    scores = torch.matmul(q, k.transpose(3, 4).contiguous()).masked_fill(~seen[:, :, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.where(total == 0, 0, torch.matmul(p, v) / total)
    return o.transpose(2, 3).reshape(B, H, N, D).to(s["q"].dtype)


def _weigh_plain(s):
    case = s["case"]
    scores, seen = _scores(s, case)
    lse = s["lse"].reshape(case["B"], case["Hk"], -1, case["N"]).transpose(2, 3).flatten(2)[..., None]
    new = torch.where(seen, torch.exp(scores - lse), 0).sum(2)
    return new if s["weights"] is None else s["weights"] + new


def _evict_plain(s):
    case, cache = s["case"], s["cache"]
    page, keep, w = case["page"], s["new_page_table"].shape[1] * case["page"], s["weights"]
    length = s["lengths"].long()[:, None, None]
    slot = torch.arange(w.shape[2], device=w.device)
    rank = torch.where((slot < case["first"]) | (slot >= length - case["last"]), math.inf, w).masked_fill(slot >= length, -math.inf)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :case["keep"]]
    kept = torch.where(torch.arange(kept.shape[2], device=w.device) < length, kept, w.shape[2]).sort(-1).values   # [B, Hk, places]
    there = kept < length
    from_page = torch.where(there, s["page_table"].long().gather(1, (kept.clamp_max(w.shape[2] - 1) // page).flatten(1)).view_as(kept), s["spare"].long())
    place = torch.arange(kept.shape[2], device=w.device)
    to_page = torch.where(there, s["new_page_table"].long()[:, None, place // page], s["spare"].long())
    h = torch.arange(case["Hk"], device=w.device)[:, None]
    for t in cache:
        t[to_page, h, place % page] = t[from_page, h, kept % page]
    new = torch.zeros(*w.shape[:2], keep, device=w.device)
    new[..., :kept.shape[2]] = torch.where(there, w.gather(2, kept.clamp_max(w.shape[2] - 1)), 0)
    out = torch.full((*w.shape[:2], case["keep"]), -1, dtype=torch.int32, device=w.device)
    out[..., :kept.shape[2]] = torch.where(there, kept, -1)
    rows = [torch.where(there[..., None], _values(side, (to_page, h, place % page)), 0).bfloat16() for side in (cache[:3], cache[3:])]
    return (out, new, s["lengths"].clamp_max(case["keep"]), *rows)


# ------------------------------------------------------------------------------------------------------------------- run
def _select_own(s):
    import quant_flash_attn_amd as qfa
    case = s["case"]
    qfa.paged_bounds_update(s["bounds"], s["cache"], s["page_table"], s["starts"], case["N"], s["counts"])
    return qfa.paged_select_blocks(s["q"], s["cache"], s["bounds"], s["page_table"], s["starts"], case["keep"], s["counts"], first=case["first"],
                                   last=case["last"], return_scores=True)


def _attend_own(s):
    import quant_flash_attn_amd as qfa
    return qfa.quant_flash_attn_paged_blocks(s["q"], s["cache"], s["page_table"], s["starts"], s["blocks"], s["counts"],
                                             sm_scale=1 / math.sqrt(s["case"]["D"]))


def _weigh_own(s):
    import quant_flash_attn_amd as qfa
    return qfa.paged_attention_weights(s["q"], s["cache"], s["lse"], s["page_table"], s["starts"], s["counts"],
                                       sm_scale=1 / math.sqrt(s["case"]["D"]), weights=s["weights"])


def _evict_own(s):
    import quant_flash_attn_amd as qfa
    case = s["case"]
    kept, weights, lengths = qfa.paged_cache_evict(s["cache"], s["page_table"], s["lengths"], s["weights"], case["keep"], s["new_page_table"],
                                                   first=case["first"], last=case["last"])
    rows = qfa.paged_cache_read(s["cache"], s["new_page_table"], torch.zeros_like(lengths), min(case["keep"], case["keys_high"]), lengths,
                                dtype=torch.bfloat16)
    return (kept, weights, lengths, *rows)


def run(state):
    kind = state["case"]["kind"]
    with torch.no_grad():
        if own:
            return {"select": _select_own, "attend": _attend_own, "weigh": _weigh_own, "evict": _evict_own}[kind](state)
        return {"select": _select_plain, "attend": _attend_plain, "weigh": _weigh_plain, "evict": _evict_plain}[kind](state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    B, Hk, D, page, kind = case["B"], case["Hk"], case["D"], case["page"], case["kind"]
    keys = _spread(case["keys_low"], case["keys_high"], B)
    row = D + 1 + _ES[case["scale"]]   # bytes of a row in the cache
    if kind == "evict":
        kept = sum(min(k, case["keep"]) for k in keys)
        # weights in and out, the list, rows out of old pages, into new ones and out of those, and all rows of the answer
        new = min(case["keep"], case["keys_high"])
        return {"bytes": Hk * (4 * sum(keys) + 4 * B * (-(-new // page) * page + case["keep"]) + 6 * kept * row + 4 * B * new * D), "flops": 4 * D * Hk * kept}
    H, N, tokens = case["H"], case["N"], _tokens(case)
    q = B * H * N * D * _ES[case["dtype"]]
    if kind == "select":
        blocks = [-(-k // page) for k in keys]
        touched = sum(k - (k - t) // page * page for k, t in zip(keys, tokens))   # rows of the pages that the tokens lie in
        lists = B * Hk * N * (4 * case["keep"] + 4 * -(-case["keys_high"] // page))
        return {"bytes": touched * Hk * row + sum(blocks) * Hk * 2 * (D + 5) + q + lists, "flops": H * 4 * D * sum(n * t for n, t in zip(blocks, tokens))}
    if kind == "attend":   # the blocks of a token's list, of the last one what it sees; what several tokens list is read once
        lists = [[min(case["keep"], (k - i - 1) // page + 1) * page - (page - 1 - (k - i - 1) % page) for i in range(t)] for k, t in zip(keys, tokens)]
        read = sum(min(k, sum(x)) for k, x in zip(keys, lists))
        return {"bytes": 2 * Hk * read * row + 2 * q + 4 * B * Hk * N * case["keep"], "flops": 4 * D * H * sum(map(sum, lists))}
    pairs = H * sum(t * (k - (t - 1) / 2) for t, k in zip(tokens, keys))
    slots = -(-case["keys_high"] // page) * page
    return {"bytes": Hk * (sum(keys) * row + 4 * B * slots * (2 if case["before"] else 1)) + q + 4 * B * H * N, "flops": 2 * D * pairs}


# ----------------------------------------------------------------------------------------------------------------- exact
def _rows64(side, pages, h):
    """Rows of one key head on those pages, in order, in 64 bits."""
    codes, scale, zero = (t[pages, h].flatten(0, 1).double() for t in side)
    return (codes - zero) * scale


def _quantized64(x):
    """The whole numbers that the codes of rows stand for, and their scale (codes are what they are in 32 bits)."""
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    near = lambda y: y.float().double()   # noqa: E731
    away = lambda y: torch.sign(y) * torch.floor(torch.abs(y) + 0.5)   # noqa: E731
    span = near(high - low)
    scale = torch.where(span > 0, near(span / 255.0), 1.0)
    zero = away(near(-128.0 - near(low / scale))).clip(-128, 127)
    return away(near(near(x / scale) + zero)).clip(-128, 127) - zero, scale


def _each(case, s):
    """Every sequence: its number, tokens, keys, and the pages that hold them."""
    starts = s["starts"].tolist()
    counts = s["counts"].tolist() if s["counts"] is not None else [case["N"]] * case["B"]
    for b, (start, n) in enumerate(zip(starts, counts)):
        yield b, n, start + n, s["page_table"][b, :-(-(start + n) // case["page"])].long()


def _exact_select(case, s):
    B, H, N, Hk, page, keep = (case[n] for n in ("B", "H", "N", "Hk", "page", "keep"))
    G, device = H // Hk, s["q"].device
    lists = torch.full((B, Hk, N, keep), -1, dtype=torch.int32, device=device)
    scores = torch.full((B, Hk, N, s["page_table"].shape[1]), -math.inf, dtype=torch.float64, device=device)
    for b, n, end, pages in _each(case, s):
        whole, scale = _quantized64(s["q"][b, :, :n].double())
        for h in range(Hk):
            k = torch.nn.functional.pad(_rows64(s["cache"][:3], pages, h).float().double()[:end], (0, 0, 0, -end % page), value=math.nan).view(pages.numel(), page, -1)
            hidden = k.isnan()
            bounds = [_quantized64(x) for x in (k.masked_fill(hidden, math.inf).amin(1), k.masked_fill(hidden, -math.inf).amax(1))]
            e = whole[h * G:(h + 1) * G]
            low, high = (c * f for c, f in bounds)
            value = ((e.clip(max=0) @ low.T) + (e.clip(min=0) @ high.T)) * scale[h * G:(h + 1) * G]   # [G, n, blocks]
            value = value.max(0).values
            mine = (torch.arange(end - n, end, device=device) // page)[:, None]
            j = torch.arange(pages.numel(), device=device)
            value = value.masked_fill(j > mine, -math.inf)
            scores[b, h, :n, :pages.numel()] = value
            value = value.float().double().masked_fill(((j < case["first"]) | (j > mine - case["last"])) & (j <= mine), math.inf)
            best = value.sort(dim=-1, descending=True, stable=True)
            m = min(keep, pages.numel())
            chosen = torch.where(best.values[:, :m] > -math.inf, best.indices[:, :m], 1 << 30).sort(-1).values
            lists[b, h, :n, :m] = torch.where(chosen < 1 << 30, chosen, -1).int()
    return lists, scores


def _exact_attend(case, s):
    B, H, N, D, Hk, page = (case[n] for n in ("B", "H", "N", "D", "Hk", "page"))
    if B * N * Hk > 1500:   # one list after the other
        return None
    G = H // Hk
    o = torch.zeros(B, H, N, D, dtype=torch.float64, device=s["q"].device)
    for b, n, end, _ in _each(case, s):
        whole, scale = _quantized64(s["q"][b, :, :n].double())
        q = whole * scale
        for h in range(Hk):
            for i in range(n):
                listed = s["blocks"][b, h, i].long()
                listed = listed[listed >= 0]
                at = (listed[:, None] * page + torch.arange(page, device=listed.device)).flatten()
                hidden = at > end - n + i
                pages = s["page_table"][b, listed].long()
                k, v = (_rows64(side, pages, h) for side in (s["cache"][:3], s["cache"][3:]))
                score = (q[h * G:(h + 1) * G, i] @ k.T) / math.sqrt(D)
                o[b, h * G:(h + 1) * G, i] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    return o


def _exact_weigh(case, s):
    B, H, D, Hk = (case[n] for n in ("B", "H", "D", "Hk"))
    G, w = H // Hk, s["weights"]
    out = torch.zeros(B, Hk, s["page_table"].shape[1] * case["page"], dtype=torch.float64, device=s["q"].device)
    if w is not None:
        out += w.double()
    for b, n, end, pages in _each(case, s):
        whole, scale = _quantized64(s["q"][b, :, :n].double())
        q = whole * scale
        hidden = torch.arange(end, device=q.device) > end - n + torch.arange(n, device=q.device)[:, None]
        for h in range(Hk):
            heads = slice(h * G, (h + 1) * G)
            score = (q[heads] @ _rows64(s["cache"][:3], pages, h)[:end].T) / math.sqrt(D)
            out[b, h, :end] += torch.exp(score - s["lse"][b, heads, :n, None].double()).masked_fill(hidden, 0.0).sum((0, 1))
    return out


def _exact_evict(case, s):
    B, Hk, D, page, keep = (case[n] for n in ("B", "Hk", "D", "page", "keep"))
    device, lengths, most = s["weights"].device, s["lengths"].tolist(), min(keep, case["keys_high"])
    kept = torch.full((B, Hk, keep), -1, dtype=torch.int32, device=device)
    weights = torch.zeros(B, Hk, s["new_page_table"].shape[1] * page, dtype=torch.float64, device=device)
    rows = [torch.zeros(B, Hk, most, D, dtype=torch.float64, device=device) for _ in range(2)]
    for b, n in enumerate(lengths):
        pages, m = s["page_table"][b, :-(-n // page)].long(), min(n, keep)
        for h in range(Hk):
            w = s["weights"][b, h, :n].double()
            free = torch.arange(min(case["first"], n), max(n - case["last"], min(case["first"], n)), device=device)
            chosen = torch.ones(n, dtype=torch.bool, device=device)
            if m < n:
                by_weight = free[torch.argsort(w[free], descending=True, stable=True)]
                chosen[by_weight[m - (n - free.numel()):]] = False
            at = chosen.nonzero()[:, 0]
            kept[b, h, :m] = at.int()
            weights[b, h, :m] = w[at]
            for to, side in zip(rows, (s["cache"][:3], s["cache"][3:])):
                to[b, h, :m] = _rows64(side, pages, h)[at]
    return (kept, weights, s["lengths"].clamp(max=keep), *rows)


def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        return {"select": _exact_select, "attend": _exact_attend, "weigh": _exact_weigh, "evict": _exact_evict}[case["kind"]](case, s)
