"""Plain implementations of the operators for long paged caches, in 64 bits and on the CPU, and problems for them (not collected by pytest)."""
import math

import torch

import paged_model as m

DEV = "cuda:0"


def dev(t):
    return [dev(x) for x in t] if isinstance(t, (list, tuple)) else None if t is None else t.to(DEV)


class Problem:
    """A batch of sequences with `keys` keys each (the new tokens among them) on a cache whose other rows hold garbage."""

    def __init__(self, B, H, Hk, N, D, page, keys, dtype=torch.bfloat16, scale_dtype=torch.float16, counts=None, seed=0, width=None, spare=3, layout="bhnd",
                 size=1.0):
        g = torch.Generator().manual_seed(seed)
        self.B, self.H, self.Hk, self.N, self.D, self.page, self.G = B, H, Hk, N, D, page, H // Hk
        q = (2 * torch.randn(B, H, N, D, generator=g)).to(dtype)
        self.q = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) if layout == "bnhd" else q
        self.width = width or max(1, -(-max(keys) // page))
        self.table, self.pages = m.shared_pages(B, self.width, 0, seed, spare)
        self.cache = m.garbage_cache(self.pages, Hk, page, D, scale_dtype, seed + 1)
        offset = torch.randn(Hk, 1, D, generator=g)
        self.rows = ([], [])   # keys and values of every sequence, [Hk, n, D] in 64 bits
        for b in range(B):
            n = max(keys[b], 0)
            about = torch.randn(Hk, -(-n // page), 1, D, generator=g).expand(Hk, -1, page, D).reshape(Hk, -1, D)[:, :n]
            for side, x in ((0, torch.randn(Hk, n, D, generator=g) + offset + 0.5 * about), (3, torch.randn(Hk, n, D, generator=g))):
                c, s, z = m.quantized(size * x) if n else (torch.zeros(Hk, 0, D), torch.zeros(Hk, 0, 1), torch.zeros(Hk, 0, 1))
                m.place(self.cache, self.table, b, 0, c, s, z, side)
                self.rows[side // 3].append(m.values(c, s.to(scale_dtype), z))
        self.counts = None if counts is None else torch.tensor(counts, dtype=torch.int32)
        self.tokens = [N if counts is None else max(0, min(c, N)) for c in (counts or [N] * B)]
        self.starts = (torch.tensor(keys) - torch.tensor(self.tokens)).int()
        self.v_scale = float(max([x.abs().max() for x in self.rows[1] if x.numel()] or [1.0])) / 64

    def places(self):
        return dev((self.table, self.starts))

    def fake_lists(self, keep, seed=0):
        """For every token and key head some distinct blocks that it sees, in no order, -1 behind."""
        g = torch.Generator().manual_seed(seed)
        out = torch.full((self.B, self.Hk, self.N, keep), -1, dtype=torch.int32)
        for b in range(self.B):
            for n in range(self.tokens[b]):
                last = int(self.starts[b]) + n
                if last < 0:
                    continue
                for h in range(self.Hk):
                    seen = torch.randperm(min(last // self.page, self.width - 1) + 1, generator=g)[:keep]
                    out[b, h, n, :seen.numel()] = seen.int()
        return out


def bounds_of_page(k):
    """Codes, scale and zero point of the low and the high row of keys [rows, D] (64-bit values that are rounded to 32 first)."""
    k = k.float()
    return m.quantized(torch.stack([k.amin(0), k.amax(0)]))


def scores_of(q, bounds):
    """Of queries [G, D] (32-bit values) against bounds (codes [blocks, 2, D], scale, zero point): [blocks], the largest over G, rounded to fp32."""
    c, s, z = m.quantized(q.float())
    e = (c.double() - z.double())
    bc, bs, bz = (t.double() for t in bounds)
    whole = bc - bz
    u = bs[:, 1, 0] * (e.clamp_min(0) @ whole[:, 1].T) + bs[:, 0, 0] * (e.clamp_max(0) @ whole[:, 0].T)
    u = (u * s.double()).float()
    return torch.nan_to_num(u, nan=-math.inf, neginf=-math.inf, posinf=math.inf).amax(0).clamp_min(torch.finfo(torch.float32).min)


def select(scores, candidates, mine, keep, first, last):
    """The list of one token: scores [blocks], which of them are candidates, its own block."""
    rank = []
    for j in candidates:
        forced = j < first or j > mine - last
        rank.append((0 if forced else 1, -float(scores[j]), j))
    taken = sorted(j for _, _, j in sorted(rank)[:keep])
    return taken + [-1] * (keep - len(taken))


def attention_on(q, keys, values, seen, sm):
    """O [D] and sum p |v| of one row (a 64-bit query) on keys [n, D] where seen."""
    if not bool(seen.any()):
        return torch.zeros_like(q), torch.zeros_like(q)
    p = torch.softmax((keys @ q * sm).masked_fill(~seen, -math.inf), 0)
    return p @ values, p @ values.abs()


def log_sums(p, causal, sm):
    """[B, H, N] in 64 bits, and the scores' sizes (largest |score|)."""
    qh = m.values(*m.quantized(p.q.float()))
    out, size = torch.full((p.B, p.H, p.N), -math.inf, dtype=torch.float64), 0.0
    for b in range(p.B):
        for n in range(p.tokens[b]):
            end = max(0, min(int(p.starts[b]) + (n + 1 if causal else p.tokens[b]), p.rows[0][b].shape[1]))
            if end:
                s = torch.stack([p.rows[0][b][h // p.G, :end] @ qh[b, h, n] * sm for h in range(p.H)])
                out[b, :, n] = torch.logsumexp(s, -1)
                size = max(size, s.abs().max().item())
    return out, size


def weights_of(p, lse, causal, sm, slots):
    """What every key gets, [B, Hk, slots] in 64 bits, with a log-sum-exp as it is given."""
    qh = m.values(*m.quantized(p.q.float()))
    out = torch.zeros(p.B, p.Hk, slots, dtype=torch.float64)
    for b in range(p.B):
        for n in range(p.tokens[b]):
            end = max(0, min(int(p.starts[b]) + (n + 1 if causal else p.tokens[b]), p.rows[0][b].shape[1]))
            for h in range(p.H if end else 0):
                out[b, h // p.G, :end] += torch.exp(p.rows[0][b][h // p.G, :end] @ qh[b, h, n] * sm - lse[b, h, n].double())
    return out


def weights_bound(want, size, rows):
    """Relative: a score is the exact whole number times two scales, each of them and their products rounded to 32 bits (4 roundings of the score, whose
    size in log2 units is at most size / ln 2), the log-sum-exp turned to log2 units (its own rounding and the product's, of at most
    size / ln 2 + 20) and the difference (one); v_exp_f32 is good for 1 ulp; then a sum of `rows` terms."""
    log2 = size / math.log(2)
    return want * (math.log(2) * m.U32 * (4 * log2 + 3 * (log2 + 20)) + 2 * m.U32 + rows * m.U32) + 1e-37


def evict(weights, length, keep, first, last):
    """The kept slots of one sequence and key head."""
    n, k = length, min(length, keep)
    rank = []
    for i in range(n):
        w = float(weights[i])
        rank.append((0, 0.0, i) if i < first or i >= n - last else (1, math.inf if math.isnan(w) else -w, i))
    # (NaN below -inf)
    rank.sort(key=lambda r: (r[0], r[1], 1 if r[0] and math.isnan(float(weights[r[2]])) else 0, r[2]))
    return sorted(i for _, _, i in rank[:k])
