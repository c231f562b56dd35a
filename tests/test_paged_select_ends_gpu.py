"""paged_select_blocks where a sequence's table ends: the last blocks that a token sees are taken, wherever the token's position lies."""
import pytest
import torch

import long_model as lm
import paged_model as m

DEV = "cuda:0"
dev = lm.dev


# one launch and two, of few rows and of many, numbers in a wave, in LDS and in memory
@pytest.mark.gpu
@pytest.mark.parametrize("G,N,width", [(1, 1, 9), (4, 3, 30), (3, 7, 200), (2, 1, 700), (8, 5, 300), (1, 2, 1100), (1, 1, 17000)])
@pytest.mark.parametrize("past", [0, 1, 16, 5000, 2147483647])
def test_past_the_end(qfa, G, N, width, past):
    page, D, pages = 16, 64, 30
    g = torch.Generator().manual_seed(width)
    q = torch.randn(1, G, N, D, generator=g).bfloat16()
    rows = torch.randn(1, 1, pages * page, D, generator=g).to(DEV)
    cache = qfa.make_paged_cache(pages, 1, page, D, device=DEV)
    own, zero = torch.arange(pages, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV)
    qfa.paged_cache_append(cache, rows, rows, own, zero)
    bounds = qfa.make_page_bounds(cache)
    qfa.paged_bounds_update(bounds, cache, own, zero, pages * page)
    pick = torch.randint(0, pages, (width,), generator=g)
    start = min(width * page - 2 + past, 2147483647 - N)   # its first token is the last one inside, or past the end
    keep, first, last = 6, 1, 3
    blocks, scores = qfa.paged_select_blocks(q.to(DEV), cache, bounds, pick.int()[None].to(DEV), torch.tensor([start], dtype=torch.int32, device=DEV), keep, first=first,
                                             last=last, return_scores=True)
    for n in range(N):
        mine = min((start + n) // page, width - 1)
        s = lm.scores_of(q[0, :, n], [t[:, 0].cpu() for t in bounds])[pick]
        assert torch.equal(scores[0, 0, n].cpu(), s)
        want = lm.select(s, list(range(width)), mine, keep, first, last)
        assert blocks[0, 0, n].tolist() == want and want[-3:] == [width - 3, width - 2, width - 1] and want[0] == 0
