"""Eviction where pages are not there (a window has left them behind, say): their tokens are seen by nobody, and none of
them may come back as a key of the new pages."""
import math

import pytest
import torch

from oracle import kv_cache_oracle as O
from test_kv_cache_gpu import check_attn, ints, make, randn

# lens, budget, sinks, recent, kv heads, dim, page, weights, pages that are not there (of each sequence)
GAPS = [
    ([1000, 300, 64], 200, 4, 50, 2, 128, 64, "tail", [range(1, 9), range(0, 2), [0]]),     # left behind, sinks kept or not
    ([200, 100, 50], 300, 4, 20, 2, 64, 16, "tail", [[2, 3, 9], [0], [3]]),                 # within the budget, with gaps
    ([1000, 300], 290, 10, 280, 1, 128, 32, "tail", [[0, 1, 31], [9]]),                     # among sinks and recent tokens
    ([700, 700], 130, 2, 60, 2, 64, 256, "equal", [[1], [0, 1, 2]]),                        # nothing is there
    ([700, 650], 130, 2, 60, 2, 64, 64, "wild", [[0, 10], [10]]),
    ([900, 800], 600, 0, 0, 1, 64, 16, "short", [range(0, 30), range(1, 50, 3)]),           # fewer there than the budget
    ([40000, 9000, 33000], 1000, 4, 64, 1, 64, 128, "tail", [range(1, 300), [0, 70], range(8, 258)]),
    ([40000, 9000, 33000], 9000, 4, 64, 1, 64, 128, "few", [range(1, 313), [40], range(20, 258, 2)]),
    ([40000, 20000], 4000, 100, 3000, 1, 64, 16, "equal", [range(3, 2500, 2), range(1000, 1250)]),
]


def call(case):
    lens, budget, sinks, recent, hk, dim, size, kind, gone = GAPS[case]
    per = -(-budget // size)
    cache, table, seqlens, free = make(lens, hk, dim, size, 150 + case, spare=per * len(lens), wild=False)
    new_table = ints(free[:per * len(lens)]).view(len(lens), per)
    for b, pages in enumerate(gone):
        for i, page in enumerate(pages):
            table[b, page] = (-1, cache.k.shape[0], -2 ** 31, 2 ** 31 - 1)[i % 4]
    g = torch.Generator().manual_seed(450 + case)
    width = max(lens) if kind != "short" else 400
    w = torch.exp(2 * torch.randn(len(lens), hk, width, generator=g))
    if kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "wild":
        w = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -1.0, 1.0, 3.0])[torch.randint(0, 7, w.shape, generator=g)]
    elif kind == "few":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    # what is not there weighs most: the sums that its tokens earned while they were seen
    for b, pages in enumerate(gone):
        for page in pages:
            w[b, :, page * size:(page + 1) * size] = 1e6
    return cache, w.cuda(), table, seqlens, new_table, budget, sinks, recent


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(GAPS)))
def test_tokens_without_a_page_are_not_kept(case):
    from ring_swa import kv_cache_attn, kv_cache_evict

    cache, w, table, seqlens, new_table, budget, sinks, recent = call(case)
    lens, size, gone = GAPS[case][0], GAPS[case][6], GAPS[case][8]
    want, want_n, want_w, want_kept = O.evict(cache, w, table, seqlens, new_table, budget, sinks, recent)
    n, new_w, kept = kv_cache_evict(cache, w, table, seqlens, new_table, budget, num_sink_tokens=sinks, num_recent=recent)
    missing = [sum(min(length, p * size + size) - p * size for p in pages) for length, pages in zip(lens, gone)]
    assert n.tolist() == [min(budget, length - m) for length, m in zip(lens, missing)] == want_n.tolist()
    assert torch.equal(kept.cpu(), want_kept)
    assert torch.equal(new_w.cpu().nan_to_num(nan=77.0), want_w.nan_to_num(nan=77.0)) and not bool((new_w == 1e6).any())
    assert O.same_bytes(cache, want)
    for b, pages in enumerate(gone):
        assert not bool(torch.isin(kept[b] // size, torch.tensor(list(pages), device="cuda")).any())
    # a query sees the kept tokens and no others
    q = randn(torch.Generator().manual_seed(1), torch.bfloat16, len(lens), 1, 4 * w.shape[1], GAPS[case][5])
    out, lse = kv_cache_attn(q, cache, new_table, n, return_lse=True)
    check_attn(q, cache, new_table, n, out, lse)
    assert bool(((lse[..., 0] == -math.inf).all(1) == (n == 0)).all())


def test_the_restatement_keeps_tokens_that_are_there():
    from ring_swa import KVCache

    cache = KVCache.empty(9, 1, 64, 16)
    for t in cache[:2]:
        t.view(torch.uint8).fill_(0x38)
    table = torch.tensor([[3, -1, 5, 9]], dtype=torch.int32)
    w = torch.arange(64.0).view(1, 1, 64)
    new = torch.tensor([[6, 7]], dtype=torch.int32)
    _, n, new_w, kept = O.evict(cache, w, table, torch.tensor([60]), new, 20, 2, 14)
    assert n.tolist() == [20] and kept[0, 0].tolist() == [0, 1] + list(range(14, 16)) + list(range(32, 48))
    assert new_w[0, 0, :20].tolist() == kept[0, 0].tolist()
    _, n, _, kept = O.evict(cache, w, table, torch.tensor([60]), new, 32, 2, 14)
    assert n.tolist() == [32] and kept[0, 0].tolist() == list(range(16)) + list(range(32, 48))
