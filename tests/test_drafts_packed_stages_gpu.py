"""Packed drafts over large vocabularies: of few nodes on average, some of them large trees, and of many."""
import random

import pytest
import torch

from oracle import drafts_oracle as R
from test_drafts_gpu import drawn, ints, probabilities

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [65535, 65536, 70001])
@pytest.mark.parametrize("sizes", [[6, 6, 6, 6], [1, 30, 1, 0, 1, 2], [12, 0, 9, 20], [8, 8], [9]])
def test_packed_drafts_over_large_vocabularies(sizes, vocab):
    from ring_swa import draft_tree, verify_drafts

    g = torch.Generator().manual_seed(vocab + len(sizes))
    rng = random.Random(vocab + len(sizes))
    total = sum(sizes)
    base = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    # chains where they are short, else siblings of the root with a chain behind the first
    parents = [[i - 1 for i in range(n)] if n <= 8 else [-1] + [0] * (n - 4) + [1, n - 3, n - 2] for n in sizes]
    cu = ints(base)
    tree = draft_tree(ints(sum(parents, [])), cu, max_nodes=max(sizes))
    p, q = probabilities(g, total, vocab, torch.float32, 1.0)
    for trial in range(3):
        tokens = []
        for b, own in enumerate(parents):
            rows = slice(base[b], base[b + 1])
            if own and trial == 0:  # tokens that the target likes less than the draft does
                tokens += (q[rows.start] / p[rows.start]).topk(len(own)).indices.tolist()
            else:
                tokens += drawn(rng, own, q[rows])
        u = torch.rand(total, generator=g)
        path, accepted, token = verify_drafts(tree, ints(tokens), p.cuda(), q.cuda(), u.cuda(), cu)
        for b, own in enumerate(parents):
            rows = slice(base[b], base[b + 1])
            want, following = R.verify(own, tokens[rows], p[rows], q[rows], u[rows].tolist())
            assert path[b].tolist() == want + [-1] * (path.shape[1] - len(want)), (trial, b)
            assert int(accepted[b]) == len(want) and int(token[b]) == following, (trial, b)
