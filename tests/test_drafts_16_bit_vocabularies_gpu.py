"""Verification over vocabularies of many pieces in 16 bits, with a draft and with drafts named outright, choice for choice
against the 64-bit restatement: rows whose last vector overlaps the one before it, tokens tried in it, draws from the last pieces."""
import random

import pytest
import torch

from oracle import drafts_oracle as R
from test_drafts_gpu import DTYPES, drawn, ints, tree_tensors

pytestmark = pytest.mark.gpu


def rows_of(g, rows, vocab, dtype):
    """Target and draft; the last tokens among the likeliest, of both."""
    common = 2 * torch.randn(rows, vocab, generator=g)
    common[:, -9:] += 9
    return [torch.softmax(common + 0.7 * torch.randn(rows, vocab, generator=g), -1).to(dtype) for _ in range(2)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("vocab", [32767, 32769, 50001, 65537, 131071])
def test_verification_in_16_bits(vocab, dtype, sampled, packed):
    from ring_swa import verify_drafts

    batch, nodes = 4, 14
    g = torch.Generator().manual_seed(vocab + sampled)
    rng = random.Random(vocab + sampled)
    parents = [[-1] + [0] * (nodes - 4) + [1, nodes - 4, nodes - 2]] * batch
    p, q = rows_of(g, batch * nodes, vocab, DTYPES[dtype])
    p, q = p.view(batch, nodes, vocab), q.view(batch, nodes, vocab)
    tree = tree_tensors(parents, packed)
    cu = ints([nodes * b for b in range(batch + 1)]) if packed else None
    shape = (batch * nodes,) if packed else (batch, nodes)
    lengths, in_last = set(), 0
    for trial in range(4):
        tokens = torch.stack([torch.tensor(drawn(rng, own, q[b])) for b, own in enumerate(parents)])
        if trial % 2 == 0:  # tokens of the last vector, one of them twice, and ones that the target hardly likes
            tokens[:, 1:6] = torch.tensor([vocab - 1, vocab - 2, vocab - 9, vocab - 1, vocab - 5])
            tokens[:, 6:9] = p[:, 0].float().topk(3, largest=False).indices
        u = torch.rand(batch, nodes, generator=g)
        if trial > 0:
            u[:2] = 0.9999  # (all rejected, or nearly)
        u[0, 0], u[1, 0], u[2, 0] = 1 - 2.0 ** -24, 0.98, 0.0
        path, accepted, token = verify_drafts(tree, tokens.view(shape).int().cuda(), p.view(*shape, vocab).cuda(),
                                              q.view(*shape, vocab).cuda() if sampled else None, u.view(shape).cuda(), cu)
        for b, own in enumerate(parents):
            want, following = R.verify(own, tokens[b].tolist(), p[b], q[b] if sampled else None, u[b].tolist())
            assert path[b].tolist() == want + [-1] * (path.shape[1] - len(want)), (trial, b)
            assert int(accepted[b]) == len(want) and int(token[b]) == following, (trial, b)
            lengths.add(len(want))
            in_last += following >= vocab - 9
    assert 1 in lengths and len(lengths) > 1 and in_last > 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_named_drafts_that_take_what_is_left(dtype):
    """Rows that sum to more than 1, whose likeliest tokens are rejected one after the other until S is below a token's."""
    from ring_swa import draft_tree, verify_drafts

    vocab = 2000
    dtype = {**DTYPES, "fp32": torch.float32}[dtype]
    row = torch.zeros(vocab)
    row[[7, 500, 1999, 1024]] = torch.tensor([0.75, 0.125, 0.3125, 0.25])
    parents, tokens = [-1, 0, 0, 0, 0, 0], [0, 7, 500, 3, 7, 1999]
    u = [[0.5, 0.9375, 0.96875, 0.0, 0.0, 1 - 2.0 ** -24],  # S: 1, 0.25, 0.125, .., and 0.3125 is taken
         [0.5, 0.9375, 0.25, 0.0, 0.0, 0.0],
         [0.5, 0.5, 0.0, 0.0, 0.0, 0.0]]
    target = row.to(dtype).expand(len(u), len(parents), vocab)
    path, accepted, token = verify_drafts(draft_tree(ints([parents] * len(u))), ints([tokens] * len(u)), target.cuda(), None,
                                          torch.tensor(u).cuda())
    for b in range(len(u)):
        want, following = R.verify(parents, tokens, target[b], None, u[b])
        assert path[b, :int(accepted[b])].tolist() == want and int(token[b]) == following
    assert path[:, 1].tolist() == [5, 2, 1]


@pytest.mark.parametrize("sampled", [True, False])
def test_the_last_of_many_elements(sampled):
    """The last sequences of a batch whose rows pass 2^31 elements, against the restatement."""
    from ring_swa import verify_drafts

    batch, nodes, vocab = 43, 27, 1999999
    assert (batch - 2) * nodes * vocab >= 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(4)
    parents = [[-1] + [max(0, i - 6) for i in range(1, nodes)]] * batch
    tree = tree_tensors(parents, False)
    p = torch.zeros(batch, nodes, vocab, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros_like(p) if sampled else None
    base = 3 * torch.randn(2, nodes, vocab, generator=g, device="cuda")
    for t in (p, q) if sampled else (p,):
        t[-2:] = torch.softmax(base + 0.5 * torch.randn(2, nodes, vocab, generator=g, device="cuda"), -1).bfloat16()
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g, device="cuda")
    tokens[-2:, 1:] = (q if sampled else p)[-2:, 0].float().topk(nodes - 1).indices
    u = torch.rand(batch, nodes, generator=g, device="cuda")
    u[-1, 1:4] = 0.9999
    got = verify_drafts(tree, tokens, p, q, u)
    for b in (-2, -1):
        want, following = R.verify(parents[b], tokens[b].tolist(), p[b], q[b] if sampled else None, u[b].tolist())
        assert got[0][b].tolist() == want + [-1] * (nodes - len(want)) and int(got[2][b]) == following
    assert got[1][:-2].tolist() == [1] * (batch - 2) and got[2][:-2].tolist() == [-1] * (batch - 2)  # (nothing in their rows)
