"""Rows of probabilities that do not sum to 1 (rounded to 16 bits, say): what the restated choice makes of them, by its formula."""
import math

import pytest
import torch

from oracle import drafts_oracle as R


def distribution(p, q, tokens):
    """The probability of each first token, for children that are `tokens` in order: drawn from norm(q), each, or (q None)
    named outright.  R.verify's formula with the uniforms' lengths in the place of draws."""
    n = p.numel()
    found = torch.zeros(n, dtype=torch.float64)
    for drafts in (tokens if q is None else torch.cartesian_prod(*[torch.arange(n)] * 2).tolist()):
        chance = 1.0 if q is None else math.prod(float(q[x] / q.sum()) for x in drafts)
        left, mass, a = p.clone(), 1.0, 0.0
        for x in drafts:
            wanted = mass * (1.0 if q is None else float(q[x]))
            take = 0.0 if left[x] <= 0 else min(1.0, float(left[x]) / wanted) if wanted > 0 else 1.0
            found[x] += chance * take
            chance *= 1 - take
            if q is None:
                mass = max(0.0, mass - float(left[x]))
                left[x] = 0
            else:
                a += mass
                left = torch.clamp(p - a * q, min=0)
                mass = float(left.sum())
        found += chance * (left / left.sum() if left.sum() > 0 else p / p.sum())
    return found


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("named", [True, False])
def test_off_by_what_the_sums_are(named, dtype):
    """In total variation at most what the target's sum and, for each of two draws, the draft's differ from 1.

    Named: a child has min(p, what is left of 1) instead of p / s with s the sum, the others what is left, shared as p is.  Drawn from
    q / t, t its sum: a child is reached with min(p, q) / t instead of min(p, q), and so on; what is left is normalised by its own
    sum, so that only chances are off, by |1 - 1 / t| a draw, and by |1 - s| at the first."""
    dtype = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)[dtype]
    g = torch.Generator().manual_seed(7)
    worst = 0.0
    for trial in range(60):
        n = 12 if not named else 400
        p, q = (torch.softmax(2.5 * torch.randn(n, generator=g, dtype=torch.float64), -1).to(dtype).double() for _ in range(2))
        if trial % 3 == 0:
            p = (p * (1 + 0.02 * (torch.rand(1, generator=g, dtype=torch.float64) - 0.5))).to(dtype).double()
        s, t = float(p.sum()), float(q.sum())
        tokens = [p.topk(7).indices.tolist()]
        off = 0.5 * float((distribution(p, None if named else q, tokens) - p / s).abs().sum())
        bound = abs(s - 1) / min(1, s) + (0 if named else 2 * abs(t - 1) / min(1, t))
        assert off <= bound + 1e-12, (trial, off, s, t)
        worst = max(worst, off)
    assert worst > 1e-4  # (rows whose sums are off do show)


def test_named_drafts_that_take_what_is_left():
    """S is 1 less what the rejected ones had, whatever the row's sum is: a child with that much or more is taken.  (So S stays above
    0: a rejected child has at most uniform * S, and uniforms are below 1.)"""
    p = torch.tensor([[0.75, 0.3125, 0.125, 0.0, 0.25]], dtype=torch.float64).expand(5, 5)
    below = 1 - 2.0 ** -24
    assert R.verify([-1, 0, 0], [0, 0, 1], p, None, [0.5, 0.9375, below]) == ([0, 2], 0)  # below * 0.25 < 0.3125
    assert R.verify([-1, 0, 0], [0, 0, 2], p, None, [0.5, 0.9375, below]) == ([0], 1)     # half of 0.3125 + 0.25 lies in 0.3125
    # a token without probability, one that was tried before, and one with what is left
    assert R.verify([-1, 0, 0, 0, 0], [0, 0, 3, 0, 4], p, None, [0.5, 0.9375, 0.0, 0.0, below]) == ([0, 4], 0)
    assert R.verify([-1, 0, 0, 0], [0, 0, 3, 0], p, None, [0.5, 0.9375, 0.0, 0.0])[0] == [0]
