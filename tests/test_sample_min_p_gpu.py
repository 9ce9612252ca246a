"""min-p of 1 and above: kept are the tokens with weight at least min_p, the first one always.
The first token's weight is 1, so 1 keeps those that tie with it and any more keeps it alone."""

from __future__ import annotations

import math

import pytest
import torch

from nanoengine_amd import kernels

ABOVE = 1.0 + 2.0**-23


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab,ties", [(1, 1), (40, 3), (5000, 700), (50021, 50021), (50021, 6000)])
@pytest.mark.parametrize("k,p", [(0, 1.0), (0, 0.6), (2, 1.0), (20000, 0.9)])
def test_min_p_of_one_and_more_among_ties(dtype, vocab, ties, k, p):
    """Few and many tokens at the top, the many past what one work-group sorts at once."""
    g = torch.Generator().manual_seed(vocab + ties)
    x = torch.full((4, vocab), -2.0)
    for r in range(4):
        x[r, torch.randperm(vocab, generator=g)[:ties]] = 1.25
    first = x.argmax(1)
    u = torch.tensor([0.0, 0.3, 0.7, 1.0 - 2.0**-24], device="cuda")
    logits = x.to(dtype).cuda()
    tied = (x == 1.25).sum(1)  # the same number in each row
    n = int(tied[0]) if k == 0 else min(int(tied[0]), k)
    if p < 1:
        # top-p's share is of the first top-k's weight, ties and what follows them
        rest = (vocab if k == 0 else min(k, vocab)) - n
        n = min(n, math.ceil(p * (n + rest * math.exp(-3.25))))
    _, probs = kernels.sample(logits, u, top_k=k, top_p=p, min_p=1.0, probs=True)
    assert ((probs > 0).sum(1) == n).all()
    for m in (ABOVE, 1.5, 3e38, math.inf):
        tokens, probs = kernels.sample(logits, u, top_k=k, top_p=p, min_p=m, probs=True)
        assert tokens.cpu().tolist() == first.tolist()
        want = torch.zeros_like(probs).scatter_(1, first[:, None].cuda(), 1.0)
        assert torch.equal(probs, want)


@pytest.mark.gpu
def test_min_p_above_one_in_some_rows():
    vocab = 9000
    x = torch.zeros(6, vocab, dtype=torch.bfloat16, device="cuda")
    m = torch.tensor([0.0, 1.0, ABOVE, 2.0, math.nan, -1.0], device="cuda")
    u = torch.full((6,), 0.5, device="cuda")
    assert kernels.sample(x, u, min_p=m).tolist() == [4500, 4500, 0, 0, 4500, 4500]
