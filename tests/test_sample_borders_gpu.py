"""Sampling where a border falls next to a special value: ``kernels.sample`` against the order
of tokens itself, on rows whose kept tokens follow from a count."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nanoengine_amd import kernels


def first_tokens(x: np.ndarray, n: int) -> np.ndarray:
    """The first ``n`` tokens by logit (descending), then index; zeros of either sign are equal."""
    return np.argsort(-(x.astype(np.float64) + 0.0), kind="stable")[:n]


@pytest.mark.gpu
@pytest.mark.parametrize("zero", [0.0, -0.0])
@pytest.mark.parametrize("zeros,negatives,top_k", [(3000, 3900, 6000), (3000, 5000, 6000), (100, 4100, 3000), (5000, 5000, 5003)])
def test_a_border_among_subnormal_numbers_below_zero(zero, zeros, negatives, top_k):
    """More tokens next to zero than are sorted at once: the range of keys that holds the border
    ends between the negative numbers and zero."""
    rng = np.random.default_rng(zeros + negatives)
    close = np.array([0x3C7FFFFF], np.uint32).view(np.float32)  # its key is whole buckets above zero's
    row = np.concatenate([[100.0], close, np.full(zeros, zero), np.full(negatives, -1e-40)]).astype(np.float32)
    x = np.stack([rng.permutation(row) for _ in range(3)])
    u = torch.tensor([0.0, 0.5, 0.999], device="cuda")
    logits = torch.from_numpy(x).cuda()
    tokens, probs = kernels.sample(logits, u, top_k=top_k, probs=True)
    # e^-100 for all but the first: below fp32's steps, so the first token is drawn ...
    assert tokens.tolist() == [int(r.argmax()) for r in x]
    for r in range(3):
        kept = np.zeros(row.size, bool)
        kept[first_tokens(x[r], top_k)] = True
        # ... and e^-100, 3.7e-44, is what the others' probabilities hold
        assert np.array_equal(probs[r].cpu().numpy() > 0, kept)
    # the hundred left out, the rest is drawn evenly: token floor(u n) of the order
    logits[logits == 100.0] = -torch.inf
    tokens, probs = kernels.sample(logits, u, top_k=top_k, probs=True)
    x[x == 100.0] = -np.inf
    n = min(top_k, zeros + negatives + 1)
    for r in range(3):
        order = first_tokens(x[r], n)
        kept = np.zeros(row.size, bool)
        kept[order] = True
        assert np.array_equal(probs[r].cpu().numpy() > 0, kept)
        w = np.exp(x[r][order].astype(np.float64))
        want = np.searchsorted(np.cumsum(w), float(u[r]) * w.sum(), side="right")
        assert tokens[r].item() == order[want]


# (tokens of 1.1, tokens of 1.0, top-p): the first kind's end is where top-p ends, to within a unit of
# the integer weights per token, and the two ways of adding up the second kind lie on either side of it
@pytest.mark.gpu
@pytest.mark.parametrize("more,less,top_p", [(3993, 10145, 0.3178494870662689), (3942, 7020, 0.39943596720695496),
                                             (3919, 12403, 0.2723730206489563), (3718, 11151, 0.28358253836631775),
                                             (3652, 10841, 0.2858269512653351)])
def test_a_top_p_share_next_to_a_bins_end(more, less, top_p):
    """The share of the first top-k is found from a histogram, then from the exact weight: whichever
    token that makes the last, it is next to the end of the tokens of 1.1."""
    vocab, parts = 20480, 6
    x = np.full(vocab, -np.inf, np.float32)
    x[0] = 5.0  # alone in its part of the row, so that the others' weights are brought to its base
    first = [80 * c // parts * 256 for c in range(parts)] + [vocab]
    for c in range(parts - 1):
        a, b = (n // 5 + (c < n % 5) for n in (more, less))
        at = first[c + 1]
        assert at + a + b < first[c + 2]
        x[at : at + a], x[at + a : at + a + b] = 1.1, 1.0
    x[vocab - 1] = -5.0  # one token past top-k
    logits, u = torch.from_numpy(x[None]).cuda(), torch.tensor([0.999999], device="cuda")
    kept = set()
    for _ in range(8):
        token, probs = kernels.sample(logits, u, 0.77, 1 + more + less, top_p, probs=True)
        kept.add(int((probs > 0).sum()))
        assert x[int(token)] == np.float32(1.1) or int((probs > 0).sum()) == 2 + more
    assert len(kept) == 1 and kept <= {1 + more, 2 + more}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("u", [1.0, 7.5, float("inf")])
def test_uniforms_of_one_and_more_take_the_last_kept_token(dtype, u):
    """Also where the tokens before it hold all the weight that any sum can hold."""
    rng = np.random.default_rng(4)
    rows = [np.array([0.0, -200.0]), np.array([-200.0, 3.0, -210.0, -210.0]),
            rng.permutation(np.concatenate([[40.0], np.zeros(300), np.full(80, -60.0)])),
            rng.permutation(np.concatenate([np.full(9000, 1.0), np.full(50, -90.0)])),
            rng.permutation(np.concatenate([np.full(9000, 1.0), np.full(7000, -90.0)])),
            rng.permutation(np.concatenate([[60.0], rng.normal(size=20000)])), rng.normal(size=30000)]
    uniform = torch.tensor([u], device="cuda")
    for row in rows:
        logits = torch.from_numpy(row[None]).to(dtype).cuda()
        x = logits.float().cpu().numpy()[0]
        order = first_tokens(x, x.size)
        n = x.size
        for k in {0, 2, n - 1, n // 2 + 1}:
            kept = n if k in (0, n) or k > n else max(k, 1)
            assert kernels.sample(logits, uniform, top_k=k).item() == order[kept - 1], (n, k)
        # min-p: those within 30 of the first, none of these rows has a logit near that border
        near = int((x >= x.max() - 30.0).sum())
        assert kernels.sample(logits, uniform, min_p=float(np.exp(-30.0))).item() == order[near - 1], n


@pytest.mark.gpu
@pytest.mark.parametrize("less", [4500, 9000, 16000])
def test_a_uniform_of_one_where_the_histogram_holds_less_than_the_sum(less):
    """The last kept token by its rank, whatever units the histogram dropped."""
    vocab, parts = 20480, 6
    x = np.full(vocab, -np.inf, np.float32)
    x[0] = 5.0
    first = [80 * c // parts * 256 for c in range(parts)]
    for c in range(parts - 1):
        x[first[c + 1] : first[c + 1] + less // 5] = 1.0
    x[vocab - 1] = -16.0  # past top-k: of no weight
    token = kernels.sample(torch.from_numpy(x[None]).cuda(), torch.ones(1, device="cuda"), 0.77, 1 + less)
    assert token.item() == np.flatnonzero(x == 1.0)[-1]
