"""Sampling from given uniforms (``kernels.sample``) against its definition in 64 bits.

The definition: tokens in order of logit (descending) then index; the first
min(n_k, n_p, n_m) are kept; the token is the first whose running weight exceeds u times
the kept weight.  Tokens have to be equal: the kernel's borders are within 2^-40 of the
64-bit ones, so a uniform between the two is met once in 10^11 draws.  A probability is
the 64-bit one rounded to fp32 (half a step, 2^-24 relative) up to the weights' own error:
a sum of integers that are each off by at most one half of 2^-45 of the largest weight
(2^18 of them: 2^-28 relative) and exponents whose argument, up to 2^9 sixteenths, is
rounded to 2^-53 (below 2^-40): 2^-24 + 2^-28 + 2^-40 < 1.1 * 2^-24 relative.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nanoengine_amd import kernels

PROB_REL = 1.1 * 2.0**-24
VOCAB = 151936


def reference_row(x: np.ndarray, u: float, t: float, k: int, p: float, m: float):
    """(token, indices kept in order, their probabilities) of one row of fp64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    x = np.minimum(x, np.finfo(np.float32).max)
    order = np.argsort(-x, kind="stable")
    n = int(np.count_nonzero(x > -np.inf))
    if n == 0:
        return -1, order[:0], np.zeros(0)
    if not t > 0:
        return int(order[0]), order[:1], np.ones(1)
    xs = x[order[:n]]
    w = np.exp((xs - xs[0]) / t)
    keep = min(n, k) if k > 0 else n
    mass = np.cumsum(w)
    if p < 1:
        keep = min(keep, 1 + int(np.searchsorted(mass[:keep], p * mass[keep - 1], side="left")))
    if m > 0:
        keep = min(keep, int(np.count_nonzero(w >= min(m, 1.0))))
    keep = max(keep, 1)
    total = mass[keep - 1]
    if not u > 0:
        at = 0
    else:
        at = min(int(np.searchsorted(mass[:keep], u * total, side="right")), keep - 1) if u < 1 else keep - 1
    return int(order[at]), order[:keep], w[:keep] / w[:keep].sum()


def check(logits, u, t=1.0, k=0, p=1.0, m=0.0, probs=True):
    """Runs both on ``logits`` (GPU) and compares every row's token and distribution."""
    rows, vocab = logits.shape
    got = kernels.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m, probs=probs)
    tokens, table = got if probs else (got, None)
    x = logits.double().cpu().numpy()
    value = lambda v, r, cast: cast(v[r]) if isinstance(v, torch.Tensor) else cast(np.float32(v) if cast is float else v)
    tokens, uu = tokens.cpu().tolist(), u.cpu().numpy()
    table = table.double().cpu().numpy() if probs else None
    for r in range(rows):
        want, kept, dist = reference_row(x[r], float(uu[r]), value(t, r, float), value(k, r, int), value(p, r, float),
                                         value(m, r, float))
        assert tokens[r] == want, (r, tokens[r], want, len(kept))
        if probs:
            full = np.zeros(vocab)
            full[kept] = dist
            assert not table[r][full == 0].any() and (table[r][full > 2e-45] > 0).all(), r  # fp32's smallest: 1.4e-45
            assert np.all(np.abs(table[r] - full) <= PROB_REL * full + 1e-44), r


def make_logits(rows, vocab, dtype, seed, spread=2.0, peaks=30):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    if peaks:
        at = torch.randint(0, vocab, (rows, peaks), generator=g)
        x.scatter_add_(1, at, 3.0 + 8.0 * torch.rand(rows, peaks, generator=g))
    return x.to(dtype).cuda(), torch.rand(rows, generator=g).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 63, 511, 4097, 32003])
def test_types_and_vocabularies(dtype, vocab):
    x, u = make_logits(9, vocab, dtype, vocab)
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.02), (1.3, 0, 0.7, 0.0), (0.6, 2000, 1.0, 0.0),
                       (1.0, 0, 1.0, 0.1), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, vocab, 0.5, 0.0)]:
        check(x, u, t, k, p, m)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("filters", [(0.8, 50, 0.95, 0.02), (0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.2, 5000, 0.99, 0.0),
                                     (1.0, 3000, 1.0, 1e-4), (0.7, 1024, 1.0, 0.0), (0.7, 1025, 0.8, 0.0)])
def test_a_language_models_rows(rows, filters):
    x, u = make_logits(rows, VOCAB, torch.bfloat16, rows)
    check(x, u, *filters, probs=rows < 70)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.1, 0.5])
def test_flat_rows(dtype, spread):
    """Nuclei of more tokens than the sorted list holds, bins of more, and runs of equal logits."""
    x, u = make_logits(4, 50021, dtype, 3, spread=spread, peaks=0)
    x += 1.5
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 30000, 0.6, 0.0), (1.0, 20, 1.0, 0.0), (1.0, 20, 0.5, 0.0),
                       (1.0, 0, 1.0, 0.7), (1.0, 0, 0.999, 0.95), (1.0, 700, 0.9, 0.5), (1.0, 0, 1.0, 1.0), (50.0, 0, 1.0, 0.99)]:
        check(x, u, t, k, p, m)


@pytest.mark.gpu
def test_equal_logits_split_exactly():
    """With equal logits token i is drawn for u in [i / V, (i + 1) / V), the borders included."""
    vocab = 8192
    u = torch.tensor([0.0, 0.25, 0.5, 4095 / 8192, 0.5 - 2.0**-25, 1 - 2.0**-24, 2.0**-13], device="cuda")
    x = torch.full((7, vocab), 0.3, device="cuda", dtype=torch.bfloat16)
    assert kernels.sample(x, u).tolist() == [0, 2048, 4096, 4095, 4095, 8191, 1]
    check(x, u, p=0.5)
    check(x, u, k=4096)


@pytest.mark.gpu
def test_ties_at_the_borders_go_to_the_lowest_index():
    x = torch.zeros(6, 5000, device="cuda", dtype=torch.bfloat16)
    x[:, 100:4000:7] = 2.0
    x[:, 3] = -0.0
    x[1, 4999] = 2.5
    u = torch.linspace(0, 0.999, 6, device="cuda")
    for k in (1, 5, 557, 558, 559, 600, 5000):
        check(x, u, k=k)
        check(x, u, k=k, p=0.37)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_infinite_and_nan_logits(dtype):
    x, u = make_logits(8, 3001, dtype, 5)
    x[0] = -math.inf  # nothing left
    x[1] = -math.inf
    x[1, 2999] = -3.0  # one token left
    x[2, ::2] = -math.inf
    x[3, 1::3] = math.nan
    x[4, [17, 900]] = math.inf  # these two share the row
    x[5] = torch.finfo(dtype).min  # masked with the type's lowest value
    x[5, 44] = 1.0
    x[6] = torch.finfo(dtype).min
    x[7] = math.nan
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.05), (1.0, 2000, 0.5, 0.0), (0.0, 0, 1.0, 0.0)]:
        check(x, u, t, k, p, m)
    assert kernels.sample(x, u)[0].item() == -1 and kernels.sample(x, u, 0.0)[7].item() == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale", [2.0**-14, 2.0**-7, 2.0**5, 2.0**9])
def test_logits_of_any_magnitude(dtype, scale):
    """Rows of tiny and huge logits, at the temperature that makes them ordinary ones, and rows with a few."""
    x, u = make_logits(6, 40000, torch.float32, 5)
    x = (x * scale).to(dtype)
    x[3:, ::977] = torch.randn_like(x[3:, ::977].float()).to(dtype) * 2.0  # among them
    for k, p, m in [(0, 1.0, 0.0), (50, 0.95, 0.02), (0, 0.8, 0.0), (3000, 0.99, 0.001)]:
        check(x, u, max(scale, 2.0**-7), k, p, m)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_zeros_of_either_sign_are_equal(dtype):
    g = torch.Generator().manual_seed(8)
    x = torch.where(torch.rand(5, 3000, generator=g) < 0.5, 0.0, -0.0).to(dtype)
    x[1:, : 40 * 5 : 1] = -math.inf
    x[2:][torch.rand(3, 3000, generator=g) < 0.99] = -math.inf
    u = torch.rand(5, generator=g).cuda()
    for t, k, p, m in [(0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (0.7, 5, 0.8, 0.1), (1.0, 0, 1.0, 1.0)]:
        check(x.cuda(), u, t, k, p, m)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("p", [1.0, 0.97])
def test_min_p_among_tokens_of_no_weight(dtype, p):
    """Steps of e^-20 among many tokens: min-p keeps the second and cuts the third, whose weight no sum holds."""
    g = torch.Generator().manual_seed(3)
    x = -torch.randint(0, 4, (3, 30000), generator=g).to(dtype).cuda()
    for m in (1e-9, 1e-8, 1e-17, 1e-18, 1e-30):
        for k in (0, 20000):
            check(x, torch.rand(3, generator=g).cuda(), 0.05, k, p, m)


@pytest.mark.gpu
def test_uniforms_off_their_range():
    x, _ = make_logits(5, 4000, torch.bfloat16, 8)
    check(x, torch.tensor([-1.0, 1.0, 7.5, math.inf, math.nan], device="cuda"), 0.9, 30, 0.9, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1e-30, 1e-6, 0.01, 30.0, 1e6])
def test_temperatures(t):
    x, u = make_logits(6, 20000, torch.float32, 9)
    x[2, 5] = x[2].max()  # a tie at the top
    check(x, u, t, 0, 1.0, 0.0)
    check(x, u, t, 900, 0.9, 0.01)


@pytest.mark.gpu
def test_rows_of_their_own_parameters():
    rows = 40
    x, u = make_logits(rows, 40000, torch.bfloat16, 11)
    g = torch.Generator().manual_seed(1)
    t = (0.3 + torch.rand(rows, generator=g)).cuda()
    t[::5] = 0.0
    t[3], t[4] = -1.0, math.nan  # greedy
    k = torch.randint(-1, 3000, (rows,), generator=g).to(torch.int32).cuda()
    p = (0.2 + torch.rand(rows, generator=g)).cuda()
    p[7] = 0.0
    m = (0.1 * torch.rand(rows, generator=g)).cuda()
    m[::3] = 0.0
    check(x, u, t, k, p, m)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,stride", [(1, 1003), (3, 1100), (8, 2048), (7, 1001)])
def test_rows_off_the_vector_grid(dtype, offset, stride):
    """Views whose rows start and end inside 16-byte vectors; what lies around them is not read into a row."""
    store = torch.full((11 * stride + 64,), 1e4, device="cuda", dtype=dtype)
    x, u = make_logits(11, 990, dtype, 12)
    view = store[offset:].as_strided((11, 990), (stride, 1))
    view.copy_(x)
    check(view, u, 0.9, 0, 0.9, 0.0)
    check(view, u, 0.9, 40, 1.0, 0.0)
    # and the distribution into a strided table, its surroundings left alone
    table = torch.full((11, 1000), -1.0, device="cuda")
    kernels.sample(view, u, 0.9, probs=table[:, 3:993])
    assert torch.equal(table[:, 3:993], kernels.sample(view, u, 0.9, probs=True)[1])
    assert (table[:, :3] == -1).all() and (table[:, 993:] == -1).all()


@pytest.mark.gpu
def test_many_rows_share_the_workspace_in_batches():
    x, u = make_logits(2500, 300, torch.float16, 13)
    check(x, u, 1.0, 40, 0.9, 0.0)


@pytest.mark.gpu
def test_same_bits_every_time_and_in_a_replayed_graph():
    x, u = make_logits(33, 30000, torch.bfloat16, 14)
    first = kernels.sample(x, u, 1.1, 0, 0.97, 0.0, probs=True)
    out, table = torch.empty_like(first[0]), torch.empty_like(first[1])
    graph = torch.cuda.CUDAGraph()
    kernels.sample(x, u, 1.1, 0, 0.97, 0.0, out=out, probs=table)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kernels.sample(x, u, 1.1, 0, 0.97, 0.0, out=out, probs=table)
    for seed in range(4):
        y, v = make_logits(33, 30000, torch.bfloat16, 20 + seed)
        x.copy_(y)
        u.copy_(v)
        out.zero_()
        table.zero_()
        graph.replay()
        eager = kernels.sample(x, u, 1.1, 0, 0.97, 0.0, probs=True)
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(table, eager[1])
        again = kernels.sample(x, u, 1.1, 0, 0.97, 0.0, probs=True)
        assert torch.equal(again[0], eager[0]) and torch.equal(again[1], eager[1])


@pytest.mark.gpu
def test_streams_and_concurrent_calls():
    a, ua = make_logits(64, 50000, torch.bfloat16, 15)
    b, ub = make_logits(64, 50000, torch.bfloat16, 16)
    want = kernels.sample(a, ua, 0.9, 0, 0.9), kernels.sample(b, ub, 0.9, 0, 0.9)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s, x, u in zip(streams, (a, b), (ua, ub)):
            with torch.cuda.stream(s):
                got.append(kernels.sample(x, u, 0.9, 0, 0.9))
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        assert torch.equal(t, want[i % 2])


@pytest.mark.gpu
def test_the_distribution_feeds_sampled_acceptance():
    """probs rows are what accept takes as draft_probs: a guess drawn from them is kept with
    probability min(1, p / q); with q = p every guess is kept."""
    x, u = make_logits(8, 5000, torch.bfloat16, 17)
    tokens, probs = kernels.sample(x, u, 0.8, probs=True)
    target = torch.stack([x, x], 1).reshape(16, 5000).contiguous()
    zeros = lambda dtype: torch.zeros(8, dtype=dtype, device="cuda")
    out, kept = kernels.accept(
        tokens[:, None].contiguous(), torch.ones(8, dtype=torch.int32, device="cuda"),
        torch.arange(0, 16, 2, dtype=torch.int32, device="cuda"), 5000, logits=target, temperature=0.8,
        seeds=zeros(torch.int64) + 5, steps=zeros(torch.int64),
        draft_probs=probs, draft_row_start=torch.arange(8, dtype=torch.int32, device="cuda"))
    # p / q differs from 1 by the two sides' fp32 roundings at most: below it u < p / q all but surely
    assert torch.equal(out[:, 0], tokens) and (kept == 2).all()


@pytest.mark.gpu
def test_empty_batch():
    x = torch.empty(0, 50, device="cuda", dtype=torch.bfloat16)
    assert kernels.sample(x, torch.empty(0, device="cuda")).shape == (0,)


@pytest.mark.gpu
def test_refusals():
    x, u = make_logits(4, 1000, torch.bfloat16, 18)
    for bad in (dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(top_p=math.nan),
                dict(min_p=math.nan), dict(temperature=torch.ones(3, device="cuda")),
                dict(top_k=torch.ones(4, device="cuda")), dict(top_p=torch.ones(4, device="cuda", dtype=torch.float64)),
                dict(out=torch.empty(4, dtype=torch.int64, device="cuda")),
                dict(probs=torch.empty(4, 999, device="cuda")),
                dict(workspace=torch.empty(16, device="cuda"))):
        with pytest.raises(ValueError):
            kernels.sample(x, u, **bad)
    with pytest.raises(ValueError):
        kernels.sample(x, u[:3])
    with pytest.raises(ValueError):
        kernels.sample(x.t(), u)
    with pytest.raises(ValueError):
        kernels.sample(x.to(torch.float64), u)
    with pytest.raises(ValueError):  # a vocabulary past the kernel's bound
        kernels.sample(torch.empty(1, (1 << 20) + 1, device="cuda", dtype=torch.bfloat16), u[:1])
    with pytest.raises(RuntimeError, match="NE_EWORKSPACE"):
        kernels.sample(x, u, workspace=torch.empty(256, device="cuda", dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        kernels.sample(x.cpu(), u.cpu())
