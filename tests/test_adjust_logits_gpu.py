"""Penalties, biases and masks on logits against their definition in 64 bits.

The kernel computes x1 (one rounding), f c and f c + p (one each), x2 and x3 (one each) in fp32, then
rounds to the output's type: |got - x3| <= 2^-24 (|x1| + 2 (|f c| + |p|) + |x2| + |x3|) * 1.01 + half a
step of the output (bf16 2^-8, fp16 2^-11, fp32 2^-24 of |x3|, and fp16's least step 2^-25).
Infinities and NaN have to be in the same places.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from nanoengine_amd import _native, kernels

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def parameter(value, row: int) -> float:
    return float(value[row]) if isinstance(value, torch.Tensor) else float(np.float32(value))


def reference(logits, penalties=None, bias=None, allowed=None, allowed_rows=None):
    """(values, the fp32 steps' bound) in 64 bits, row by row."""
    x = logits.double().cpu().numpy().copy()
    bound = np.zeros_like(x)
    rows, vocab = x.shape
    for r in range(rows):
        if penalties is not None:
            b = r if penalties.row_seq is None else int(penalties.row_seq[r])
            tokens, made = [], []
            if 0 <= b < penalties.history.shape[0]:
                n = min(max(int(penalties.history_len[b]), 0), penalties.history.shape[1])
                tokens = penalties.history[b, :n].tolist()
                made = tokens[max(0, int(penalties.prompt_len[b])) if penalties.prompt_len is not None else 0 :]
                if penalties.drafts is not None:
                    extra = penalties.drafts[b, : max(0, int(penalties.row_drafts[r]))].tolist()
                    tokens, made = tokens + extra, made + extra
            rep, pres, freq = (parameter(v, r) for v in (penalties.repetition, penalties.presence, penalties.frequency))
            rep = rep if 0 < rep < np.inf else 1.0
            pres, freq = (0.0 if v != v else v for v in (pres, freq))
            for t in {t for t in tokens if 0 <= t < vocab}:
                c = made.count(t)
                with np.errstate(invalid="ignore"):
                    x[r, t] = x[r, t] / rep if x[r, t] > 0 else x[r, t] * rep
                    bound[r, t] += abs(x[r, t])
                    if c:
                        x[r, t] -= freq * c + pres
                        bound[r, t] += 2 * (abs(freq * c) + abs(pres)) + abs(x[r, t])
        if bias is not None:
            entries = {}
            for i in range(int(bias.start[r]), int(bias.start[r + 1])):
                entries[int(bias.tokens[i])] = float(bias.values[i])
            for t, v in entries.items():
                if 0 <= t < vocab:
                    x[r, t] += v
                    bound[r, t] += abs(x[r, t])
        if allowed is not None:
            which = r if allowed_rows is None else int(allowed_rows[r])
            if which >= 0:
                bits = np.zeros(vocab, bool)
                if which < allowed.shape[0]:
                    raw = allowed[which].cpu().numpy().view(np.uint8)
                    bits = np.unpackbits(raw, bitorder="little")[:vocab].astype(bool)
                x[r, ~bits] = -np.inf
                bound[r, ~bits] = 0
    return x, bound * 2.0**-24 * 1.01


def check(got, logits, **kw) -> None:
    want, bound = reference(logits, **kw)
    value = got.double().cpu().numpy()
    assert value.shape == want.shape
    assert np.array_equal(np.isnan(value), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(value[inf], want[inf])
    fine = np.isfinite(want)
    half = HALF_STEP[got.dtype] * np.abs(want[fine]) + (2.0**-25 if got.dtype == torch.float16 else 1e-45)
    assert (np.abs(value[fine] - want[fine]) <= bound[fine] * (1 + 2.0**-7) + half).all()


def make_penalties(rows, vocab, seqs=None, capacity=40, seed=0, drafts=0, prompt=True, scalar=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    seqs = rows if seqs is None else seqs
    u = lambda *shape: torch.rand(shape, device="cuda", generator=g)
    # a few tokens again and again, and some outside the vocabulary
    history = (u(seqs, capacity).pow(3) * (vocab + 2)).int() - 1
    length = (u(seqs) * (capacity + 2)).int()  # up to one past the capacity
    if seqs > 1:
        length[1] = 0
    kw = {}
    if drafts:
        kw = dict(drafts=(u(seqs, drafts) * vocab).int(), row_drafts=(u(rows) * (drafts + 1)).int(),
                  row_seq=(u(rows) * seqs).int())
    if scalar:
        return kernels.TokenPenalties(history, length, None, 1.25, 0.5, 0.125, **kw)
    return kernels.TokenPenalties(history, length, (length * u(seqs)).int() if prompt else None, 0.5 + u(rows), 2 * u(rows) - 0.5,
                                  u(rows), **kw)


def make_bias(rows, vocab, each, seed=0):
    g = torch.Generator().manual_seed(seed)
    dicts = [{int(t): float(v) for t, v in zip(torch.randint(0, vocab, (each,), generator=g), 4 * torch.randn(each, generator=g))}
             if r % 3 != 1 else None for r in range(rows)]
    return kernels.TokenBias.from_dicts(dicts, torch.device("cuda"))


def make_logits(rows, vocab, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (4 * torch.randn(rows, vocab, device="cuda", generator=g)).to(DTYPES[dtype])


def make_mask(rows, vocab, share, seed=0):
    g = torch.Generator().manual_seed(seed)
    return kernels.allowed_mask([torch.nonzero(torch.rand(vocab, generator=g) < share).flatten().tolist() for _ in range(rows)],
                                vocab, torch.device("cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 7), (3, 8), (2, 33), (5, 300), (3, 8191), (2, 8192), (2, 8193), (3, 32003)])
def test_everything_at_once(rows, vocab, dtype, out):
    logits = make_logits(rows, vocab, dtype)
    kw = dict(penalties=make_penalties(rows, vocab), bias=make_bias(rows, vocab, min(5, vocab)), allowed=make_mask(rows, vocab, 0.7))
    target = torch.full((rows, vocab), 5.0, device="cuda", dtype=DTYPES[out])
    got = kernels.adjust_logits(logits, out=target, **kw)
    assert got is target
    check(got, logits, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("penalty,bias,mask", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1), (0, 0, 0)])
@pytest.mark.parametrize("place", ["new", "in place"])
def test_each_part(penalty, bias, mask, place):
    rows, vocab = 6, 20011
    logits = make_logits(rows, vocab, "bf16", seed=3)
    kw = dict(penalties=make_penalties(rows, vocab, prompt=False) if penalty else None,
              bias=make_bias(rows, vocab, 50) if bias else None, allowed=make_mask(rows, vocab, 0.02) if mask else None)
    given = logits.clone()
    got = kernels.adjust_logits(given, out=given if place == "in place" else None, **kw)
    assert (got is given) == (place == "in place")
    if place == "new":
        assert torch.equal(given, logits)
    check(got, logits, **kw)


@pytest.mark.gpu
def test_scalars_and_full_vocabulary():
    rows, vocab = 4, 151936
    logits = make_logits(rows, vocab, "bf16")
    p = make_penalties(rows, vocab, capacity=3000, scalar=True)
    check(kernels.adjust_logits(logits, penalties=p), logits, penalties=p)


@pytest.mark.gpu
@pytest.mark.parametrize("capacity", [0, 1, 3, 255, 513, 2048, 2304, 5001, 8192, 10500, 32767, 32768, 70000])
def test_history_lengths(capacity):
    rows, vocab = 3, 9000
    logits = make_logits(rows, vocab, "fp32")
    p = make_penalties(rows, vocab, capacity=capacity, seed=capacity)
    check(kernels.adjust_logits(logits, penalties=p), logits, penalties=p)


@pytest.mark.gpu
@pytest.mark.parametrize("capacity", [6000, 40000])
@pytest.mark.parametrize("length", [1, 2, 255, 256, 257, 2047, 2049, 4096, 4100, 5999])
def test_prompts_that_end_anywhere(length, capacity):
    """One token again and again at both ends of the vocabulary's ranges, and tokens far outside it."""
    vocab = 16389
    g = torch.Generator(device="cuda").manual_seed(length)
    pool = torch.tensor([0, 4095, 4096, 8191, 8192, 16388, 16389, -1, -(2**31), 2**31 - 1, 2**30 + 5], dtype=torch.int32, device="cuda")
    history = pool[torch.randint(0, 11, (8, capacity), device="cuda", generator=g)]
    prompts = torch.tensor([0, 1, length // 2, length - 1, length, length + 1, 250, -3], dtype=torch.int32, device="cuda")
    p = kernels.TokenPenalties(history, torch.full((8,), length, dtype=torch.int32, device="cuda"), prompts, 1.5, 0.25, 0.125)
    logits = make_logits(8, vocab, "bf16", seed=length)
    check(kernels.adjust_logits(logits, penalties=p), logits, penalties=p)


@pytest.mark.gpu
def test_rows_of_a_verify_step():
    """Several rows per sequence, each with the guesses before it; rows without a sequence have no history."""
    rows, vocab = 40, 5000
    logits = make_logits(rows, vocab, "bf16")
    p = make_penalties(rows, vocab, seqs=7, drafts=4)
    p.row_seq[5], p.row_seq[6], p.row_drafts[8] = -1, 7, -3
    check(kernels.adjust_logits(logits, penalties=p), logits, penalties=p)


@pytest.mark.gpu
def test_guesses_without_any_history():
    logits = make_logits(4, 64, "fp32")
    dev = dict(device="cuda", dtype=torch.int32)
    p = kernels.TokenPenalties(torch.empty(2, 0, **dev), torch.zeros(2, **dev), presence=1.0,
                               drafts=torch.tensor([[3, 4, 3], [5, 6, 63]], **dev), row_seq=torch.tensor([0, 0, 1, 1], **dev),
                               row_drafts=torch.tensor([0, 3, 1, 3], **dev))
    check(kernels.adjust_logits(logits, penalties=p), logits, penalties=p)


@pytest.mark.gpu
def test_parameters_that_turn_a_penalty_off():
    rows, vocab = 6, 500
    logits = make_logits(rows, vocab, "fp32")
    p = make_penalties(rows, vocab, prompt=False)
    p.history_len.fill_(40)
    p.repetition.copy_(torch.tensor([0.0, -1.0, float("nan"), float("inf"), 2.0, 1.0]))
    p.presence.copy_(torch.tensor([float("nan"), 0.0, 0.0, 0.0, 0.0, 1.0]))
    p.frequency.copy_(torch.tensor([0.0, float("nan"), 0.0, 0.0, 0.0, -1.0]))
    got = kernels.adjust_logits(logits, penalties=p)
    check(got, logits, penalties=p)
    assert torch.equal(got[:4], logits[:4]) and not torch.equal(got[4], logits[4])


@pytest.mark.gpu
def test_a_token_listed_twice_takes_its_last_bias():
    logits = torch.zeros(2, 20000, device="cuda")
    i32 = dict(device="cuda", dtype=torch.int32)
    tokens = torch.tensor([5, 19999, 5, 7, -1, 20000, 5], **i32)
    bias = kernels.TokenBias(torch.tensor([0, 4, 7], **i32), tokens, torch.arange(1.0, 8.0, device="cuda"))
    got = kernels.adjust_logits(logits, bias=bias)
    assert got[0, 5] == 3 and got[0, 19999] == 2 and got[0, 7] == 4 and got[1, 5] == 7
    assert int((got != 0).sum()) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9000, 30001])
@pytest.mark.parametrize("penalty", [False, True])
def test_lists_of_many_biases(vocab, penalty):
    """More entries than 16 bits count, most of them for a token that is listed again."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = make_logits(3, vocab, "bf16")
    tokens = (torch.rand(66500, device="cuda", generator=g) * vocab).int()
    start = torch.tensor([0, 700, 66400, 66500], device="cuda", dtype=torch.int32)
    bias = kernels.TokenBias(start, tokens, 4 * torch.randn(66500, device="cuda", generator=g))
    kw = dict(bias=bias, penalties=make_penalties(3, vocab) if penalty else None)
    check(kernels.adjust_logits(logits, **kw), logits, **kw)
    # the same lists, each in a call of its own
    for row in range(3):
        a, b = int(start[row]), int(start[row + 1])
        one = kernels.TokenBias(torch.tensor([0, b - a], device="cuda", dtype=torch.int32), tokens[a:b], bias.values[a:b])
        if not penalty:
            whole = kernels.adjust_logits(logits, bias=bias)
            assert torch.equal(kernels.adjust_logits(logits[row : row + 1], bias=one), whole[row : row + 1])


@pytest.mark.gpu
def test_infinities_and_nan_and_rows_that_allow_nothing():
    vocab = 700
    logits = make_logits(4, vocab, "fp32")
    logits[:, 10], logits[:, 11], logits[:, 12] = float("nan"), float("inf"), -float("inf")
    i32 = dict(device="cuda", dtype=torch.int32)
    p = kernels.TokenPenalties(torch.tensor([[10, 11, 12]] * 4, **i32), torch.full((4,), 3, **i32), repetition=2.0, presence=1.0)
    mask = kernels.allowed_mask([None, [11, 13], [], [10]], vocab, torch.device("cuda"))
    got = kernels.adjust_logits(logits, penalties=p, allowed=mask)
    check(got, logits, penalties=p, allowed=mask)
    assert got[0, 10].isnan() and got[0, 11] == float("inf") and (got[2] == -float("inf")).all()
    # the sampler: nothing allowed gives -1, a NaN is never drawn
    tokens = kernels.sample(got[1:], torch.full((3,), 0.5, device="cuda"))
    assert tokens.tolist() == [11, -1, -1]


@pytest.mark.gpu
def test_masks_by_row_index():
    rows, vocab = 6, 1000
    logits = make_logits(rows, vocab, "bf16")
    mask = make_mask(2, vocab, 0.3)
    index = torch.tensor([1, 0, -1, 1, 2, -7], device="cuda", dtype=torch.int32)
    got = kernels.adjust_logits(logits, allowed=mask, allowed_rows=index)
    check(got, logits, allowed=mask, allowed_rows=index)
    assert torch.equal(got[2], logits[2]) and (got[4] == -float("inf")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_what_lies_beside_the_rows(dtype):
    rows, vocab = 5, 8200
    base = make_logits(rows, vocab + 3, dtype)
    logits = base[:, 1 : vocab + 1]
    buffer = torch.full((rows + 2, vocab + 5), 9.0, device="cuda", dtype=DTYPES[dtype])
    p = make_penalties(rows, vocab)
    wide = torch.full((rows, 50), 3, device="cuda", dtype=torch.int32)
    wide[:, :40] = p.history
    p = kernels.TokenPenalties(wide[:, :40], p.history_len, p.prompt_len, p.repetition, p.presence, p.frequency)
    kw = dict(penalties=p, allowed=make_mask(rows, vocab, 0.5))
    got = kernels.adjust_logits(logits, out=buffer[1 : rows + 1, 2 : vocab + 2], **kw)
    check(got, logits, **kw)
    buffer[1 : rows + 1, 2 : vocab + 2] = 9.0
    assert (buffer == 9.0).all()
    want = kernels.adjust_logits(logits, **kw)
    kernels.adjust_logits(logits, out=logits, **kw)
    assert torch.equal(logits, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab,capacity,drafts", [(8193, 1, 0), (8193, 509, 3), (9001, 0, 4), (9001, 341, 0), (9001, 342, 0),
                                                   (20000, 1249, 0), (20000, 1250, 0), (87377, 5457, 4), (87377, 5458, 4),
                                                   (87377, 5461, 0), (151936, 2048, 4), (151936, 6000, 0)])
@pytest.mark.parametrize("few", [False, True])
def test_in_place_under_penalties_alone(vocab, capacity, drafts, few, dtype):
    """A row's own tokens in one table (many rows): tokens again and again, all different, none and outside
    the vocabulary; the same bits as into other memory."""
    rows, ld = 9 if few else 520 // -(-vocab // 8192) + 1, vocab + 5
    g = torch.Generator(device="cuda").manual_seed(capacity)
    p = make_penalties(rows, vocab, seqs=5, capacity=capacity, seed=capacity, drafts=drafts) if drafts else \
        make_penalties(rows, vocab, capacity=capacity, seed=capacity)
    p.history_len[0] = capacity
    p.history_len[2:4] = capacity
    if capacity:
        p.history[2] = torch.randperm(vocab + 7, device="cuda", generator=g)[:capacity].int() - 3
        p.history[3] = vocab - 1
    if drafts:
        p.row_seq[1], p.row_drafts[2], p.row_seq[:1] = 9, -1, 3
    base = make_logits(rows, ld, dtype, seed=vocab)
    base[:, 7], base[:, vocab - 1] = float("inf"), float("nan")
    logits = base[:, 2 : vocab + 2]
    want = kernels.adjust_logits(logits, penalties=p)
    if capacity < 400 and few:
        check(want, logits, penalties=p)
    inside = base.clone()
    view = inside[:, 2 : vocab + 2]
    assert kernels.adjust_logits(view, penalties=p, out=view) is view
    assert torch.equal(view.nan_to_num(123.0), want.nan_to_num(123.0))
    inside[:, 2 : vocab + 2] = logits
    assert torch.equal(inside.nan_to_num(123.0), base.nan_to_num(123.0))  # nothing beside the rows


@pytest.mark.gpu
def test_in_place_call_replayed():
    rows, vocab = 200, 30000
    p = make_penalties(rows, vocab, seqs=4, capacity=500, drafts=4)
    logits = make_logits(rows, vocab, "bf16")
    graph = torch.cuda.CUDAGraph()
    kernels.adjust_logits(logits, penalties=p, out=logits)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kernels.adjust_logits(logits, penalties=p, out=logits)
    for seed in range(4):
        fresh = make_logits(rows, vocab, "bf16", seed=seed)
        logits.copy_(fresh)
        p.history_len.random_(0, 501)
        p.row_drafts.random_(0, 5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, kernels.adjust_logits(fresh, penalties=p))


@pytest.mark.gpu
def test_logits_past_32_bit_offsets():
    """2.3 10^9 logits, in place and not: the rows around the limits against their definition."""
    rows, vocab = 15_000, 151_936
    base = make_logits(8, vocab, "bf16", seed=9)
    logits = base.repeat(rows // 8, 1)
    p = make_penalties(rows, vocab, capacity=300, seed=9)
    before = logits.clone()
    got = kernels.adjust_logits(logits, penalties=p)
    assert torch.equal(logits, before)
    del before
    kernels.adjust_logits(logits, penalties=p, out=logits)
    for row in (0, (1 << 31) // vocab, rows - 1):
        one = slice(row, row + 1)
        part = kernels.TokenPenalties(p.history[one], p.history_len[one], p.prompt_len[one], p.repetition[one], p.presence[one],
                                      p.frequency[one])
        check(got[one], base[row % 8 : row % 8 + 1], penalties=part)
        assert torch.equal(got[one], logits[one])
    assert torch.equal(got, logits)


@pytest.mark.gpu
def test_captured_call_follows_its_inputs():
    rows, vocab = 8, 30000
    logits = make_logits(rows, vocab, "bf16")
    p = make_penalties(rows, vocab, capacity=900)
    mask = make_mask(rows, vocab, 0.5)
    out = torch.empty(rows, vocab, device="cuda")
    graph = torch.cuda.CUDAGraph()
    kernels.adjust_logits(logits, penalties=p, allowed=mask, out=out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kernels.adjust_logits(logits, penalties=p, allowed=mask, out=out)
    stream = torch.cuda.Stream()
    for seed in range(4):
        logits.copy_(make_logits(rows, vocab, "bf16", seed=seed + 50))
        p.history_len.random_(0, 900)
        p.prompt_len.copy_(p.history_len // 3)
        mask.bitwise_not_()
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            eager = kernels.adjust_logits(logits, penalties=p, allowed=mask, out=torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager)
        check(eager, logits, penalties=p, allowed=mask)


@pytest.mark.gpu
def test_no_rows_and_no_entries():
    logits = make_logits(3, 100, "bf16")
    assert kernels.adjust_logits(logits[:0]).shape == (0, 100)
    bias = kernels.TokenBias.from_dicts([None, {}, None], torch.device("cuda"))
    assert torch.equal(kernels.adjust_logits(logits, bias=bias), logits)


@pytest.mark.gpu
def test_wrapper_refuses_what_the_kernel_does_not_take():
    dev = torch.device("cuda")
    logits = make_logits(3, 100, "bf16")
    p = make_penalties(3, 100)
    i32 = dict(device="cuda", dtype=torch.int32)

    def refused(error=ValueError, logits=logits, **kw):
        with pytest.raises(error):
            kernels.adjust_logits(logits, **kw)

    refused(logits=logits[0])
    refused(RuntimeError, logits=logits.cpu())
    refused(TypeError, logits=logits.double())
    refused(logits=logits.to(torch.int8))
    refused(out=torch.empty(3, 100, device="cuda", dtype=torch.float16))
    refused(out=torch.empty(3, 99, device="cuda", dtype=torch.bfloat16))
    overlapping = torch.empty(4, 100, device="cuda", dtype=torch.bfloat16)
    refused(_native.NativeError, logits=overlapping[:3], out=overlapping[1:])
    t = lambda **kw: kernels.TokenPenalties(**{"history": p.history, "history_len": p.history_len, **kw})
    refused(penalties=t(history=p.history.long()))
    refused(penalties=t(history_len=p.history_len[:2]))
    refused(penalties=t(prompt_len=p.history_len.long()))
    refused(penalties=t(repetition=torch.ones(2, device="cuda")))
    refused(penalties=t(drafts=torch.zeros(3, 2, **i32)))
    refused(RuntimeError, penalties=t(history_len=p.history_len.cpu()))
    refused(_native.NativeError, penalties=t(repetition=0.0))
    refused(_native.NativeError, penalties=t(presence=float("nan")))
    refused(_native.NativeError, logits=make_logits(4, 100, "bf16"), penalties=t())
    refused(bias=kernels.TokenBias.from_dicts([{1: 1.0}] * 2, dev))
    refused(allowed=torch.zeros(3, 3, **i32))
    refused(allowed=torch.zeros(0, 4, **i32))
    refused(_native.NativeError, allowed=torch.zeros(2, 4, **i32))
    refused(allowed=torch.zeros(2, 4, **i32), allowed_rows=torch.zeros(2, **i32))


def test_masks_from_lists():
    mask = kernels.allowed_mask([[0, 31, 32, 69], None, []], 70, torch.device("cpu"))
    assert mask.shape == (3, kernels.allowed_words(70)) == (3, 3)
    assert mask[0].tolist() == [1 - 2**31, 1, 1 << 5] and mask[1].tolist() == [-1, -1, -1] and mask[2].tolist() == [0, 0, 0]
    with pytest.raises(ValueError):
        kernels.allowed_mask([[70]], 70, torch.device("cpu"))
    with pytest.raises(ValueError):
        kernels.allowed_mask([[-1]], 70, torch.device("cpu"))


def test_entry_point_refuses_bad_arguments_without_launching():
    if not _native.library_path().exists():
        pytest.skip("libnanoengine_hip.so is not built")
    lib = _native.load()
    p, null, far = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0), ctypes.c_void_p(1 << 30)

    def call(logits=p, dtype=0, ld=100, rows=3, vocab=100, history=null, stride=50, capacity=50, length=p, seqs=3, drafts=null,
             max_drafts=0, row_seq=null, row_drafts=null, rep=1.0, pres=0.0, freq=0.0, bias=null, tokens=null, values=null, entries=0,
             allowed=null, words=4, masks=3, allowed_rows=null, out=far, out_dtype=0, ld_out=100):
        return lib.ne_adjust_logits(logits, dtype, ld, rows, vocab, history, stride, capacity, length, null, seqs, drafts, max_drafts,
                                    row_seq, row_drafts, null, rep, null, pres, null, freq, bias, tokens, values, entries, allowed,
                                    words, masks, allowed_rows, out, out_dtype, ld_out, null)

    assert call(rows=0, logits=null) == 0
    for bad in (dict(rows=-1), dict(vocab=0), dict(logits=null), dict(out=null), dict(dtype=3), dict(out_dtype=1), dict(ld=99),
                dict(ld_out=99), dict(logits=ctypes.c_void_p((1 << 20) + 1)), dict(out=ctypes.c_void_p((1 << 20) + 100)),
                dict(out=p, out_dtype=2), dict(out=p, ld_out=101), dict(history=p, length=null), dict(history=p, stride=49),
                dict(history=p, capacity=-1), dict(history=p, seqs=2), dict(history=p, drafts=p, max_drafts=2),
                dict(history=p, rep=0.0), dict(history=p, rep=float("inf")), dict(history=p, pres=float("nan")),
                dict(history=p, freq=float("nan")), dict(bias=p, entries=2), dict(bias=p, entries=-1), dict(allowed=p, words=3),
                dict(allowed=p, masks=2)):
        assert call(**bad) == -1, bad
    assert call(vocab=(1 << 24) + 1, ld=1 << 25, ld_out=1 << 25) == -2
