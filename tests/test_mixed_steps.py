"""Steps of the model runner that mix a prompt's prefill with many answers on shared blocks: one
sequence of many queries among single ones, whose plan is sized by the longest."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from nanoengine_amd import kernels, model_runner
from nanoengine_amd.interface import GenerationRequest, SamplingParams
from nanoengine_amd.memory import PrefixCachingSlotAllocator
from nanoengine_amd.model_runner import ModelRunner
from nanoengine_amd.sequence_state import Sequence
from test_answers import build, rel, request, unit_norms

CPU = torch.device("cpu")


class Recorder:
    """A model that keeps the batches it is given."""

    max_rows = 1 << 20
    eager_workspace = None

    def __init__(self):
        self.config = SimpleNamespace(num_attention_heads=16, num_key_value_heads=8)
        self.batches = []

    def ensure_rope(self, positions):
        pass

    def forward(self, rows, tokens, batch, pool, workspace=None):
        self.batches.append(batch)
        return torch.zeros(rows, 8)


def forward(counts: list[int], prefix: int = 2048):
    """The batch of a step in which sequence i brings ``counts[i]`` tokens after ``prefix`` shared ones."""
    model = Recorder()
    pool = SimpleNamespace(block_size=16, scratch_slot=0, key_caches=[torch.zeros(1, dtype=torch.int8)], value_caches=[],
                           key_scales=[torch.zeros(1, dtype=torch.bfloat16)], value_scales=None)
    allocator = PrefixCachingSlotAllocator(prefix // 16 + sum(-(-n // 16) for n in counts) + 8, 16, CPU)
    runner = ModelRunner(model, pool, allocator, CPU, shared_prefix=True)
    parent = Sequence.from_request(GenerationRequest("p", list(range(prefix)), SamplingParams(max_new_tokens=8)))
    allocator.reserve(parent, prefix)
    sequences = []
    for i, n in enumerate(counts):
        s = Sequence.from_request(GenerationRequest(f"{i}", list(range(prefix + n)), SamplingParams(max_new_tokens=8)))
        allocator.fork(parent, s, prefix)
        allocator.reserve(s, prefix + n)
        s.num_cached_tokens = prefix
        sequences.append(s)
    runner._forward(model_runner.build_step_inputs(sequences, allocator, pool, CPU), sequences)
    return model.batches[0]


def workspace_bytes(batch) -> int:
    return kernels.shared_prefix_workspace_bytes(batch.ctx_len.shape[0], batch.prefix_groups.prefix_len.shape[0], 16, 8, batch.max_q_len,
                                                 batch.max_ctx_len, batch.prefix_groups.max_prefix_len)


@pytest.mark.parametrize("counts", [[1024] + [1] * 63, [1] * 40 + [3000, 200] + [2] * 20])
def test_a_long_prompt_does_not_size_a_plan_of_many_sequences(counts):
    """64 sequences of 1,024 queries would need 1 GiB of partial sums, for a thousandth of those rows."""
    batch = forward(counts)
    assert batch.prefix_groups is None or workspace_bytes(batch) <= 1 << 28


@pytest.mark.parametrize("counts", [[1] * 64, [5] * 64, [100] + [1] * 63, [9, 5, 1, 2] * 16])
def test_steps_of_like_sequences_share(counts):
    batch = forward(counts)
    assert batch.prefix_groups is not None and 0 < workspace_bytes(batch) <= 1 << 28


def test_large_steps_without_padding_share():
    """What the rows themselves need is not held against them."""
    batch = forward([300] * 64)
    assert batch.prefix_groups is not None and workspace_bytes(batch) > 1 << 28


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("most", [None, 0])
def test_a_prompt_prefilled_beside_answers(int8, most, monkeypatch):
    """The mixed step through shared prefixes, or (no workspace allowed) through ordinary attention:
    the logits of one that never shares."""
    monkeypatch.setattr(kernels, "SHARED_PREFIX_MIN_BYTES", 1)
    if most is not None:
        monkeypatch.setattr(model_runner, "SHARED_PREFIX_MAX_PADDED", most)
    plans = []
    plan = kernels.shared_prefix_plan
    monkeypatch.setattr(kernels, "shared_prefix_plan", lambda *a, **k: plans.append(plan(*a, **k)) or plans[-1])
    state = unit_norms()
    g = torch.Generator().manual_seed(5)
    prompt, other = torch.randint(0, 4096, (1557,), generator=g).tolist(), torch.randint(0, 4096, (230,), generator=g).tolist()
    results = []
    for shared in (True, False):
        runner = build(state, int8, True, shared, 180)
        logits = []
        compute = runner._model.compute_logits
        monkeypatch.setattr(runner._model, "compute_logits", lambda h, **kw: logits.append(compute(h, **kw)) or logits[-1])
        parent = Sequence.from_request(request("parent", prompt))
        runner.allocator.reserve(parent, parent.num_tokens)
        while parent.num_uncached_tokens:
            runner.run_step([parent], [min(150, parent.num_uncached_tokens)])
        batch = [runner.fork(parent, request(f"r{i}", prompt + [i] * (i % 3))) for i in range(24)]
        late = Sequence.from_request(request("late", other))
        batch.insert(7, late)
        plans.clear()
        for counts in ([100 if s is late else s.num_uncached_tokens for s in batch], None):
            for s in batch:
                runner.allocator.reserve(s, s.num_tokens)
            if counts is None:  # the rest of the late prompt beside the answers' next tokens
                counts = [100 if s is late else 1 for s in batch]
                for s in batch:
                    if s is not late:
                        s.token_ids.append(17)
                        runner.allocator.reserve(s, s.num_tokens)
            logits.clear()
            runner.run_step(batch, counts)
            results.append(logits[0][0].clone())
        assert len(plans) == (2 if shared and most is None else 0)
        assert all(p.error_flag() == 0 for p in plans)
    for ours, theirs in zip(results[:2], results[2:]):
        assert rel(ours, theirs) <= 2e-2
