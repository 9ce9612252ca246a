"""Pools that ordinary attention serves and shared-prefix attention does not (int8 with fp32 scales):
the runners keep the former, whatever the batch would save."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from nanoengine_amd import kernels
from nanoengine_amd.memory import KVCachePool, PrefixCachingSlotAllocator
from nanoengine_amd.model_runner import ModelRunner
from nanoengine_amd.qwen3 import Qwen3VerifyModel, Qwen3Weights
from nanoengine_amd.runner import VerifyRunner
from nanoengine_amd.sequence_state import Sequence
from test_answers import CFG, request, unit_norms

CPU = torch.device("cpu")


@pytest.mark.parametrize("cache,scale,shares", [(torch.int8, torch.float32, False), (torch.int8, torch.bfloat16, True),
                                                (torch.int8, torch.float16, True), (torch.bfloat16, None, True),
                                                (torch.float16, None, False)])
def test_the_model_runner_shares_in_pools_that_are_served(cache, scale, shares):
    pool = SimpleNamespace(block_size=16, key_caches=[torch.zeros(1, dtype=cache)],
                           key_scales=None if scale is None else [torch.zeros(1, dtype=scale)])
    allocator = PrefixCachingSlotAllocator(400, 16, CPU)
    model = SimpleNamespace(config=SimpleNamespace(num_attention_heads=16, num_key_value_heads=8))
    runner = ModelRunner(model, pool, allocator, CPU, shared_prefix=True)
    parent = Sequence.from_request(request("p", list(range(2048))))
    allocator.reserve(parent, 2048)
    sequences = []
    for i in range(80):
        s = Sequence.from_request(request(f"{i}", list(range(2049))))
        allocator.fork(parent, s, 2048)
        allocator.reserve(s, 2049)
        sequences.append(s)
    assert (runner._prefix_groups(sequences, [1] * 80, 2049) is not None) == shares


@pytest.mark.gpu
def test_runners_of_a_pool_with_fp32_scales(monkeypatch):
    monkeypatch.setattr(kernels, "SHARED_PREFIX_MIN_BYTES", 1)
    dev, state = torch.device("cuda"), unit_norms()
    g = torch.Generator().manual_seed(4)
    prompt = torch.randint(0, 512, (16,), generator=g).tolist() * 6
    forked, verified = [], []
    for shared in (True, False):
        parts = lambda: (Qwen3VerifyModel(Qwen3Weights.from_state_dict(CFG, state, dev, torch.bfloat16), 160, dev),
                         KVCachePool(2, 8, 128, 60 * 16, dev, torch.float32, True, 16), PrefixCachingSlotAllocator(60, 16, dev))
        runner = ModelRunner(*parts(), dev, shared_prefix=shared)
        parent = Sequence.from_request(request("p", prompt))
        runner.allocator.reserve(parent, len(prompt))
        runner.run_step([parent])
        answers = [runner.fork(parent, request(f"{i}", prompt + [i])) for i in range(4)]
        for s in answers:
            runner.allocator.reserve(s, s.num_tokens)
        forked.append(runner.run_step(answers))
        verify = VerifyRunner(*parts(), 4, 4, 3, 300, frozenset(), shared_prefix=shared)
        seqs = [Sequence.from_request(request(f"{i}", prompt + [i], ignore_eos=True)) for i in range(4)]
        verify.add(seqs[:1])
        verify.add(seqs[1:])
        assert not verify.sharing
        verify.step()
        verified.append([s.token_ids for s in seqs])
    assert forked[0] == forked[1] and verified[0] == verified[1]
