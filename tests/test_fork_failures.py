"""Forks that fail after the allocator has given out the child's blocks."""

from __future__ import annotations

import pytest
import torch

from nanoengine_amd.interface import GenerationRequest, SamplingParams
from nanoengine_amd.memory import PagedSlotAllocator, PrefixCachingSlotAllocator
from nanoengine_amd.model_runner import ModelRunner
from nanoengine_amd.sequence_state import Sequence

CPU = torch.device("cpu")


class FailingCopies:
    block_size = 16

    def __init__(self):
        self.fails = True

    def copy_blocks(self, src, dst):
        if self.fails:
            raise RuntimeError("no launch")


@pytest.mark.parametrize("caching", [False, True])
@pytest.mark.parametrize("registered", [False, True])
def test_a_fork_whose_copy_fails_leaves_nothing_behind(caching, registered):
    allocator = (PrefixCachingSlotAllocator if caching else PagedSlotAllocator)(12, 16, CPU)
    pool = FailingCopies()
    runner = ModelRunner(None, pool, allocator, CPU)
    prompt = list(range(40))
    parent = Sequence.from_request(GenerationRequest("p", prompt, SamplingParams(max_new_tokens=8)))
    allocator.reserve(parent, 40)
    parent.num_cached_tokens = 40
    if registered:
        allocator.on_tokens_cached(parent)
    free = allocator.num_free_blocks
    child = GenerationRequest("c", prompt + [7], SamplingParams(max_new_tokens=8))
    for _ in range(3):
        with pytest.raises(RuntimeError, match="no launch"):
            runner.fork(parent, child)
        assert allocator.block_table("c") == [] and allocator.num_free_blocks == free
        if caching:
            assert [allocator.pool.reference_count(b) for b in allocator.block_table(parent)] == [1, 1, 1]
        assert allocator.first_writable_position("c") == 0
    pool.fails = False  # the request's id is free again
    assert runner.fork(parent, child).num_cached_tokens == 40
    allocator.free("c")
    allocator.free(parent)
    assert allocator.num_free_blocks == 12
