"""When the runners read shared prefixes once: never where that was measured to be slower."""

from __future__ import annotations

import pytest
import torch

from nanoengine_amd import kernels

BF16, INT8 = torch.bfloat16, torch.int8


# (sequences sharing, common tokens, cache): steps of 28 layers and 8 KV heads
@pytest.mark.parametrize("members,tokens,dtype", [(16, 2048, BF16), (8, 4096, BF16), (4, 8192, BF16), (16, 2048, INT8), (64, 512, INT8)])
def test_batches_measured_slower_do_not_share(members, tokens, dtype):
    assert not kernels.shared_prefix_pays((members - 1) * tokens, 8, dtype)


@pytest.mark.parametrize("members,tokens,dtype", [(64, 1024, INT8), (64, 2048, INT8), (64, 8192, INT8), (52, 2048, BF16)])
def test_batches_measured_faster_share(members, tokens, dtype):
    assert kernels.shared_prefix_pays((members - 1) * tokens, 8, dtype)
