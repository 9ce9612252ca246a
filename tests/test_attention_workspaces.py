"""AttentionWorkspace, host side: which buffers a captured graph holds."""

from __future__ import annotations

import pytest
import torch

from nanoengine_amd.kernels import AttentionWorkspace

CPU = torch.device("cpu")


def test_a_graph_of_one_kind_of_attention_does_not_hold_the_others_buffer():
    """A captured step that reads shared prefixes uses the plans' buffer alone: the step that comes
    after sharing has ended allocates its own, and the other way round."""
    ws = AttentionWorkspace()
    ws.get_prefix(CPU, 1000)
    ws.frozen = True  # as binding a graph does
    first = ws.get(CPU, 500, (1,))
    assert first.numel() >= 500 and ws.get(CPU, 400, (1,)) is first
    other = AttentionWorkspace()
    other.get(CPU, 500, (1,))
    other.frozen = True
    assert other.get_prefix(CPU, 1000).numel() >= 1000


def test_buffers_that_a_graph_holds_do_not_move():
    ws = AttentionWorkspace()
    ws.get(CPU, 500, (1,))
    ws.get_prefix(CPU, 1000)
    ws.frozen = True
    with pytest.raises(RuntimeError, match="held by a captured HIP graph"):
        ws.get(CPU, 501, (1,))
    with pytest.raises(RuntimeError, match="held by a captured HIP graph"):
        ws.get_prefix(CPU, 1001)
