"""Captured verify steps of a batch that shares prefixes now and then: each kind of step is
captured once, and replays whenever the batch is of its kind."""

from __future__ import annotations

import pytest
import torch

from nanoengine_amd import kernels
from nanoengine_amd.sequence_state import Sequence
from test_answers import engine, request, unit_norms


@pytest.mark.gpu
def test_each_kind_of_step_is_captured_once(monkeypatch):
    monkeypatch.setattr(kernels, "SHARED_PREFIX_MIN_BYTES", 1)
    captured = []
    capture = torch.cuda.graph
    monkeypatch.setattr(torch.cuda, "graph", lambda *a, **k: captured.append(1) or capture(*a, **k))
    state = unit_norms()
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, 512, (16,), generator=g).tolist() * 6
    eager, graph = (engine(state, 4, True, graphs).runner for graphs in (False, True))
    kinds = {(False, False)} if captured else set()  # the engine's own, made when it is created
    all_tokens = [[], []]
    for turn in range(12):
        sampled, shared = turn // 2 % 2 == 1, turn % 2 == 1
        for runner, kept in zip((eager, graph), all_tokens):
            seqs = [Sequence.from_request(request(f"{turn}.{i}", prompt + [turn, i] if shared or i == 0 else [5 + turn, i, 3], seed=i,
                                                  ignore_eos=True, temperature=0.8 if sampled and i == 1 else 0.0)) for i in range(3)]
            runner.add(seqs[:1])
            runner.add(seqs[1:])
            assert (runner.any_sampled, runner.sharing) == (sampled, shared)
            for _ in range(3):
                runner.step()
            kept.append([list(s.token_ids) for s in seqs])
            for slot in runner.active_slots:
                runner.release(slot)
        assert (graph.graph_sampled, graph.graph_shared) == (sampled, shared)
        kinds.add((sampled, shared))
        assert len(captured) == len(kinds)
    assert len(kinds) == 4 and all_tokens[0] == all_tokens[1]
    assert graph.model.workspace.error_flag() == 0
