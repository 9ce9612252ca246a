"""Penalties that no runner takes are refused before a step, by name."""

from __future__ import annotations

from collections import deque

import pytest

from nanoengine_amd.interface import SamplingParams
from nanoengine_amd.model_runner import ModelRunner
from nanoengine_amd.runner import VerifyRunner
from nanoengine_amd.sequence_state import Sequence
from test_answers import request

NAN, INF = float("nan"), float("inf")
REFUSED = [
    (dict(repetition_penalty=0.0), "repetition_penalty"), (dict(repetition_penalty=-1.0), "repetition_penalty"),
    (dict(repetition_penalty=INF), "repetition_penalty"), (dict(repetition_penalty=NAN), "repetition_penalty"),
    (dict(presence_penalty=NAN), "presence_penalty"), (dict(frequency_penalty=NAN), "frequency_penalty"),
    # a repeated token's logit would be NaN
    (dict(presence_penalty=INF, frequency_penalty=-INF), "presence_penalty"),
    (dict(presence_penalty=-INF, frequency_penalty=INF), "presence_penalty"),
]


class Untouched:
    """What no refused request gets to."""

    def __getattr__(self, name):
        raise AssertionError(f"a refused request reached {name}")


def verify_runner() -> VerifyRunner:
    runner = VerifyRunner.__new__(VerifyRunner)
    runner._inflight, runner._pending, runner.slots = deque(), deque(), [None, None]
    runner.max_model_len, runner.allocator = 256, Untouched()
    return runner


@pytest.mark.parametrize("kw,name", REFUSED)
def test_penalties_without_a_meaning_are_refused(kw, name):
    good, bad = (Sequence.from_request(request(rid, [1, 2, 3], **k)) for rid, k in (("good", dict(presence_penalty=0.5)), ("bad", kw)))
    runner = verify_runner()
    with pytest.raises(ValueError, match=f"bad: {name}"):
        runner.add([good, bad])
    assert runner.slots == [None, None]
    with pytest.raises(ValueError, match=f"bad: {name}"):
        ModelRunner(Untouched(), None, Untouched(), None).run_step([good, bad])


@pytest.mark.parametrize("kw", [dict(), dict(presence_penalty=INF), dict(frequency_penalty=INF), dict(presence_penalty=INF, frequency_penalty=INF),
                                dict(repetition_penalty=1e-3, presence_penalty=-2.0, frequency_penalty=-2.0)])
def test_penalties_with_a_meaning_pass(kw):
    """An infinite one bans the tokens that it is for."""
    seq = Sequence.from_request(request("good", [1, 2, 3], **kw))
    runner, placed = verify_runner(), []
    runner._prefill = lambda run: placed.extend(run) or {}
    runner.add([seq])
    assert placed == [(0, seq)]
    with pytest.raises(AssertionError, match="a refused request reached"):  # (the refusals are past)
        ModelRunner(Untouched(), None, Untouched(), None).run_step([seq])
