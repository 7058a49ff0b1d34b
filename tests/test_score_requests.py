"""What is asked of scoring is checked on the host, before a lane or a GPU is touched."""

from types import SimpleNamespace

import pytest

from glm_tpu_b200.entrypoints.cli import trace as trace_cli
from glm_tpu_b200.exceptions import RequestValidationError
from glm_tpu_b200.runner.lane_runner import LaneRunner

from tests.test_scores import Runner


@pytest.mark.parametrize("tokens, asked", [([1, 2], {"next": 10}), ([1, 2], {"top": 11}), ([1, 2], {"top": 32}), ([1, 10], {}), ([-1, 2], {}), ([1, "x"], {}), ([True, 1], {}), ([], {}), ([1 << 40], {})])
def test_a_step_that_asks_for_too_much_does_not_begin(tokens, asked):
    runner = Runner()
    runner.g = SimpleNamespace(vocab_size=10)
    session = trace_cli.TraceReplay(runner)
    with pytest.raises(RequestValidationError):
        session.step({"step": 0, "entries": [{"id": "b", "tokens": [1, 2], "want": []}, {"id": "a", "tokens": tokens, "score": asked}]})
    assert runner.calls == [] and session.lane_of == {} and session.free == [0, 1]


def test_a_step_that_asks_for_all_there_is_runs():
    runner = Runner()
    runner.g = SimpleNamespace(vocab_size=10)
    trace_cli.TraceReplay(runner).step({"step": 0, "entries": [{"id": "a", "tokens": [0, 9], "score": {"top": 10, "next": 9}}]})
    assert runner.calls == [("score", 0, [0, 9], 9, 10)]


@pytest.mark.parametrize("tokens, asked", [([1, 10], {}), ([1, -1], {}), ([10], {}), ([-1, 1], {}), ([1 << 40], {}), ([1], {"following": 10}), ([1], {"following": -1}), ([1], {"following": 1 << 40}),
                                           ([1], {"top": 11}), ([1], {"top": -1}), ([], {}), ([1] * 9, {})])
def test_a_runner_refuses_before_it_runs(tokens, asked):
    runner = SimpleNamespace(lengths=[0], world=1, cache=SimpleNamespace(context_capacity=8), g=SimpleNamespace(vocab_size=10))  # nothing that could run
    with pytest.raises(ValueError):
        LaneRunner.score(runner, 0, tokens, **asked)
    assert runner.lengths == [0]
