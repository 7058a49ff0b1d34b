"""Scoring through the trace command without a GPU: which entries are scored, what is written, what is refused."""

import json
import math

import pytest
import torch

from glm_tpu_b200.entrypoints.cli import trace as trace_cli
from glm_tpu_b200.exceptions import RequestValidationError
from glm_tpu_b200.layers.contracts import TokenLogprobs


class Runner:
    """Scores token k as -k, remembers its calls."""

    lanes = 2

    def __init__(self):
        self.lengths, self.calls = [0, 0], []

    def open_lane(self, lane):
        self.lengths[lane] = 0

    def extend(self, lane, tokens, want=()):
        self.calls.append(("extend", lane, list(tokens)))
        self.lengths[lane] += len(tokens)
        return torch.zeros(len(want), 3)

    def decode_logits(self, tokens):
        self.calls.append(("decode", dict(tokens)))
        for lane in tokens:
            self.lengths[lane] += 1
        return {lane: torch.ones(3) for lane in tokens}

    def score(self, lane, tokens, *, following=None, top=0):
        self.calls.append(("score", lane, list(tokens), following, top))
        self.lengths[lane] += len(tokens)
        asked = [*tokens[1:], math.nan if following is None else following]
        n = len(tokens)
        return TokenLogprobs(-torch.tensor(asked, dtype=torch.float32), torch.full((n,), 0.5), torch.full((n,), -0.25), torch.arange(top).int().expand(n, top) if top else None,
                             -torch.arange(top).float().expand(n, top) if top else None)


def test_scored_entries_are_written_beside_wanted_logits(tmp_path):
    runner = Runner()
    lines = [json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [5, 7, 3], "score": {"top": 2, "next": 9}}, {"id": "b", "tokens": [1, 2], "want": [1]}]}),
             json.dumps({"step": 1, "entries": [{"id": "b", "tokens": [4], "want": [0]}, {"id": "a", "tokens": [6], "score": {}}], "end": ["a"]}),
             json.dumps({"step": 2, "entries": [{"id": "b", "tokens": [4], "want": []}]})]
    trace_cli.replay(runner, lines, tmp_path, emit=lambda *a, **k: None)
    assert runner.calls == [("score", 0, [5, 7, 3], 9, 2), ("extend", 1, [1, 2]), ("decode", {1: 4}), ("score", 0, [6], None, 0), ("decode", {1: 4})]
    first, second = (json.loads((tmp_path / f"{i}.scores.json").read_text()) for i in (0, 1))
    assert first == [{"id": "a", "logprob": [-7.0, -3.0, -9.0], "entropy": [0.5] * 3, "best": [-0.25] * 3, "top": [[[0, 0.0], [1, -1.0]]] * 3}]
    assert second == [{"id": "a", "logprob": [None], "entropy": [0.5], "best": [-0.25]}]
    assert not (tmp_path / "2.scores.json").exists() and (tmp_path / "0.f32").stat().st_size == 12


@pytest.mark.parametrize("entry", [{"score": {"top": 33}}, {"score": {"top": -1}}, {"score": {"top": True}}, {"score": {"next": -1}}, {"score": {"next": "x"}}, {"score": {"best": 1}},
                                   {"score": 3}, {"score": {}, "want": [0]}])
def test_refused_before_anything_runs(entry):
    runner = Runner()
    with pytest.raises(RequestValidationError):
        trace_cli.TraceReplay(runner).step({"step": 0, "entries": [{"id": "b", "tokens": [1, 2], "want": []}, {"id": "a", "tokens": [1, 2]} | entry]})
    assert runner.calls == []
