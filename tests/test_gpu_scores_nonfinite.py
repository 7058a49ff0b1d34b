"""Places without probabilities do not cost the other places, or the other entries of a step, their scores."""

import json
import math

import pytest
import torch

from glm_tpu_b200.config.namizen import tiny_namizen
from glm_tpu_b200.entrypoints.cli import trace as trace_cli
from glm_tpu_b200.exceptions import DeviceStatusError
from glm_tpu_b200.runner.gpu_runner import build_runner


def runner_of(**options):
    return build_runner(tiny_namizen(), device="cuda:0", seed=3, context_capacity=320, prefill_chunk=128, lanes=2, **options)


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"dtype": torch.float32}])
@pytest.mark.parametrize("top", [0, 4])
def test_a_row_of_the_table_that_is_not_finite(native_lib, options, top):
    runner = runner_of(**options)
    try:
        ids = torch.randint(0, runner.g.vocab_size, (40,), generator=torch.Generator().manual_seed(2)).tolist()
        runner.open_lane(0), runner.open_lane(1)
        finite = runner.score(0, ids, following=7, top=top)
        assert not bool(torch.isnan(finite.logprob).any())
        runner.model.head_table[5].fill_(math.inf)  # a logit of plus or minus infinity, or a NaN, by the signs of a hidden row
        none = runner.score(1, ids, following=7, top=top)
        assert runner.lengths == [40, 40]
        bad = torch.isnan(none.best)
        assert bool(bad.any()) and torch.equal(torch.isnan(none.entropy), bad) and bool(torch.isnan(none.logprob)[bad].all())
        if top:
            assert bool((none.top_ids[bad] == -1).all()) and bool(torch.isnan(none.top_logprobs[bad]).all()) and bool((none.top_ids[~bad] >= 0).all())
        runner.model.head_table[5].fill_(0.0)
        assert bool(torch.isfinite(runner.score(1, ids, following=7, top=top).logprob).all())  # and nothing is left behind
    finally:
        runner.close()


@pytest.mark.gpu
def test_trace_writes_null_beside_the_other_entries(native_lib, tmp_path):
    runner = runner_of()
    try:
        runner.model.head_table[5].fill_(math.nan)
        lines = [json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [1, 2, 3], "want": [2]}, {"id": "b", "tokens": [1, 2], "score": {"top": 2}}]}),
                 json.dumps({"step": 1, "entries": [{"id": "a", "tokens": [4], "want": [0]}]})]
        with pytest.raises(DeviceStatusError, match="non-finite"):  # a decoding step, which picks a token, reports such logits as ever
            trace_cli.replay(runner, lines, tmp_path, emit=lambda *a, **k: None)
        (entry,) = json.loads((tmp_path / "0.scores.json").read_text())
        assert entry == {"id": "b", "logprob": [None] * 2, "entropy": [None] * 2, "best": [None] * 2, "top": [[[-1, None]] * 2] * 2}
        assert (tmp_path / "0.f32").exists()
    finally:
        runner.close()
