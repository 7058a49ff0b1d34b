"""Scored tokens of every model family against the logits that the same runner gives (``extend``), in 64 bits.

``extend`` rounds GLM logits to bf16 (2^-8 of a logit, which a log probability sees twice); the others' are fp32 sums of at most 256 products of the same
operands in another order: (256 + 16) 2^-23 sum |h w|, below 1e-3 for logits and operands of these random models."""

import math

import pytest
import torch

from glm_tpu_b200.config.model import tiny_geometry
from glm_tpu_b200.config.namizen import tiny_namizen
from glm_tpu_b200.config.zikevik import tiny_zikevik
from glm_tpu_b200.oracle import scoring
from glm_tpu_b200.runner.gpu_runner import build_runner

FAMILIES = {"glm": (tiny_geometry, {}), "namizen": (tiny_namizen, {}), "namizen32": (tiny_namizen, {"dtype": torch.float32}), "zikevik": (tiny_zikevik, {}), "zikevik32": (tiny_zikevik, {"dtype": torch.float32})}


def runner_of(name, **more):
    geometry, options = FAMILIES[name]
    options = {"stripe": 8, **options} if name == "glm" else options
    return build_runner(geometry(), device="cuda:0", seed=3, context_capacity=320, prefill_chunk=128, lanes=2, **options, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 7])
@pytest.mark.parametrize("name", list(FAMILIES))
def test_scores_are_those_of_the_logits(native_lib, name, top):
    runner = runner_of(name)
    try:
        ids = torch.randint(0, runner.g.vocab_size, (301,), generator=torch.Generator().manual_seed(1)).tolist()
        runner.open_lane(0), runner.open_lane(1)
        # in portions: across chunks, one token, a few; the logits in the same ones, for how a step is cut decides which kernels make its bf16 hidden states
        logits = torch.cat([runner.extend(0, ids[a:b], range(b - a)) for a, b in ((0, 260), (260, 261), (261, 300))])
        parts = [runner.score(1, ids[:260], following=ids[260], top=top), runner.score(1, ids[260:261], following=ids[261], top=top), runner.score(1, ids[261:300], following=ids[300], top=top)]
        assert runner.lengths == [300, 300]
        got = {n: torch.cat([getattr(p, n) for p in parts]) for n in ("logprob", "entropy", "best")}
        want = scoring.token_logprobs(logits, torch.tensor(ids[1:]), top)
        slack = 2 * 2.0**-8 * float(logits.abs().max()) if name == "glm" else 1e-3
        for n, g in got.items():
            bound = slack * (1 if n != "entropy" else 1 + math.log(runner.g.vocab_size))
            assert float((g - getattr(want, n)).abs().max()) <= bound, n
        assert bool((got["best"] >= got["logprob"]).all())
        if top:
            ids_of, values = torch.cat([p.top_ids for p in parts]), torch.cat([p.top_logprobs for p in parts])
            exact = torch.log_softmax(logits.double(), 1)
            assert float((exact.gather(1, ids_of.long()) - values).abs().max()) <= slack
            assert float((exact.topk(top, dim=1).values - values).abs().max()) <= slack
        else:
            assert parts[0].top_ids is None
        # the lane goes on from there: its next step sees what was scored
        more = runner.score(1, [ids[300]])
        assert more.logprob.shape == (1,) and math.isnan(float(more.logprob)) and math.isfinite(float(more.entropy))
    finally:
        runner.close()


@pytest.mark.gpu
def test_scoring_is_refused(native_lib):
    runner = runner_of("namizen")
    try:
        runner.open_lane(0)
        for bad in (lambda: runner.score(0, []), lambda: runner.score(0, [1] * 321), lambda: runner.score(0, [1], top=33), lambda: runner.score(0, [1], top=-1)):
            with pytest.raises(ValueError):
                bad()
        assert runner.lengths[0] == 0
    finally:
        runner.close()


@pytest.mark.gpu
def test_trace_writes_scores(native_lib, tmp_path):
    import json

    from glm_tpu_b200.entrypoints.cli import trace as trace_cli

    runner = runner_of("zikevik")
    try:
        ids = [3, 17, 200, 5]
        lines = [json.dumps({"step": 0, "entries": [{"id": "a", "tokens": ids, "want": [0, 1, 2, 3]}, {"id": "b", "tokens": ids, "score": {"top": 3, "next": 9}}]})]
        trace_cli.replay(runner, lines, tmp_path, emit=lambda *a, **k: None)
        logits = torch.from_file(str(tmp_path / "0.f32"), size=4 * runner.g.vocab_size).view(4, -1)
        (entry,) = json.loads((tmp_path / "0.scores.json").read_text())
        want = torch.log_softmax(logits.double(), 1).gather(1, torch.tensor([*ids[1:], 9])[:, None])[:, 0]
        assert entry["id"] == "b" and torch.allclose(torch.tensor(entry["logprob"]).double(), want, atol=1e-3) and [len(t) for t in entry["top"]] == [3] * 4
    finally:
        runner.close()
