"""Log probabilities of given tokens without a GPU: the CPU statement against plain torch, and the refusals."""

import math

import pytest
import torch

from glm_tpu_b200.layers import logprobs


def test_plain_rows_against_torch():
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(0)) * 3
    tokens = torch.randint(0, 300, (6,))
    got = logprobs.token_logprobs(x, tokens, top=5)
    logp = torch.log_softmax(x.double(), 1)
    assert torch.allclose(got.logprob.double(), logp.gather(1, tokens[:, None])[:, 0], atol=1e-6)
    assert torch.allclose(got.entropy.double(), -(logp.exp() * logp).sum(1), atol=1e-6) and torch.allclose(got.best.double(), logp.amax(1), atol=1e-6)
    values, ids = logp.topk(5)
    assert torch.equal(got.top_ids.long(), ids) and torch.allclose(got.top_logprobs.double(), values, atol=1e-6)
    h, w = torch.randn(6, 24).bfloat16(), torch.randn(300, 24).bfloat16()
    got = logprobs.head_logprobs(h, w, tokens, vocab=290)
    logp = torch.log_softmax(h.double() @ w[:290].double().T, 1)
    known = tokens < 290
    assert torch.allclose(got.logprob.double()[known], logp[known].gather(1, tokens[known][:, None])[:, 0], atol=1e-5) and bool(torch.isnan(got.logprob[~known]).all())


def test_rows_without_probabilities():
    inf = math.inf
    x = torch.tensor([[-inf, -inf, -inf], [0.0, -inf, 0.0], [0.0, math.nan, 1.0], [inf, 0.0, 0.0], [1.0, 1.0, 0.0]])
    got = logprobs.token_logprobs(x, torch.tensor([0, 1, 0, 0, -1]), top=3)
    assert got.logprob.tolist()[:2] == [-inf, -inf] and bool(torch.isnan(got.logprob[2:]).all())
    assert got.entropy.tolist()[0] == 0.0 and got.entropy[1].item() == pytest.approx(math.log(2)) and bool(torch.isnan(got.entropy[2:4]).all())
    assert got.top_ids.tolist() == [[0, 1, 2], [0, 2, 1], [-1] * 3, [-1] * 3, [0, 1, 2]] and got.top_logprobs[1, 2].item() == -inf


def test_refusals():
    x, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    for bad in (lambda: logprobs.token_logprobs(x.double(), t), lambda: logprobs.token_logprobs(x[0], t), lambda: logprobs.token_logprobs(x, t[:1]), lambda: logprobs.token_logprobs(x, t.float()),
                lambda: logprobs.token_logprobs(x, t, top=6), lambda: logprobs.token_logprobs(x, t, status=torch.zeros(1)), lambda: logprobs.token_logprobs(x, t, status=torch.zeros(2, dtype=torch.int32)), lambda: logprobs.token_logprobs(x, t, top=-1), lambda: logprobs.token_logprobs(torch.zeros(2, 50), t, top=33),
                lambda: logprobs.token_logprobs(torch.zeros(2, 0), t), lambda: logprobs.head_logprobs(x, torch.zeros(7, 4), t), lambda: logprobs.head_logprobs(x, torch.zeros(7, 5).bfloat16(), t),
                lambda: logprobs.head_logprobs(x, torch.zeros(7, 5), t, vocab=8), lambda: logprobs.head_logprobs(x, torch.zeros(7, 5), t, vocab=0)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_refusals_on_a_gpu(native_lib):
    x, t = torch.zeros(4, 64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    half = x.bfloat16()
    for bad in (lambda: logprobs.token_logprobs(x.T, torch.zeros(64, dtype=torch.int64, device="cuda")), lambda: logprobs.token_logprobs(x, t.cpu()), lambda: logprobs.head_logprobs(half, half.cpu(), t),
                lambda: logprobs.head_logprobs(half[:, :60], half[:, :60], t), lambda: logprobs.head_logprobs(half[:, 4:60], half[:, 4:60], t)):
        with pytest.raises(ValueError):
            bad()
