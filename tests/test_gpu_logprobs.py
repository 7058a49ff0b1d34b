"""Log probabilities of given tokens on a GPU, from logits and from hidden states, against the statement in 64 bits (``oracle.scoring``).

Tolerances.  ``s``, a sum of ``e^(x - m)`` in fp32, is off by at most (terms one after another + 16) 2^-24 of itself for the additions, and by what its terms
are off: 2^-22 for the exponential and |x - m| 2^-23 for its argument, where terms with |x - m| > 32 do not count any more (e^-32 times 2^17 tokens is 2^-29).
A thread adds at most 128 terms of these rows one after another: 144 2^-24 + 2^-22 + 32 2^-23 = 1.3e-5.  The logarithm turns this into an absolute error of ``lse``;
a log probability adds the rounding of its own terms, 2^-22 of its size.  ``t / s``, the mean of x - m, has the same relative errors, twice (numerator and
denominator), of the mean of |x - m|.  Logits from hidden states are off by (width + 16) 2^-23 sum |h w| themselves (products of bf16 are exact in fp32).
"""

import math

import pytest
import torch

from glm_tpu_b200.layers import logprobs
from glm_tpu_b200.oracle import scoring

BASE = 1.3e-5
NONFINITE, BAD_INDEX = 4, 2


def check(got, logits, tokens, top=0, logit_error=0.0):
    """``logits``: on the CPU, as the kernel saw them or in 64 bits; ``logit_error``: largest error of a logit (a number, or one per row)."""
    want = scoring.token_logprobs(logits, tokens.cpu(), top)
    x = logits.double()
    finite = torch.isfinite(x).any(1) & ~torch.isnan(x).any(1) & ~(x == math.inf).any(1)
    away = torch.where(torch.isfinite(x), (x - x.amax(1, keepdim=True)).abs(), torch.zeros_like(x))
    mean = (torch.softmax(x, 1).nan_to_num() * away).sum(1)
    err = torch.as_tensor(logit_error, dtype=torch.float64).expand(x.shape[0])
    bounds = {"logprob": lambda w: BASE + 2 * err + 2.0**-22 * (w.abs().nan_to_num(posinf=0, neginf=0) + 1), "best": lambda w: BASE + 2 * err + 2.0**-22 * w.abs().nan_to_num(posinf=0, neginf=0),
              "entropy": lambda w: BASE + (2 * BASE + 4 * err) * (1 + mean) + 2.0**-22 * w.abs().nan_to_num()}
    for name, bound in bounds.items():
        g, w = getattr(got, name).cpu().double(), getattr(want, name).double()
        assert torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(torch.isinf(g), torch.isinf(w)), (name, g, w)
        live = torch.isfinite(w)
        off = (g - w).abs()[live]
        assert bool((off <= bound(w)[live]).all()), (name, float((off - bound(w)[live]).max()), off)
        assert torch.equal(g[torch.isinf(w)], w[torch.isinf(w)])
    assert bool((got.best.cpu()[finite] >= got.logprob.cpu().nan_to_num(nan=-math.inf)[finite]).all())
    if top:
        assert torch.equal(got.top_ids.cpu(), want.top_ids)
        g, w = got.top_logprobs.cpu().double(), want.top_logprobs.double()
        assert torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(g == -math.inf, w == -math.inf)
        live = torch.isfinite(w)
        assert bool(((g - w)[live].abs() <= BASE + 2.0**-22 * (w[live].abs() + 1)).all())
        assert torch.equal(got.top_logprobs[:, 0].cpu()[finite], got.best.cpu()[finite])
    else:
        assert got.top_ids is None and got.top_logprobs is None


def rows_of(rows, vocab, dtype, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 11.0
    return x.to(dtype), torch.randint(0, vocab, (rows,), generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, vocab, dtype, top", [
    (1, 1, "f32", 1), (3, 2, "bf16", 2), (2, 31, "f32", 0), (5, 32, "bf16", 32), (1, 33, "f32", 32), (7, 257, "f32", 20), (300, 1000, "bf16", 5), (1, 4099, "bf16", 20),
    (4, 20001, "f32", 1), (149, 8191, "f32", 20), (33, 16384, "bf16", 0), (600, 777, "f32", 3), (1, 154880, "bf16", 20), (2, 131072, "f32", 32), (9, 65521, "bf16", 7)])
def test_sizes(native_lib, rows, vocab, dtype, top):
    x, tokens = rows_of(rows, vocab, {"f32": torch.float32, "bf16": torch.bfloat16}[dtype], seed=rows + vocab)
    got = logprobs.token_logprobs(x.cuda(), tokens.cuda(), top=top)
    check(got, x, tokens, top)
    again = logprobs.token_logprobs(x.cuda(), tokens.cuda(), top=top)
    assert all(torch.equal(a, b) for a, b in zip(vars(got).values(), vars(again).values()) if a is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first, stride", [(0, 1003), (1, 1003), (3, 1008), (8, 1016), (5, 1001)])
def test_rows_that_begin_anywhere(native_lib, dtype, first, stride):
    wide = torch.full((6, stride + first), 1e30).to(dtype)
    x, tokens = rows_of(6, 1000, dtype, seed=first)
    wide[:, first : first + 1000] = x
    got = logprobs.token_logprobs(wide.cuda()[:, first : first + 1000], tokens.int().cuda(), top=9)
    check(got, x, tokens, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [1, 20, 32])
@pytest.mark.parametrize("vocab", [64, 1500, 40000])
def test_ties_go_to_the_lowest_id(native_lib, vocab, top):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randint(-3, 4, (5, vocab), generator=g).float()
    x[1] = 2.0
    x[2] = torch.where(torch.randint(0, 2, (vocab,), generator=g) > 0, 0.0, -0.0)  # equal, whatever their sign
    x[3] = torch.arange(vocab).float()          # ever larger
    x[4] = -torch.arange(vocab).float()
    tokens = torch.zeros(5, dtype=torch.int64)
    check(logprobs.token_logprobs(x.cuda(), tokens.cuda(), top=top), x, tokens, top)
    half = x.bfloat16()
    check(logprobs.token_logprobs(half.cuda(), tokens.cuda(), top=top), half, tokens, top)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50, 3001, 70000])
def test_masked_infinite_and_missing(native_lib, vocab):
    x, tokens = rows_of(10, vocab, torch.float32, seed=5)
    inf, lowest = math.inf, torch.finfo(torch.float32).min
    x[0, ::2] = -inf
    x[1] = -inf                                  # nothing is left
    x[2] = -inf
    x[2, vocab - 1] = -4.0                       # one token is left
    x[3, 7] = math.nan
    x[4, vocab // 2] = inf
    x[5] = lowest
    x[6, 3:] = lowest
    x[7] += 30000.0
    x[8, : vocab - 9] = -inf
    tokens[0], tokens[2], tokens[8], tokens[9] = 2, 0, 1, -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(logprobs.token_logprobs(x.cuda(), tokens.cuda(), top=20, status=status), x, tokens, 20)
    assert int(status) == NONFINITE
    keep = [0, 1, 2, 5, 6, 7, 8, 9]
    status.zero_()
    check(logprobs.token_logprobs(x[keep].cuda(), tokens[keep].cuda(), top=0, status=status), x[keep], tokens[keep])
    assert int(status) == 0  # a masked token, an empty row and a token that is not asked for are in order


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_tokens_outside_the_vocabulary(native_lib, kind):
    x, _ = rows_of(4, 100, torch.float32)
    tokens = torch.tensor([100, -2, 99, 2**31 - 1], dtype=kind)
    if kind == torch.int64:
        tokens[3] = (1 << 32) + 5
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = logprobs.token_logprobs(x.cuda(), tokens.cuda(), status=status)
    check(got, x, tokens)
    assert int(status) == BAD_INDEX and torch.isnan(got.logprob).tolist() == [True, True, False, True]


@pytest.mark.gpu
def test_no_rows(native_lib):
    got = logprobs.token_logprobs(torch.empty(0, 100, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), top=3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)
    got = logprobs.head_logprobs(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16), torch.empty(10, 64, device="cuda", dtype=torch.bfloat16), torch.empty(0, dtype=torch.int32, device="cuda"))
    assert got.entropy.shape == (0,)


# ------------------------------------------------------------------------------------------------ from hidden states
def states_of(rows, width, vocab, dtype=torch.bfloat16, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed * 31 + rows + width + vocab)
    head = (torch.randn(vocab + extra, width, generator=g) * 2 * width**-0.5).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    hidden = (torch.randn(rows, width, generator=g) + 2.0 * head[tokens].float()).to(dtype)
    return hidden, head, tokens


def check_head(got, hidden, head, tokens):
    x = hidden.double() @ head.double().T
    err = (hidden.shape[1] + 16) * 2.0**-23 * (hidden.double().abs() @ head.double().abs().T).amax(1)
    check(got, x, tokens, 0, err)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width, vocab", [
    (1, 8, 1), (1, 64, 100), (2, 6144, 1000), (8, 256, 4099), (9, 72, 300), (17, 512, 255), (64, 1032, 2000), (127, 200, 513), (128, 128, 4096), (129, 136, 777), (200, 520, 3001),
    (255, 64, 256), (256, 1024, 1025), (257, 504, 130), (300, 2048, 5000), (600, 96, 20001), (1100, 640, 700), (33, 64, 60000)])
def test_head_sizes(native_lib, rows, width, vocab):
    hidden, head, tokens = states_of(rows, width, vocab)
    args = hidden.cuda(), head.cuda(), tokens.cuda()
    got = logprobs.head_logprobs(*args)
    check_head(got, hidden, head, tokens)
    again = logprobs.head_logprobs(*args)
    assert torch.equal(got.logprob, again.logprob) and torch.equal(got.entropy, again.entropy) and torch.equal(got.best, again.best)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 50, 400])
def test_head_rows_behind_the_vocabulary_do_not_count(native_lib, rows):
    hidden, head, tokens = states_of(rows, 192, 701, extra=3)
    head[701:] = math.nan
    got = logprobs.head_logprobs(hidden.cuda(), head.cuda(), tokens.cuda(), vocab=701)
    check_head(got, hidden, head[:701], tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 40, 300])
def test_head_strided_rows_and_a_row_that_is_not_finite(native_lib, rows):
    hidden, head, tokens = states_of(rows, 256, 900)
    wide, table = torch.full((rows, 264), math.nan).bfloat16().cuda(), torch.full((900, 320), math.nan).bfloat16().cuda()
    wide[:, :256], table[:, :256] = hidden.cuda(), head.cuda()
    wide[2, 17] = math.nan
    tokens[1] = 900
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = logprobs.head_logprobs(wide[:, :256], table[:, :256], tokens.int().cuda(), status=status)
    assert int(status) == NONFINITE | BAD_INDEX
    assert torch.isnan(got.logprob).nonzero()[:, 0].tolist() == [1, 2] and torch.isnan(got.entropy).nonzero()[:, 0].tolist() == [2]
    keep = [r for r in range(rows) if r != 2]
    check_head(type(got)(got.logprob[keep], got.entropy[keep], got.best[keep], None, None), hidden[keep], head, tokens[keep])


@pytest.mark.gpu
def test_head_most_likely_token_has_the_best_log_probability(native_lib):
    for rows in (4, 60, 300):
        hidden, head, _ = states_of(rows, 512, 3000)
        tokens = (hidden.double() @ head.double().T).argmax(1)
        got = logprobs.head_logprobs(hidden.cuda(), head.cuda(), tokens.cuda())
        assert torch.equal(got.logprob, got.best)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 70])
def test_head_in_fp32(native_lib, rows):
    hidden, head, tokens = states_of(rows, 136, 1003, torch.float32)
    check_head(logprobs.head_logprobs(hidden.cuda(), head.cuda(), tokens.cuda()), hidden, head, tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 20, 200])
def test_head_table_of_more_than_32_bits(native_lib, rows):
    """2^31 elements and more; but for its last 64 tokens the table is zeros, so those tokens' logits are."""
    width, few = 8192, 64
    vocab = (1 << 31) // width + 200
    g = torch.Generator().manual_seed(rows)
    last = (torch.randn(few, width, generator=g) * 4 * width**-0.5).bfloat16()
    head = torch.zeros(vocab, width, dtype=torch.bfloat16, device="cuda")
    head[-few:] = last.cuda()
    k = torch.randint(0, few, (rows,), generator=g)
    hidden = (torch.randn(rows, width, generator=g) + 2.0 * last[k].float()).bfloat16()
    got = logprobs.head_logprobs(hidden.cuda(), head, (vocab - few + k).cuda())
    x = hidden.double() @ last.double().T
    lse = torch.logaddexp(torch.logsumexp(x, 1), torch.tensor(math.log(vocab - few), dtype=torch.float64))
    # the zeros: a thread of the widest run adds 1,024 terms of them one after another, so (1,024 + 16) 2^-24 takes the place of 144 2^-24 in the bound
    bound = (1040 + 4) * 2.0**-24 + 32 * 2.0**-23 + 2 * (width + 16) * 2.0**-23 * (hidden.double().abs() @ last.double().abs().T).amax(1) + 2.0**-21 * lse.abs()
    assert bool(((got.logprob.cpu().double() - (x[torch.arange(rows), k] - lse)).abs() <= bound).all())
    assert bool(((got.best.cpu().double() - (x.amax(1) - lse)).abs() <= bound).all())


@pytest.mark.gpu
def test_many_rows(native_lib):
    x, tokens = rows_of(70001, 37, torch.bfloat16)
    check(logprobs.token_logprobs(x.cuda(), tokens.cuda(), top=2), x, tokens, 2)


# ------------------------------------------------------------------------------------------------ streams and graphs
@pytest.mark.gpu
def test_on_a_stream_of_its_own_and_in_two_graphs(native_lib):
    x, tokens = rows_of(3, 30011, torch.bfloat16)
    hidden, head, k = states_of(40, 256, 3000)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        on = [t.cuda() for t in (x, tokens, hidden, head, k)]
        got = logprobs.token_logprobs(on[0], on[1], top=4), logprobs.head_logprobs(on[2], on[3], on[4])
    side.synchronize()
    check(got[0], x, tokens, 4)
    check_head(got[1], hidden, head, k)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((logprobs.token_logprobs(on[0], on[1], top=4), logprobs.head_logprobs(on[2], on[3], on[4])))
        graphs.append(graph)
    y, tokens2 = rows_of(3, 30011, torch.bfloat16, seed=9)
    hidden2, _, k2 = states_of(40, 256, 3000, seed=9)
    for a, b in zip((on[0], on[1], on[2], on[4]), (y, tokens2, hidden2, k2)):
        a.copy_(b)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):  # both at once
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        check(out[0], y, tokens2, 4)
        check_head(out[1], hidden2, head, k2)
