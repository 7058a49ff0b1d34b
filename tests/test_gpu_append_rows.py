"""What append leaves alone: slots that nobody named, rows with a bad index, and what lies around the rows that it reads."""

import math

import pytest
import torch

from glm_tpu_b200.oracle import scoring

from tests.test_gpu_paged import append_case, cuda, run_append

BAD_INDEX = 2


def exact(c, pairs=False):
    """Queries and pools in 64 bits, and which slots are written."""
    k, v = c["k"].double(), c["v"].double()
    q = scoring.append(c["qkv"].double(), k, v, c["table"], c["positions"], c["seqs"], c["slots"], heads=c["heads"], q_norm=c["q_norm"], k_norm=c["k_norm"], eps=c["eps"], rot=c["rot"], pairs=pairs)
    pages, page = c["k"].shape[:2]
    written = torch.zeros(pages, page, dtype=torch.bool)
    for r in range(c["qkv"].shape[0]):
        position = int(c["positions"][r])
        at = scoring.page_of(c["table"], int(c["seqs"][r]), int(c["slots"][r]), page, pages)
        if at >= 0 and (c["rot"] is None or 0 <= position < c["rot"].shape[0]):
            written[at, int(c["slots"][r]) % page] = True
    return q, k, v, written


def assert_rows(c, d, q, pairs=False):
    """One rounding, 2^-8 |y|, beside the fp32 arithmetic: (dim + 16) 2^-23 of the largest value of the head."""
    want_q, want_k, want_v, written = exact(c, pairs)
    close = lambda got, w: bool(((got.cpu().double() - w).abs() <= 2.0**-8 * w.abs() + (w.shape[-1] + 16) * 2.0**-23 * w.abs().amax(-1, keepdim=True)).all())  # noqa: E731
    assert close(q, want_q) and close(d["k"][written.cuda()], want_k[written])
    assert torch.equal(d["v"].cpu()[written], want_v.bfloat16()[written])
    for name in ("k", "v"):  # bit for bit
        assert torch.equal(d[name].cpu()[~written].view(torch.int16), c[name][~written].view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rot", [32, 20, 0])
def test_a_bad_index_writes_nothing(native_lib, rot, pairs):
    c = append_case(14, 4, 2, 32, 32, 8, rot=rot)
    if rot:
        c["positions"][0], c["positions"][1] = -1, 5000
    c["seqs"][2], c["seqs"][3] = -1, 3
    c["slots"][4], c["slots"][6] = 8 * c["table"].shape[1], -1
    c["table"][2, 0], c["table"][1, 0] = -1, c["k"].shape[0]
    c["k"][:, 5], c["v"][:, 5] = math.nan, math.nan  # as a slot may that nobody has written
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = cuda(c)
    q = run_append(d, status=status, pairs=pairs)
    assert int(status) == BAD_INDEX
    # where a NaN was and a row now lies, both sides hold the row; elsewhere the comparison is of bits
    assert_rows(c, d, q, pairs)
    bad = (exact(c)[0] == 0).all(-1).all(-1)
    assert bad.tolist()[2:5] == [True] * 3 and not bad[6] and bool((q.cpu()[bad] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows, H, G, dim, rot", [(1, 1, 1, 16, 2), (3, 1, 1, 16, 14), (2, 2, 1, 16, 10), (6, 4, 2, 32, 2), (5, 3, 1, 32, 30), (4, 1, 1, 48, 20), (9, 9, 2, 64, 34), (7, 5, 3, 80, 40),
                                                  (3, 1, 1, 128, 90), (2, 3, 1, 256, 250)])
def test_few_heads_between_other_memory(native_lib, rows, H, G, dim, rot):
    """Fewer heads than a warp takes at once, halves that are no multiple of four channels, rows that lie between NaN."""
    for norm in (True, False):
        c = append_case(rows, H, G, dim, dim, 8, rot=rot, norm=norm)
        wide = torch.full((rows + 2, c["qkv"].shape[1] + 24), math.nan, dtype=torch.bfloat16, device="cuda")
        inside = wide[1:-1, 8:-16]
        inside.copy_(c["qkv"])
        d = cuda(c) | {"qkv": inside}
        assert_rows(c, d, run_append(d))
