"""Inputs whose rows lie at one place (``expand``) give what their copies give; buffers that are written to are refused then."""

import pytest
import torch

from glm_tpu_b200.layers import logprobs
from glm_tpu_b200.layers.attention import paged

from tests.paged_cases import to_cuda, tree_case


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 40, 300])
def test_one_hidden_state_asked_for_many_tokens(native_lib, rows, dtype):
    g = torch.Generator("cuda").manual_seed(rows)
    hidden = torch.randn(1, 128, generator=g, device="cuda").to(dtype).expand(rows, 128)
    head = torch.randn(700, 128, generator=g, device="cuda").div(4).to(dtype)
    tokens = torch.arange(rows, device="cuda")
    got, want = logprobs.head_logprobs(hidden, head, tokens), logprobs.head_logprobs(hidden.contiguous(), head, tokens)
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.entropy, want.entropy) and torch.equal(got.best, want.best)
    same = head[:1].expand(700, 128)
    got = logprobs.head_logprobs(hidden, same, tokens, vocab=650)
    want = logprobs.head_logprobs(hidden, same.contiguous(), tokens, vocab=650)
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.entropy, want.entropy)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [40, 900])
def test_one_query_for_all_rows_or_heads(native_lib, length):
    d = to_cuda(tree_case([length], [5], H=4, G=2, dim=64, vdim=64, page=16))
    for q in (d["q"][:1].expand(5, 4, 64), d["q"][:, :1].expand(5, 4, 64), d["q"][:1, :1].expand(5, 4, 64)):
        assert torch.equal(paged.tree_attention(**(d | {"q": q})), paged.tree_attention(**(d | {"q": q.contiguous()})))
    with pytest.raises(ValueError):
        paged.tree_attention(**d, out=torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda").expand(5, 4, 64))


def test_pools_whose_slots_or_heads_share_memory_are_refused():
    case = tree_case([5], [2], H=4, G=2, dim=16, vdim=16, page=8)
    c, one = case["cache"], torch.zeros(2, dtype=torch.int32)
    qkv = torch.zeros(2, 4 * 16 + 4 * 16).bfloat16()
    for k in (c.k[:, :, :1].expand(-1, -1, 2, -1), c.k[:, :1].expand(-1, 8, -1, -1), c.k[:1].expand(c.k.shape[0], -1, -1, -1)):
        for cache in (paged.PagedKV(k, c.v, c.table), paged.PagedKV(c.k, k, c.table)):
            with pytest.raises(ValueError):
                paged.tree_attention(**(case | {"cache": cache}))
            with pytest.raises(ValueError):
                paged.append(qkv, cache, None, one, one, heads=4)
    one_head = c.k[:, :, :1].as_strided((c.k.shape[0], 8, 1, 16), (c.k.stride(0), c.k.stride(1), 0, 1))  # an axis of one has no second place
    assert not paged._shared(one_head)
