"""Paged caches and drafted trees without a GPU: masks, the CPU statement against plain torch, bad indices, refusals."""

import pytest
import torch

from glm_tpu_b200.layers.attention import paged

from tests.paged_cases import assert_tree, pools, table_for, tree_case


def test_masks_of_a_tree():
    masks, depths = paged.ancestor_masks([-1, 0, 0, 2, -1])
    assert masks.tolist() == [1, 3, 5, 13, 16] and depths.tolist() == [0, 1, 1, 2, 0]
    masks, depths = paged.ancestor_masks(range(-1, 63))
    assert masks[63].item() == -1 and masks[62].item() == (1 << 63) - 1 and depths.tolist() == list(range(64))
    assert paged.ancestor_masks([])[0].shape == (0,)
    for bad in ([0], [-2], [-1, 1], [-1] * 65):
        with pytest.raises(ValueError):
            paged.ancestor_masks(bad)


@pytest.mark.parametrize("sink", [False, True])
def test_attention_of_the_statement(sink):
    case = tree_case([0, 37, 5], [2, 5, 1], H=4, G=2, dim=32, vdim=16, page=8, sink=sink, spare_rows=1)
    assert_tree(paged.tree_attention(**case), case)


def test_one_token_is_ordinary_attention():
    case = tree_case([20], [1], H=2, G=1, dim=16, vdim=16, page=8)
    c = case["cache"]
    k, v = (t[c.table[0].long()].flatten(0, 1)[:21, 0].float() for t in (c.k, c.v))
    want = torch.nn.functional.scaled_dot_product_attention(case["q"].float().transpose(0, 1), k[None].expand(2, -1, -1), v[None].expand(2, -1, -1)).transpose(0, 1)
    assert torch.allclose(paged.tree_attention(**case).float(), want, atol=2.0**-7)


@pytest.mark.parametrize("pairs", [False, True])
def test_append_of_the_statement(pairs):
    g = torch.Generator().manual_seed(0)
    k, v = pools(4, 8, 1, 16, 16)
    table, _ = table_for([9, 9], 8, spare=0)
    qkv = torch.randn(3, 2 * 16 + 16 + 16, generator=g).bfloat16()
    rot = torch.randn(10, 4, 2, generator=g)
    w = torch.rand(16, generator=g).bfloat16()
    before = k.clone()
    q = paged.append(qkv, paged.PagedKV(k, v, table), torch.tensor([3, 4, 9], dtype=torch.int32), torch.tensor([0, 1, 1], dtype=torch.int32), torch.tensor([8, 0, -1], dtype=torch.int32), heads=2, rot=rot,
                     pairs=pairs, k_norm=w)
    x = qkv[1, :16].float()
    a, b = (x[:8:2], x[1:8:2]) if pairs else (x[:4], x[4:8])
    first, second = a * rot[4, :, 0] - b * rot[4, :, 1], a * rot[4, :, 1] + b * rot[4, :, 0]
    turned = torch.stack([first, second], -1).flatten() if pairs else torch.cat([first, second])
    assert torch.allclose(q[1, 0].float(), torch.cat([turned, x[8:]]), atol=2e-2)
    assert torch.equal(v[table[0, 1], 0, 0], qkv[0, 48:]) and torch.equal(v[table[1, 0], 0, 0], qkv[1, 48:])
    key = qkv[1, 32:48].float()
    assert k[table[1, 0], 0, 0, 8:].float().allclose((key * (key.square().mean() + 1e-6).rsqrt() * w.float())[8:], atol=2e-2)
    assert int((k != before).any(-1).sum()) == 2  # two rows have a slot


def test_bad_indices_are_not_followed():
    k, v = pools(4, 8, 1, 16, 16)
    table = torch.tensor([[0, 9], [-1, 2]], dtype=torch.int32)
    qkv = torch.randn(6, 48).bfloat16()
    before = k.clone()
    seqs, slots = torch.tensor([0, 0, 1, 2, -1, 1], dtype=torch.int32), torch.tensor([8, 16, 0, 0, 0, 9], dtype=torch.int32)
    q = paged.append(qkv, paged.PagedKV(k, v, table), None, seqs, slots, heads=1)
    assert (q == 0).all(-1).all(-1).tolist() == [True] * 5 + [False] and int((k != before).any(-1).sum()) == 1


def test_refusals():
    case = tree_case([5], [2], H=4, G=2, dim=16, vdim=16, page=8)
    c = case["cache"]
    cut = lambda **more: lambda: paged.tree_attention(**(case | more))  # noqa: E731
    bad = [cut(q=case["q"].float()), cut(q=case["q"][:, :3]), cut(q=case["q"][..., :8]), cut(starts=case["starts"].long()), cut(starts=case["starts"][:1]), cut(lengths=case["starts"]),
           cut(masks=case["masks"].int()), cut(masks=case["masks"][:1]), cut(max_rows=0), cut(max_rows=65), cut(scale=0.0), cut(scale=-1.0), cut(scale=float("nan")), cut(cache=paged.PagedKV(c.k[:, :4], c.v[:, :4], c.table)), cut(cache=paged.PagedKV(c.k[:0], c.v[:0], c.table)), cut(sink=torch.zeros(3)), cut(status=torch.zeros(2, dtype=torch.int32)), cut(status=torch.zeros(1)), cut(sink=torch.zeros(4).double()),
           cut(cache=paged.PagedKV(c.k.float(), c.v, c.table)), cut(cache=paged.PagedKV(c.k, c.v[:1], c.table)), cut(cache=paged.PagedKV(c.k, c.v, c.table.long())),
           cut(cache=paged.PagedKV(c.k[..., :8], c.v, c.table)), cut(cache=paged.PagedKV(c.k, c.v, c.table[0])), cut(out=torch.zeros(2, 4, 8).bfloat16())]
    qkv, one = torch.zeros(2, 4 * 16 + 4 * 16).bfloat16(), torch.zeros(2, dtype=torch.int32)
    rot = torch.zeros(9, 8, 2)
    app = lambda *a, **more: lambda: paged.append(*(a or (qkv, c, one, one, one)), **({"heads": 4} | more))  # noqa: E731
    bad += [app(status=torch.zeros(1)), app(heads=3), app(heads=0), app(qkv.float(), c, one, one, one), app(qkv, c, one, one[:1], one), app(qkv, c, one, one, one.long()), app(qkv, c, None, one, one, rot=rot),
            app(rot=rot.double()), app(rot=torch.zeros(9, 9, 2)), app(rot=torch.zeros(9, 0, 2)), app(rot=torch.zeros(0, 8, 2)), app(q_norm=torch.ones(16)), app(k_norm=torch.ones(8).bfloat16())]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_refusals_on_a_gpu(native_lib):
    case = tree_case([5], [2], H=4, G=2, dim=32, vdim=32, page=8)
    c = case["cache"]
    k, v, table = c.k.cuda(), c.v.cuda(), c.table.cuda()
    d = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in case.items()} | {"cache": paged.PagedKV(k, v, table)}
    wide = torch.zeros(2, 4, 36, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros(k.shape[0], 8, 2, 40, dtype=torch.bfloat16, device="cuda")
    for more in (dict(q=wide[..., 4:]), dict(q=wide[..., :32]), dict(out=wide[..., 4:]), dict(cache=c), dict(masks=case["masks"]), dict(cache=paged.PagedKV(pool[..., 4:36], v, table)),
                 dict(cache=paged.PagedKV(k, v, table.repeat(1, 4)[:, ::2]))):
        with pytest.raises(ValueError):
            paged.tree_attention(**(d | more))
    one = torch.zeros(2, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(2, 260, dtype=torch.bfloat16, device="cuda")
    for bad in (qkv[:, :256], qkv[:, 4:]):
        with pytest.raises(ValueError):
            paged.append(bad, d["cache"], None, one, one, heads=4)
