"""Paged caches, trees and projections for the tests of ``layers.attention.paged``, and what the attention gives in 64 bits."""

import torch

from glm_tpu_b200.layers.attention import paged


def pools(pages, page, G, dim, vdim, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(pages, page, G, dim, generator=g).to(dtype), torch.randn(pages, page, G, vdim, generator=g).to(dtype)


def table_for(slots, page, seed=0, spare=2):
    """A table in which the pages lie in no order; entries behind a sequence's last page name no page."""
    per = [-(-s // page) for s in slots]
    order = torch.randperm(sum(per) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(slots), max(max(per), 1)), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at : at + n]
        at += n
    return table, sum(per) + spare


def random_masks(sizes, seed=0):
    g = torch.Generator().manual_seed(seed)
    masks = [paged.ancestor_masks([int(torch.randint(-1, j, (1,), generator=g)) if j else -1 for j in range(n)])[0] for n in sizes]
    return torch.cat(masks) if masks else torch.zeros(0, dtype=torch.int64)


def tree_case(lengths, sizes, *, H, G, dim, vdim, page, seed=0, spare_rows=0, sink=False):
    table, pages = table_for([n + t for n, t in zip(lengths, sizes)], page, seed)
    k, v = pools(pages, page, G, dim, vdim, seed)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for s in range(n + sizes[b]):
            used[table[b, s // page], s % page] = True
    k[~used], v[~used] = float("nan"), float("nan")  # slots that belong to nobody
    g = torch.Generator().manual_seed(seed + 1)
    rows = sum(sizes) + spare_rows
    starts = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32)
    masks = torch.cat([random_masks(sizes, seed), torch.full((spare_rows,), -1, dtype=torch.int64)])
    return dict(q=(torch.randn(rows, H, dim, generator=g) * 1.5).bfloat16(), cache=paged.PagedKV(k, v, table), starts=starts, lengths=torch.tensor(lengths, dtype=torch.int32),
                masks=masks, scale=dim**-0.5, max_rows=max(max(sizes), 1), sink=torch.randn(H, generator=g) + 1 if sink else None)


def to_cuda(case):
    c = case["cache"]
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in case.items()} | {"cache": paged.PagedKV(c.k.cuda(), c.v.cuda(), c.table.cuda())}


def tree_exact(case):
    """``(result, bound on a bf16 kernel's error)`` per row and head in 64 bits; rows of no sequence: zeros.

    The bound: the result's rounding, 2^-8 |o|; weights rounded to bf16 before the second product, 2^-8 sum p |v|; weights off by twice what the scores
    are off, (dim + 8) 2^-23 scale sum |q k|, and by 2^-20 for the exponential and the sums of up to 2^12 terms: all in units of sum p |v|."""
    q, c, scale = case["q"].double(), case["cache"], case["scale"]
    page, G = c.k.shape[1:3]
    H, vdim = q.shape[1], c.v.shape[3]
    out, bound = torch.zeros(q.shape[0], H, vdim, dtype=torch.float64), torch.zeros(q.shape[0], H, vdim, dtype=torch.float64)
    for b in range(c.table.shape[0]):
        r0, r1, n = int(case["starts"][b]), int(case["starts"][b + 1]), int(case["lengths"][b])
        for r in range(r0, r1):
            slots = torch.tensor([s for s in range(n + r1 - r0) if s < n or int(case["masks"][r]) >> (s - n) & 1], dtype=torch.long)
            if not slots.numel():
                continue
            pages = c.table[b].long()[slots // page]
            k = c.k[pages, slots % page].double().repeat_interleave(H // G, 1)
            v = c.v[pages, slots % page].double().repeat_interleave(H // G, 1)
            s = torch.einsum("hd,khd->hk", q[r], k) * scale
            off = (q.shape[2] + 8) * 2.0**-23 * scale * torch.einsum("hd,khd->hk", q[r].abs(), k.abs()).amax(1)
            full = torch.cat([s, case["sink"].double()[:, None]], 1) if case["sink"] is not None else s
            p = torch.softmax(full, 1)[:, : slots.numel()]
            out[r] = torch.einsum("hk,khd->hd", p, v)
            bound[r] = 2.0**-8 * out[r].abs() + (2.0**-8 + 2.0**-20 + 2 * off)[:, None] * torch.einsum("hk,khd->hd", p, v.abs())
    return out, bound * 1.01  # terms of second order


def assert_tree(got, case):
    want, bound = tree_exact(case)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (float((off - bound).max()), (off > bound).nonzero()[:5])
