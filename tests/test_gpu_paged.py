"""Appending to a paged cache and attention of drafted trees over it on a GPU, against the formulas in 64 bits."""

import math

import pytest
import torch

from glm_tpu_b200.layers import logprobs
from glm_tpu_b200.layers.attention import paged
from glm_tpu_b200.oracle import scoring

from tests.paged_cases import assert_tree, pools, table_for, to_cuda, tree_case, tree_exact

BAD_INDEX = 2


# ------------------------------------------------------------------------------------------------ append
def append_case(rows, H, G, dim, vdim, page, *, rot=0, norm=True, seed=0):
    g = torch.Generator().manual_seed(seed + rows)
    seqs = min(3, rows)
    per = -(-rows // seqs) + 5
    table, pages = table_for([per] * seqs, page, seed)
    k, v = pools(pages, page, G, dim, vdim, seed)
    seq = torch.arange(rows) % seqs
    slots = 3 + torch.arange(rows) // seqs
    angle = torch.arange(5000, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(max(rot // 2, 1), dtype=torch.float64) / max(rot // 2, 1))
    weights = lambda: (1 + 0.2 * torch.randn(dim, generator=g)).bfloat16() if norm else None  # noqa: E731
    return dict(qkv=(2 * torch.randn(rows, H * dim + G * (dim + vdim), generator=g)).bfloat16(), k=k, v=v, table=table, positions=torch.randint(0, 5000, (rows,), generator=g).int(),
                seqs=seq.int(), slots=slots.int(), heads=H, rot=torch.stack([angle.cos(), angle.sin()], -1).float() if rot else None, q_norm=weights(), k_norm=weights(), eps=1e-5)


def run_append(c, **more):
    keep = {n: c[n] for n in ("heads", "rot", "q_norm", "k_norm", "eps")}
    return paged.append(c["qkv"], paged.PagedKV(c["k"], c["v"], c["table"]), c["positions"], c["seqs"], c["slots"], **(keep | more))


def cuda(c):
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in c.items()}


def assert_append(c, pairs=False):
    """bf16 results against 64 bits: one rounding, 2^-8 |y|, beside the fp32 arithmetic: (dim + 8) 2^-24 for the mean square, 2^-22 for root, products and rotation,
    in units of the largest value of the head (a rotation may cancel)."""
    exact_k, exact_v = c["k"].double(), c["v"].double()
    want = scoring.append(c["qkv"].double(), exact_k, exact_v, c["table"], c["positions"], c["seqs"], c["slots"], heads=c["heads"], q_norm=c["q_norm"], k_norm=c["k_norm"], eps=c["eps"],
                          rot=c["rot"], pairs=pairs)
    d = cuda(c)
    q = run_append(d, pairs=pairs)
    slack = (c["k"].shape[3] + 16) * 2.0**-23
    for got, w in ((q, want), (d["k"], exact_k), (d["v"], exact_v)):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(w))
        assert bool(((got - w).abs().nan_to_num() <= 2.0**-8 * w.abs().nan_to_num() + slack * w.nan_to_num().abs().amax(-1, keepdim=True)).all())
    assert torch.equal(d["v"].cpu(), exact_v.bfloat16())
    return q, d


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rows, H, G, dim, vdim, page, rot, norm", [
    (1, 1, 1, 16, 16, 8, 16, True), (1, 16, 4, 128, 128, 64, 64, True), (7, 8, 2, 64, 32, 40, 0, True), (33, 32, 8, 128, 128, 64, 128, True), (5, 4, 4, 80, 64, 16, 6, True),
    (65, 6, 3, 192, 256, 24, 192, False), (300, 3, 1, 256, 16, 8, 34, True), (2, 64, 8, 96, 96, 128, 48, False), (129, 12, 2, 48, 48, 56, 46, True)])
def test_append(native_lib, rows, H, G, dim, vdim, page, rot, norm, pairs):
    assert_append(append_case(rows, H, G, dim, vdim, page, rot=rot, norm=norm), pairs)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rows, H, G, dim, rot", [(40, 9, 2, 64, 24), (3, 70, 8, 128, 40), (11, 5, 5, 48, 20), (2, 33, 1, 256, 248), (6, 4, 2, 32, 2)])
def test_append_turns_part_of_a_head(native_lib, rows, H, G, dim, rot, pairs):
    for norm in (True, False):
        assert_append(append_case(rows, H, G, dim, dim, 8, rot=rot, norm=norm), pairs)


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rot, at", [(16, 16), (16, 23), (12, 12), (12, 14), (10, 10), (0, 9)])
def test_append_keeps_an_infinity_that_does_not_turn_to_itself(native_lib, rot, at, pairs):
    c = append_case(5, 2, 1, 32, 32, 8, rot=rot, norm=False)
    q, d = run_append(cuda(c), pairs=pairs), None
    c["qkv"][1, at] = math.inf
    d = cuda(c)
    with_inf = run_append(d, pairs=pairs)
    assert float(with_inf[1, 0, at]) == math.inf
    with_inf[1, 0, at] = q[1, 0, at]
    assert torch.equal(with_inf, q)


@pytest.mark.gpu
def test_append_refuses_what_its_loads_cannot_take(native_lib):
    d = cuda(append_case(4, 2, 1, 32, 32, 8, rot=16))
    odd = torch.ones(40, dtype=torch.bfloat16, device="cuda")[1:33]
    far = torch.zeros(4 * 8 * 2 + 2, device="cuda")[2:].view(4, 8, 2)
    for more in (dict(q_norm=odd), dict(k_norm=odd), dict(rot=far), dict(rot=d["rot"][:0])):
        with pytest.raises(ValueError):
            run_append(d, **more)


@pytest.mark.gpu
def test_append_strides_layouts_and_rows_without_a_slot(native_lib):
    c = append_case(9, 8, 2, 64, 64, 16, rot=32)
    c["slots"][4] = -1
    want_q, d = assert_append(c)
    # the same from wider rows, into pools whose heads lie outside the slots and keys beside values
    wide = torch.full((9, c["qkv"].shape[1] + 24), math.nan).bfloat16().cuda()
    wide[:, 8:-16] = c["qkv"].cuda()
    both = torch.empty(c["k"].shape[0], 2, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    k.copy_(c["k"]), v.copy_(c["v"])
    q = run_append(cuda(c) | {"qkv": wide[:, 8:-16], "k": k, "v": v})
    assert torch.equal(q, want_q) and torch.equal(k, d["k"]) and torch.equal(v, d["v"])
    # keys and values alone
    e = cuda(c)
    assert run_append(e, want_q=False) is None and torch.equal(e["k"], d["k"]) and torch.equal(e["v"], d["v"])
    # one weight of the two
    for name in ("q_norm", "k_norm"):
        assert_append(c | {name: None})


@pytest.mark.gpu
def test_append_never_follows_a_bad_index(native_lib):
    c = append_case(12, 4, 2, 32, 32, 8, rot=32)
    c["positions"][0], c["positions"][1] = -1, 5000
    c["seqs"][2], c["seqs"][3] = -1, 3
    c["slots"][4] = 8 * c["table"].shape[1]
    c["table"][2, 0], c["table"][1, 0] = -1, c["k"].shape[0]  # pages of rows 5, 8 (sequence 2) and 7, 10 (sequence 1), 4 and 1 beside them
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = cuda(c)
    q = run_append(d, status=status)
    assert int(status) == BAD_INDEX
    want = run_append(c)  # the statement on the CPU writes into its own pools
    assert torch.equal(d["k"].cpu() != 0, c["k"] != 0) and float((d["k"].cpu().float() - c["k"].float()).abs().max()) <= 2.0**-7 * float(c["k"].abs().max())
    bad = (want == 0).all(-1).all(-1)
    assert bad.tolist()[:6] == [True] * 6 and torch.equal((q == 0).all(-1).all(-1).cpu(), bad) and not bad.all()


@pytest.mark.gpu
def test_append_of_zero_rows_and_of_zeros(native_lib):
    c = append_case(2, 2, 1, 32, 32, 8, rot=8)
    c["qkv"].zero_()
    q, _ = assert_append(c)
    assert bool((q == 0).all())
    e = {n: (t[:0] if n in ("qkv", "positions", "seqs", "slots") else t) for n, t in cuda(c).items()}
    assert run_append(e).shape == (0, 2, 32)


# ------------------------------------------------------------------------------------------------ attention
SHAPES = [  # lengths, drafted tokens, heads, kv heads, dim, vdim, page
    ([0], [1], 1, 1, 16, 16, 8), ([1], [1], 4, 2, 64, 64, 16), ([777], [1], 16, 4, 128, 128, 64), ([63, 64, 65], [1, 1, 1], 8, 8, 128, 128, 64), ([0, 5, 300], [3, 7, 2], 8, 2, 64, 128, 16),
    ([100], [64], 8, 1, 128, 64, 24), ([129, 0, 1000, 17], [16, 1, 33, 8], 32, 8, 128, 128, 64), ([500], [5], 12, 2, 80, 80, 48), ([255], [9], 6, 3, 192, 192, 8), ([321, 4], [11, 64], 64, 8, 128, 128, 128),
    ([2047], [2], 8, 8, 256, 256, 32), ([60], [64], 20, 1, 96, 48, 64), ([3000, 1], [4, 4], 7, 7, 32, 16, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("lengths, sizes, H, G, dim, vdim, page", SHAPES)
def test_tree(native_lib, lengths, sizes, H, G, dim, vdim, page, sink):
    case = tree_case(lengths, sizes, H=H, G=G, dim=dim, vdim=vdim, page=page, sink=sink, seed=len(lengths) + sum(sizes))
    d = to_cuda(case)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = paged.tree_attention(**d, status=status)
    assert int(status) == 0
    assert_tree(got, case)
    assert torch.equal(got, paged.tree_attention(**d))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs, length, tree, H, G", [(1, 40000, 1, 16, 4), (2, 20011, 16, 32, 8), (1, 30001, 61, 64, 8), (40, 700, 5, 8, 2), (3, 9000, 64, 16, 1)])
def test_long_contexts(native_lib, seqs, length, tree, H, G):
    """Against one product per sequence in 64 bits; the bound of ``tree_exact`` with its sums of up to 2^16 terms."""
    sizes = [max(1, tree - b) for b in range(seqs)]
    lengths = [length - 13 * b for b in range(seqs)]
    g = torch.Generator("cuda").manual_seed(length)
    table, pages = table_for([n + t for n, t in zip(lengths, sizes)], 64, 3)
    k, v = (torch.randn(pages, 64, G, 128, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    starts = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32)
    masks = torch.randint(-(1 << 62), 1 << 62, (sum(sizes),), generator=g, device="cuda")  # masks need not be trees
    q = (1.5 * torch.randn(sum(sizes), H, 128, generator=g, device="cuda")).bfloat16()
    got = paged.tree_attention(q, paged.PagedKV(k, v, table.cuda()), starts.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), masks, 128**-0.5, max_rows=tree)
    for b in range(seqs):
        r0, r1, n = int(starts[b]), int(starts[b + 1]), lengths[b]
        slots = torch.arange(n + r1 - r0, device="cuda")
        at = table[b].cuda().long()[slots // 64], slots % 64
        seen = torch.ones(r1 - r0, slots.numel(), dtype=torch.bool, device="cuda")
        for t in range(r1 - r0):
            seen[:, n + t] = (masks[r0:r1] >> t & 1) == 1
        for h in range(0, H, max(1, H // 4)):
            kk, vv, qq = k[at[0], at[1], h // (H // G)].double(), v[at[0], at[1], h // (H // G)].double(), q[r0:r1, h].double()
            p = torch.softmax((qq @ kk.T * 128**-0.5).masked_fill(~seen, -math.inf), 1)
            want, off = p @ vv, 136 * 2.0**-23 * 128**-0.5 * (qq.abs() @ kk.abs().T).amax(1, keepdim=True)
            assert bool(((got[r0:r1, h].double() - want).abs() <= 1.01 * (2.0**-8 * want.abs() + (2.0**-8 + 2.0**-17 + 2 * off) * (p @ vv.abs()))).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tree", [4, 40])
def test_what_a_row_does_not_see_stays_out(native_lib, tree, dim):
    """NaN and infinities in drafted tokens of other branches, and in the slots behind the last one of a page that ends inside a tile."""
    case = tree_case([90, 33], [tree, 3], H=8, G=2, dim=dim, vdim=dim, page=32, seed=4)
    c = case["cache"]
    for value, where in ((math.nan, "k"), (math.inf, "v"), (math.nan, "v"), (-math.inf, "k")):
        k, v = c.k.clone(), c.v.clone()
        slot = 90 + 1
        (k if where == "k" else v)[c.table[0, slot // 32], slot % 32] = value
        masks = case["masks"].clone()
        masks[: tree] &= ~2
        masks[1] = 2 | 1  # the one row that sees it
        poisoned = case | {"cache": paged.PagedKV(k, v, c.table), "masks": masks}
        got = paged.tree_attention(**to_cuda(poisoned)).cpu()
        clean = case | {"masks": masks}
        keep = [r for r in range(tree + 3) if r != 1]
        want, bound = tree_exact(clean)
        assert bool(((got.double() - want).abs() <= bound)[keep].all()), (value, where)
        assert not bool(torch.isfinite(got[1]).all()) or (where == "k" and value == -math.inf)


@pytest.mark.gpu
def test_rows_that_see_nothing(native_lib):
    case = tree_case([0, 0, 40], [3, 1, 2], H=4, G=2, dim=64, vdim=64, page=16, seed=2)
    case["masks"][0], case["masks"][3], case["masks"][4] = 0, 0, 0
    got = paged.tree_attention(**to_cuda(case))
    assert_tree(got, case)
    assert bool((got[0] == 0).all()) and bool((got[3] == 0).all()) and bool((got[4] != 0).any())
    case["sink"] = torch.randn(4)
    got = paged.tree_attention(**to_cuda(case))
    assert_tree(got, case)
    assert bool((got[0] == 0).all())


@pytest.mark.gpu
def test_rows_of_no_sequence(native_lib):
    case = tree_case([50, 20], [3, 4], H=4, G=2, dim=64, vdim=64, page=16, spare_rows=5)
    d = to_cuda(case)
    out = torch.full((12, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    assert paged.tree_attention(**d, out=out) is out
    assert bool((out[7:] == 7).all())
    torch.cuda.empty_cache()
    junk = torch.full((1 << 20,), math.nan, dtype=torch.bfloat16, device="cuda")
    del junk  # the buffer that the call makes may have held anything
    got = paged.tree_attention(**d)
    assert bool((got[7:] == 0).all()) and torch.equal(got[:7], out[:7])
    assert_tree(got, case)
    d["starts"][0] = 2  # rows before the first sequence belong to nobody either
    out.fill_(7.0)
    paged.tree_attention(**d, out=out)
    assert bool((out[:2] == 7).all()) and bool((out[2:7] != 7).any())
    assert bool((paged.tree_attention(**d)[:2] == 0).all())


@pytest.mark.gpu
def test_tree_strides(native_lib):
    case = tree_case([333, 70], [6, 2], H=8, G=2, dim=64, vdim=64, page=32, seed=8)
    d = to_cuda(case)
    want = paged.tree_attention(**d)
    wide = torch.full((8, 8 * 64 + 64), math.nan, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 64:].view(8, 8, 64)
    q.copy_(d["q"])
    c = d["cache"]
    both = torch.empty(c.k.shape[0], 2, 2, 32, 64, dtype=torch.bfloat16, device="cuda")
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    k.copy_(c.k), v.copy_(c.v)
    table = torch.full((2, c.table.shape[1] + 3), 99, dtype=torch.int32, device="cuda")
    table[:, :-3] = c.table
    out = torch.full((8, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    paged.tree_attention(**(d | {"q": q, "cache": paged.PagedKV(k, v, table[:, :-3])}), out=out[..., 64:])
    assert torch.equal(out[..., 64:], want) and bool((out[..., :64] == 3).all())
    same = case | {"q": d["q"].transpose(0, 1).contiguous().transpose(0, 1)}
    assert torch.equal(paged.tree_attention(**(d | {"q": same["q"]})), want)


@pytest.mark.gpu
def test_bad_pages_rows_and_lengths_are_not_followed(native_lib):
    case = tree_case([200, 40, 10], [4, 2, 2], H=8, G=2, dim=128, vdim=128, page=16, seed=6)
    lost = case["cache"].table.clone()
    lost[0, 3], lost[0, 7] = -1, 1 << 30  # slots 48 .. 63 and 112 .. 127 of the first sequence
    want, bound = tree_exact(case)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = to_cuda(case | {"cache": paged.PagedKV(case["cache"].k, case["cache"].v, lost)})
    got = paged.tree_attention(**d, status=status)
    assert int(status) == BAD_INDEX
    off = (got.cpu().double() - want).abs()
    assert bool((off[4:] <= bound[4:]).all())
    # 32 of 204 keys are missing: compare with the same attention over what is left
    keys = [s for s in range(204) if not (48 <= s < 64 or 112 <= s < 128)]
    _assert_first_sequence(got, case, keys)
    for change in (dict(lengths=torch.tensor([200, -5, 10], dtype=torch.int32)), dict(lengths=torch.tensor([200, 1 << 30, 10], dtype=torch.int32)),
                   dict(starts=torch.tensor([0, 4, 6, 99], dtype=torch.int32)), dict(starts=torch.tensor([0, 4, 3, 8], dtype=torch.int32)), dict(max_rows=3)):
        status.zero_()
        out = torch.zeros(8, 8, 128, dtype=torch.bfloat16, device="cuda")
        paged.tree_attention(**to_cuda(case | change), out=out, status=status)
        assert int(status) == BAD_INDEX, change
        assert bool(torch.isfinite(out[0]).all())


def _assert_first_sequence(got, case, keys):
    c, page = case["cache"], case["cache"].k.shape[1]
    for r in range(4):
        seen = torch.tensor([s for s in keys if s < 200 or int(case["masks"][r]) >> (s - 200) & 1])
        at = c.table[0].long()[seen // page], seen % page
        k, v = (t[at[0], at[1]].double().repeat_interleave(4, 1) for t in (c.k, c.v))
        p = torch.softmax(torch.einsum("hd,khd->hk", case["q"][r].double(), k) * case["scale"], 1)
        want = torch.einsum("hk,khd->hd", p, v)
        assert bool(((got[r].cpu().double() - want).abs() <= 2.0**-8 * want.abs() + (2.0**-8 + 2.0**-12) * torch.einsum("hk,khd->hd", p, v.abs())).all())


@pytest.mark.gpu
def test_offsets_beyond_32_bits(native_lib):
    """A pool of more than 2^31 elements, of which a sequence uses the last pages."""
    page, G, dim = 64, 8, 128
    pages = (1 << 31) // (page * G * dim) + 10
    k, v = (torch.zeros(pages, page, G, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    case = tree_case([100], [3], H=8, G=G, dim=dim, vdim=dim, page=page, seed=1)
    c = case["cache"]
    d = to_cuda(case)
    for b in range(c.k.shape[0]):
        k[pages - 5 + b], v[pages - 5 + b] = c.k[b].cuda(), c.v[b].cuda()
    table = torch.where(d["cache"].table >= 0, d["cache"].table + pages - 5, d["cache"].table)
    assert_tree(paged.tree_attention(**(d | {"cache": paged.PagedKV(k, v, table)})), case)
    qkv = torch.randn(1, 8 * dim + 2 * G * dim, device="cuda").bfloat16()
    at = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.append(qkv, paged.PagedKV(k, v, table), None, at, at + 101, heads=8)
    assert torch.equal(k[table[0, 1].item(), 101 - 64].flatten(), qkv[0, 8 * dim : 16 * dim]) and torch.equal(v[table[0, 1].item(), 101 - 64].flatten(), qkv[0, 16 * dim :])


@pytest.mark.gpu
@pytest.mark.parametrize("seqs, length, tree", [(700, 9, 1), (300, 700, 2), (1500, 0, 3)])
def test_many_sequences(native_lib, seqs, length, tree):
    case = tree_case([(length * (b % 7)) // 6 for b in range(seqs)], [1 + b % tree for b in range(seqs)], H=4, G=2, dim=32, vdim=32, page=8)
    assert_tree(paged.tree_attention(**to_cuda(case)), case)


# ------------------------------------------------------------------------------------------------ the operators together
def _step(p, cache, starts, lengths, masks, positions, seqs, slots, tokens, status):
    """One step over drafted tokens: projection -> append -> attention -> projection -> log probabilities."""
    qkv = p["x"] @ p["w_qkv"].T
    q = paged.append(qkv, cache, positions, seqs, slots, heads=8, rot=p["rot"], q_norm=p["norm"], k_norm=p["norm"], status=status)
    o = paged.tree_attention(q, cache, starts, lengths, masks, 64**-0.5, max_rows=7, status=status)
    hidden = o.flatten(1) @ p["w_o"].T
    return qkv, o, logprobs.head_logprobs(hidden, p["head"], tokens, status=status)


def _together(seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()  # noqa: E731
    angle = torch.arange(4096, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(16, dtype=torch.float64, device="cuda") / 16)
    p = dict(x=rand(12, 256), w_qkv=rand(8 * 64 + 4 * 64, 256) / 16, w_o=rand(256, 512) / 16, head=rand(1000, 256) / 16, norm=1 + rand(64) / 8, rot=torch.stack([angle.cos(), angle.sin()], -1).float())
    lengths, parents = [70, 200], [[-1, 0, 0, 1, 2], [-1, 0, 1, 1, 3, 2, 0]]
    table, pages = table_for([n + 8 for n in lengths], 16)
    trees = [paged.ancestor_masks(t) for t in parents]
    masks, depths = (torch.cat([t[i] for t in trees]).cuda() for i in (0, 1))
    seqs = torch.tensor([0] * 5 + [1] * 7, dtype=torch.int32, device="cuda")
    at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    order = torch.tensor([*range(5), *range(7)], dtype=torch.int32, device="cuda")
    return p, dict(cache=paged.PagedKV(rand(pages, 16, 2, 64), rand(pages, 16, 2, 64), table.cuda()), starts=torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda"), lengths=at, masks=masks,
                   positions=at[seqs.long()] + depths, seqs=seqs, slots=at[seqs.long()] + order, tokens=torch.randint(0, 1000, (12,), generator=g, device="cuda"),
                   status=torch.zeros(1, dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
def test_a_step_over_drafted_tokens(native_lib):
    """Every path of the tree scores as if its tokens had come one by one, and accepted tokens appended again continue as if they had been decoded."""
    p, a = _together(0)
    committed = a["cache"].k.clone(), a["cache"].v.clone()
    qkv, o, scores = _step(p, **a)
    assert int(a["status"]) == 0
    # the path 0, 2, 4 of the first sequence as a chain over the same committed slots
    chain = [0, 2, 4]
    cache = paged.PagedKV(committed[0].clone(), committed[1].clone(), a["cache"].table)
    one = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    q = paged.append(qkv[chain], cache, 70 + one, one * 0, 70 + one, heads=8, rot=p["rot"], q_norm=p["norm"], k_norm=p["norm"])
    row_at = lambda n: torch.tensor([0, n, n], dtype=torch.int32, device="cuda")  # noqa: E731
    alone = paged.tree_attention(q, cache, row_at(3), a["lengths"], paged.ancestor_masks([-1, 0, 1])[0].cuda(), 64**-0.5, max_rows=3)
    assert float((alone.float() - o[chain].float()).abs().max()) <= 2.0**-7 * float(o.abs().max())  # two roundings of results whose sums ran in another order
    hidden = alone.flatten(1) @ p["w_o"].T
    again = logprobs.head_logprobs(hidden, p["head"], a["tokens"][chain])
    assert float((again.logprob - scores.logprob[chain]).abs().max()) < 0.05  # hidden states in bf16, logits of deviation one
    # accepting that path: its rows once more, at consecutive slots; the cache then holds what the chain's holds
    slots = torch.full((12,), -1, dtype=torch.int32, device="cuda")
    slots[chain] = 70 + one
    assert paged.append(qkv, a["cache"], a["positions"], a["seqs"], slots, heads=8, rot=p["rot"], q_norm=p["norm"], k_norm=p["norm"], want_q=False) is None
    for s in range(73):
        where = int(a["cache"].table[0, s // 16]), s % 16
        assert torch.equal(a["cache"].k[where], cache.k[where]) and torch.equal(a["cache"].v[where], cache.v[where])


@pytest.mark.gpu
def test_two_captured_steps_at_once(native_lib):
    steps = [_together(s) for s in (1, 2)]
    want = []
    for p, a in steps:
        _, o, scores = _step(p, **a)
        want.append((o.clone(), scores.logprob.clone(), scores.entropy.clone()))
    graphs, outs = [], []
    for p, a in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(p, **a))
        graphs.append(graph)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for (_, o, scores), _ in zip(outs, want):
            o.zero_(), scores.logprob.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, o, scores), (w, lp, ent) in zip(outs, want):
            assert torch.equal(o, w) and torch.equal(scores.logprob, lp) and torch.equal(scores.entropy, ent)
    # a replay reads lengths, masks and tokens as they are then
    p, a = steps[0]
    a["lengths"].copy_(torch.tensor([40, 111], dtype=torch.int32)), a["masks"].fill_(1)
    graphs[0].replay()
    torch.cuda.synchronize()
    _, o, scores = _step(p, **a)
    assert torch.equal(outs[0][1], o) and torch.equal(outs[0][2].logprob, scores.logprob)
