"""What is measured of the operators for scoring given tokens and for steps over drafted tokens.

    append              norms of queries and keys per head, rotation, keys and values into a paged cache
    tree_attention      a tree of drafted tokens over the paged cache and its own ancestors
    token_logprobs      log probability of given tokens, entropy and top alternatives from logits
    head_logprobs       the same from hidden states and the output table, without logits in memory

``run`` computes them in plain torch operations, or through ``glm_tpu_b200.layers`` where ``own`` is true.  Head shapes, widths and vocabularies are those
of the models and benchmarks of this repository, or odd ones beside them.
"""

import math

import torch

own = False
DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one generated token of one chat with 20 alternatives: the smallest call, latency
        dict(name="logprobs_answer_token", op="token_logprobs", rows=1, vocab=154880, pad=0, dtype="bf16", top=20),
        # a short prompt with five alternatives a place; an odd vocabulary inside padded rows
        dict(name="logprobs_prompt_333_odd", op="token_logprobs", rows=333, vocab=65521, pad=15, dtype="f32", top=5),
        # a long chunk of a prompt, the most likely token beside the given one
        dict(name="logprobs_prompt_2048", op="token_logprobs", rows=2048, vocab=131072, pad=0, dtype="f32", top=1),
        # four chats' next tokens scored straight from their hidden states: the table streams once
        dict(name="head_decode_4", op="head_logprobs", rows=4, width=6144, vocab=154880),
        # a short prompt, a small model, an odd vocabulary
        dict(name="head_prompt_300_odd", op="head_logprobs", rows=300, width=2048, vocab=65521),
        # a chunk of a prompt of the medium size: the largest product
        dict(name="head_prompt_2048", op="head_logprobs", rows=2048, width=4096, vocab=131072),
        # drafted tokens of four chats
        dict(name="append_drafts_32", op="append", rows=32, heads=32, kv_heads=8, dim=128, vdim=128, rot=64, pairs=False, norm=True, page=64),
        # a prompt's chunk; rotation over whole heads, in pairs
        dict(name="append_prompt_8191", op="append", rows=8191, heads=64, kv_heads=8, dim=128, vdim=128, rot=128, pairs=True, norm=True, page=64),
        # one token of one chat over a short cache: the smallest attention
        dict(name="tree_1_token_777", op="tree_attention", seqs=1, tree=1, length=777, heads=16, kv_heads=4, dim=128, vdim=128, page=64, sink=False, ragged=False),
        # four chats, each with a tree of sixteen tokens deep into their context
        dict(name="tree_4x16_30000", op="tree_attention", seqs=4, tree=16, length=30000, heads=32, kv_heads=8, dim=128, vdim=128, page=64, sink=False, ragged=False),
        # many requests of unequal lengths with trees of unequal sizes, small pages, sinks
        dict(name="tree_ragged_48_5000", op="tree_attention", seqs=48, tree=8, length=5000, heads=32, kv_heads=8, dim=128, vdim=128, page=16, sink=True, ragged=True),
        # a wide tree at the far end of a long context
        dict(name="tree_1x60_131000", op="tree_attention", seqs=1, tree=60, length=131000, heads=64, kv_heads=8, dim=128, vdim=128, page=128, sink=False, ragged=False),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["token_logprobs", "head_logprobs", "append", "tree_attention"])
    if op == "token_logprobs":
        vocab = _log(rng, 1000, 154880)
        rows = _log(rng, 1, min(2048, 2048 * 131072 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 7]), dtype=rng.choice(["bf16", "f32"]), top=rng.choice([0, 1, 5, 20]))
    if op == "head_logprobs":
        width, vocab = 8 * _log(rng, 16, 768), _log(rng, 1000, 154880)
        rows = _log(rng, 1, min(2048, 2048 * 4096 * 131072 // (width * vocab)))
        return dict(op=op, rows=rows, width=width, vocab=vocab)
    heads, kv_heads = rng.choice([(16, 4), (32, 8), (64, 8), (8, 8), (12, 2)])
    dim = rng.choice([64, 128, 128, 128, 192, 80])
    vdim = rng.choice([dim, dim, 64])
    page = rng.choice([16, 48, 64, 64, 128])
    if op == "append":
        rot = rng.choice([0, dim // 4 // 2 * 2, dim // 2, dim])
        return dict(op=op, rows=_log(rng, 1, 8191), heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, rot=rot, pairs=rng.random() < 0.5, norm=rng.random() < 0.7,
                    page=page)
    seqs, tree = _log(rng, 1, 64), _log(rng, 1, 64)
    longest = min(131000, 240000 // seqs, 60 * 64 * 131000 // (seqs * tree * heads))
    return dict(op=op, seqs=seqs, tree=tree, length=_log(rng, 1, max(1, longest)), heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, page=page,
                sink=rng.random() < 0.5, ragged=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed * 7919 + 17)
    return {"case": case, **{"token_logprobs": _logits, "head_logprobs": _hidden, "append": _rows, "tree_attention": _trees}[case["op"]](case, g)}


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)


def _randint(g, low, high, shape, dtype=torch.int32):
    return torch.randint(low, high, shape, generator=g, device=DEVICE, dtype=dtype)


def _logits(case, g):
    """Logits of a language model: a wide bulk, some likely tokens, the given token mostly among those."""
    rows, vocab = case["rows"], case["vocab"]
    x = _randn(g, rows, vocab + case["pad"]).mul_(2.5)
    likely = _randint(g, 0, vocab, (rows, 12), torch.int64)
    x.scatter_(1, likely, 12.0 + 3.0 * _randn(g, rows, 12))
    tokens = torch.where(_randint(g, 0, 4, (rows,)) > 0, likely[:, 0], _randint(g, 0, vocab, (rows,), torch.int64))
    return dict(logits=x.to(TYPES[case["dtype"]])[:, :vocab], tokens=tokens)


def _hidden(case, g):
    """Normalized hidden states, most of which point to the given token's row of the table."""
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    head = _randn(g, vocab, width, dtype=torch.bfloat16).mul_(2.0 * width**-0.5)
    tokens = _randint(g, 0, vocab, (rows,), torch.int64)
    gain = 3.0 * (_randint(g, 0, 4, (rows, 1)) > 0)
    return dict(hidden=(_randn(g, rows, width) + gain * head[tokens].float()).to(torch.bfloat16), head=head, tokens=tokens)


def _pages(case, slots, seqs, g):
    """A pool in which the sequences' pages lie in no order; table entries behind a sequence's last page are -1."""
    per = [max(1, -(-s // case["page"])) for s in slots]
    order = torch.randperm(sum(per) + 3, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((seqs, max(per)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at : at + n]
        at += n
    k = _randn(g, sum(per) + 3, case["page"], case["kv_heads"], case["dim"], dtype=torch.bfloat16)
    v = _randn(g, sum(per) + 3, case["page"], case["kv_heads"], case["vdim"], dtype=torch.bfloat16)
    return dict(k=k, v=v, table=table)


def _rows(case, g):
    """Projections of consecutive tokens of up to four sequences, some way into their context."""
    rows, dim = case["rows"], case["dim"]
    seqs = min(4, rows)
    per = -(-rows // seqs)
    r = torch.arange(rows, device=DEVICE)
    first = _randint(g, 0, 100, (seqs,), torch.int64)
    seq = r // per
    slots = first[seq] + r % per
    far = _randint(g, 0, 100000, (seqs,), torch.int64)
    state = _pages(case, [100 + per] * seqs, seqs, g)
    half = case["rot"] // 2
    angle = torch.arange(131072, dtype=torch.float64, device=DEVICE)[:, None] * 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / max(half, 1))
    state |= dict(qkv=_randn(g, rows, case["heads"] * dim + case["kv_heads"] * (dim + case["vdim"]), dtype=torch.bfloat16) * 1.5,
                  positions=(far[seq] + slots).to(torch.int32), seqs=seq.to(torch.int32), slots=slots.to(torch.int32),
                  rot=torch.stack([angle.cos(), angle.sin()], -1).float() if half else None)
    state |= dict(q_norm=(1 + 0.1 * _randn(g, dim)).bfloat16(), k_norm=(1 + 0.1 * _randn(g, dim)).bfloat16()) if case["norm"] else dict(q_norm=None, k_norm=None)
    return state


def _sizes(case):
    """How many tokens are drafted for each sequence: as many for all, or evenly spread up to the largest tree."""
    return [max(1, case["tree"] * (b + 1) // case["seqs"]) if case["ragged"] else case["tree"] for b in range(case["seqs"])]


def _trees(case, g):
    """Committed tokens and a drafted tree behind them; every drafted token has an earlier one of its sequence, or the last committed one, as its parent."""
    seqs, tree, length = case["seqs"], case["tree"], case["length"]
    cpu = torch.Generator().manual_seed(g.initial_seed() % (1 << 40))
    pick = lambda low, high: int(torch.randint(low, high + 1, (1,), generator=cpu))  # noqa: E731
    lengths = [pick(length // 3, length) if case["ragged"] else length for _ in range(seqs)]
    lengths[0] = length
    sizes = _sizes(case)
    sizes = [sizes[i] for i in torch.randperm(seqs, generator=cpu).tolist()]
    masks = []
    for n in sizes:
        own_masks = []
        for j, u in enumerate(torch.rand(n, generator=cpu).tolist()):
            parent = int(u * (min(j, 4) + 1)) - 1 + max(0, j - 4)  # one of the last four, or (for the first ones) the committed tokens
            own_masks.append((own_masks[parent] if parent >= 0 else 0) | 1 << j)
        masks += [m - (1 << 64) if m >> 63 else m for m in own_masks]
    starts = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32)
    state = _pages(case, [n + t for n, t in zip(lengths, sizes)], seqs, g)
    return state | dict(q=(1.5 * _randn(g, sum(sizes), case["heads"], case["dim"])).bfloat16(), starts=starts.to(DEVICE), lengths=torch.tensor(lengths, dtype=torch.int32).to(DEVICE),
                        masks=torch.tensor(masks, dtype=torch.int64).to(DEVICE), scale=case["dim"] ** -0.5,
                        sink=2.0 + _randn(g, case["heads"]) if case["sink"] else None)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own(state)
    return {"token_logprobs": _plain_token_logprobs, "head_logprobs": _plain_head_logprobs, "append": _plain_append,
            "tree_attention": _plain_tree_attention}[state["case"]["op"]](state)


def _own(s):
    from glm_tpu_b200.layers import logprobs
    from glm_tpu_b200.layers.attention import paged

    case = s["case"]
    if case["op"] == "token_logprobs":
        out = logprobs.token_logprobs(s["logits"], s["tokens"], top=case["top"])
        answer = {"logprob": out.logprob, "entropy": out.entropy, "best": out.best}
        return answer | {"top_ids": out.top_ids, "top_logprobs": out.top_logprobs} if case["top"] else answer
    if case["op"] == "head_logprobs":
        out = logprobs.head_logprobs(s["hidden"], s["head"], s["tokens"])
        return {"logprob": out.logprob, "entropy": out.entropy, "best": out.best}
    cache = paged.PagedKV(s["k"], s["v"], s["table"])
    if case["op"] == "append":
        q = paged.append(s["qkv"], cache, s["positions"], s["seqs"], s["slots"], heads=case["heads"], rot=s["rot"], pairs=case["pairs"], q_norm=s["q_norm"],
                         k_norm=s["k_norm"], eps=1e-6)
        return {"q": q, "k": s["k"], "v": s["v"]}
    return paged.tree_attention(s["q"], cache, s["starts"], s["lengths"], s["masks"], s["scale"], max_rows=case["tree"], sink=s["sink"])


def _scores_of(x, tokens):
    """``x``: fp32 logits."""
    z = x - x.amax(1, keepdim=True)
    logp = z - z.exp().sum(1, keepdim=True).log()
    return {"logprob": logp.gather(1, tokens[:, None])[:, 0], "entropy": -(logp.exp() * logp).sum(1), "best": logp.amax(1)}


def _plain_token_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    out = _scores_of(x, s["tokens"])
    if top:
        # largest first, equal ones by their id: the fp32 order as integers (+0 and -0 alike), the id's complement below it
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        ids = torch.arange(x.shape[1], device=x.device)
        keys = order * (1 << 31) + ((1 << 31) - 1 - ids)
        chosen = (1 << 31) - 1 - (keys.topk(top, dim=1).values & ((1 << 31) - 1))
        lse = x.gather(1, chosen[:, :1]) - out["best"][:, None]
        out |= {"top_ids": chosen.to(torch.int32), "top_logprobs": x.gather(1, chosen) - lse}
    return out


def _plain_head_logprobs(s):
    return _scores_of(s["hidden"].float() @ s["head"].float().T, s["tokens"])


def _rotated(x, cs, pairs):
    """``x [rows, heads, dim]`` fp32; ``cs [rows, rot / 2, 2]``: the leading ``rot`` channels turned, as halves or as neighbouring pairs."""
    half = cs.shape[1]
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    head, tail = x[..., : 2 * half], x[..., 2 * half :]
    a, b = (head[..., 0::2], head[..., 1::2]) if pairs else (head[..., :half], head[..., half:])
    turned = (a * c - b * sn, a * sn + b * c)
    return torch.cat([torch.stack(turned, -1).flatten(-2) if pairs else torch.cat(turned, -1), tail], -1)


def _plain_append(s):
    case, qkv = s["case"], s["qkv"]
    rows, H, G, dim = qkv.shape[0], case["heads"], case["kv_heads"], case["dim"]
    q, k, v = qkv.split([H * dim, G * dim, G * case["vdim"]], dim=1)
    q, k = q.float().view(rows, H, dim), k.float().view(rows, G, dim)
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_norm"].float()
    if s["rot"] is not None:
        cs = s["rot"][s["positions"].long()]
        q, k = _rotated(q, cs, case["pairs"]), _rotated(k, cs, case["pairs"])
    slots = s["slots"].long()
    page = s["table"][s["seqs"].long(), slots // case["page"]].long()
    s["k"][page, slots % case["page"]] = k.bfloat16()
    s["v"][page, slots % case["page"]] = v.reshape(rows, G, case["vdim"])
    return {"q": q.bfloat16(), "k": s["k"], "v": s["v"]}


def _plain_tree_attention(s):
    case = s["case"]
    seqs, tree, H, G, dim, vdim = case["seqs"], case["tree"], case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    rows = s["q"].shape[0]
    r = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(s["starts"][1:].long(), r, right=True)
    at = r - s["starts"].long()[seq]
    q = torch.zeros((seqs, tree, H, dim), device=DEVICE)
    q[seq, at] = s["q"].float()
    masks = torch.zeros((seqs, tree), dtype=torch.int64, device=DEVICE)
    masks[seq, at] = s["masks"]
    pages = s["table"].long().clamp(min=0)
    k = s["k"][pages].flatten(1, 2).float()  # [seqs, slots, G, dim]
    v = s["v"][pages].flatten(1, 2).float()
    slots = torch.arange(k.shape[1], device=DEVICE)
    drafted = slots[None, :] - s["lengths"][:, None]
    seen = (drafted[:, None] < 0) | ((drafted[:, None] < 64) & ((masks[:, :, None] >> drafted[:, None].clamp(0, 63)) & 1).bool())
    scores = torch.matmul(q.view(seqs, tree, G, H // G, dim).permute(0, 2, 3, 1, 4).reshape(seqs, G, -1, dim), k.permute(0, 2, 3, 1)).mul_(s["scale"])
    scores = scores.view(seqs, G, H // G, tree, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, G, H // G, 1, 1)
        m = torch.maximum(m, sink)
    p = scores.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + (sink - m).exp()
    out = torch.matmul(p.view(seqs, G, -1, p.shape[-1]), v.permute(0, 2, 1, 3)).view(seqs, G, H // G, tree, vdim) / total
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, tree, H, vdim)[seq, at].bfloat16()


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("token_logprobs", "head_logprobs"):
        parts = []
        step = max(1, (1 << 28) // case["vocab"])
        table = s["head"].double().T if case["op"] == "head_logprobs" else None
        for r in range(0, case["rows"], step):
            x = s["hidden"][r : r + step].double() @ table if table is not None else s["logits"][r : r + step].double()
            p = torch.softmax(x, 1)
            norm = torch.logsumexp(x, 1)
            part = [x[torch.arange(x.shape[0]), s["tokens"][r : r + step]] - norm, norm - (p * x).sum(1), x.max(1).values - norm]
            if case.get("top"):
                part.append(x.topk(case["top"], dim=1).values - norm[:, None])
            parts.append(part)
        done = [torch.cat(column) for column in zip(*parts)]
        out = {"logprob": done[0], "entropy": done[1], "best": done[2]}
        return out | {"top_ids": None, "top_logprobs": done[3]} if case.get("top") else out
    G, page = case["kv_heads"], case["page"]
    per = case["heads"] // G
    if case["op"] == "append":
        rows, dim, half = case["rows"], case["dim"], case["rot"] // 2
        x = s["qkv"].double()[:, : (case["heads"] + G) * dim].view(rows, -1, dim).clone()
        if case["norm"]:
            weight = torch.cat([s["q_norm"].double().expand(case["heads"], dim), s["k_norm"].double().expand(G, dim)])
            x = x / (x.pow(2).sum(-1, keepdim=True) / dim + 1e-6).sqrt() * weight
        first = torch.arange(half, device=DEVICE) * (2 if case["pairs"] else 1)
        second = first + (1 if case["pairs"] else half)
        if half:
            turn = torch.view_as_complex(s["rot"].double()[s["positions"].long()])[:, None]
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
        k, v = s["k"].double(), s["v"].double()
        place = s["table"].long()[s["seqs"].long(), s["slots"].long() // page] * page + s["slots"].long() % page
        k.view(-1, G, dim)[place] = x[:, case["heads"] :]
        v.view(-1, G, case["vdim"])[place] = s["qkv"].double()[:, (case["heads"] + G) * dim :].view(rows, G, -1)
        return {"q": x[:, : case["heads"]], "k": k, "v": v}
    out = torch.zeros((s["q"].shape[0], case["heads"], case["vdim"]), dtype=torch.float64, device=DEVICE)
    starts = s["starts"].tolist()
    for b, n in enumerate(s["lengths"].tolist()):
        r0, r1 = starts[b], starts[b + 1]
        slots = torch.arange(n + r1 - r0, device=DEVICE)
        where = s["table"][b].long()[slots // page], slots % page
        seen = torch.ones((r1 - r0, slots.numel()), dtype=torch.bool, device=DEVICE)
        for t in range(r1 - r0):
            seen[:, n + t] = (s["masks"][r0:r1] >> t & 1) == 1
        for h in range(case["heads"]):
            w = s["q"][r0:r1, h].double() @ s["k"][where[0], where[1], h // per].double().T * s["scale"]
            w = torch.where(seen, w, -math.inf)
            if s["sink"] is not None:
                w = torch.cat([w, s["sink"][h].double().expand(r1 - r0, 1)], 1)
            w = torch.softmax(w, 1)[:, : slots.numel()]
            out[r0:r1, h] = w @ s["v"][where[0], where[1], h // per].double()
    return out


def work(case):
    if case["op"] == "token_logprobs":
        rows, vocab = case["rows"], case["vocab"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": rows * vocab * size + rows * (20 + 8 * case["top"]), "flops": 5.0 * rows * vocab}
    if case["op"] == "head_logprobs":
        rows, width, vocab = case["rows"], case["width"], case["vocab"]
        return {"bytes": 2 * width * (rows + vocab) + 20 * rows, "flops": 2.0 * rows * width * vocab}
    H, G, dim, vdim = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    if case["op"] == "append":
        return {"bytes": case["rows"] * (4 * ((H + G) * dim + G * vdim) + 12), "flops": 8.0 * case["rows"] * (H + G) * dim}
    length = case["length"] * (2 / 3 if case["ragged"] else 1.0)  # the mean of what is drawn
    rows = sum(_sizes(case))
    return {"bytes": 2 * (case["seqs"] * length + rows) * G * (dim + vdim) + 2 * rows * H * (dim + vdim), "flops": 2.0 * rows * H * (dim + vdim) * length}
