"""CPU restatement of the operators for scoring given tokens and for steps over drafted tokens (``layers.logprobs``, ``layers.attention.paged``).

Plain PyTorch, row by row where that is clearer, in 64 bits between the inputs and the one rounding of the result.
"""

from __future__ import annotations

import math

import torch

from glm_tpu_b200.layers.contracts import TokenLogprobs


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int) -> TokenLogprobs:
    x = logits.double()
    rows, vocab = x.shape
    bad = torch.isnan(x).any(1) | (x == math.inf).any(1)
    empty = (x == -math.inf).all(1)
    m = x.amax(1)
    shift = torch.where(bad | empty, torch.zeros_like(m), m)
    e = (x - shift[:, None]).exp()
    s = e.sum(1)
    norm = torch.where(empty, torch.zeros_like(s), s.log())
    logp = x - shift[:, None] - norm[:, None]  # minus infinity where the logit is
    entropy = torch.where(empty, torch.zeros_like(s), norm - torch.where(e > 0, (x - shift[:, None]) * e, torch.zeros_like(x)).sum(1) / s.clamp(min=1e-300))
    k = tokens.long()
    known = (k >= 0) & (k < vocab)
    given = logp.gather(1, k.clamp(0, vocab - 1)[:, None])[:, 0]
    nan = torch.full_like(given, math.nan)
    out = [torch.where(bad | ~known, nan, given), torch.where(bad, nan, entropy), torch.where(bad, nan, logp.amax(1))]
    ids = alternatives = None
    if top:
        ids = torch.sort(torch.nan_to_num(x, nan=0.0), dim=1, descending=True, stable=True).indices[:, :top]
        alternatives = torch.where(bad[:, None], nan[:, None], logp.gather(1, ids)).float()
        ids = torch.where(bad[:, None], torch.full_like(ids, -1), ids).to(torch.int32)
    return TokenLogprobs(*(v.float() for v in out), ids, alternatives)


def head_logprobs(hidden: torch.Tensor, head: torch.Tensor, tokens: torch.Tensor) -> TokenLogprobs:
    return token_logprobs(hidden.double() @ head.double().T, tokens, 0)


def page_of(table: torch.Tensor, seq: int, slot: int, page: int, pages: int) -> int:
    """The page that holds ``slot`` of a sequence, or -1."""
    if not 0 <= seq < table.shape[0] or not 0 <= slot < table.shape[1] * page:
        return -1
    at = int(table[seq, slot // page])
    return at if 0 <= at < pages else -1


def append(qkv, k_pool, v_pool, table, positions, seqs, slots, *, heads: int, q_norm, k_norm, eps: float, rot, pairs: bool) -> torch.Tensor:
    """Writes into the pools; returns the queries ``[rows, heads, dim]``."""
    pages, page, G, dim = k_pool.shape
    vdim = v_pool.shape[3]
    rows = qkv.shape[0]
    x = qkv[:, : (heads + G) * dim].double().reshape(rows, heads + G, dim)
    v = qkv[:, (heads + G) * dim :].reshape(rows, G, vdim)
    for first, last, weight in ((0, heads, q_norm), (heads, heads + G, k_norm)):
        if weight is not None:
            part = x[:, first:last]
            x[:, first:last] = part / (part.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = 0 if rot is None else rot.shape[1]
    a_at = torch.arange(half) * (2 if pairs else 1)
    b_at = a_at + (1 if pairs else half)
    for r in range(rows):
        pos, slot, seq = int(positions[r]) if rot is not None else 0, int(slots[r]), int(seqs[r])
        at = page_of(table, seq, slot, page, pages) if slot >= 0 else 0
        if at < 0 or pos < 0 or (rot is not None and pos >= rot.shape[0]):
            x[r, :heads] = 0.0
            continue
        if half:
            c, s = rot[pos, :, 0].double(), rot[pos, :, 1].double()
            a, b = x[r][:, a_at].clone(), x[r][:, b_at].clone()
            x[r][:, a_at], x[r][:, b_at] = a * c - b * s, a * s + b * c
        if slot >= 0:
            k_pool[at, slot % page] = x[r, heads:].to(k_pool.dtype)
            v_pool[at, slot % page] = v[r].to(v_pool.dtype)
    return x[:, :heads].to(qkv.dtype)


def tree_attention(q, k_pool, v_pool, table, starts, lengths, masks, scale: float, max_rows: int, sink, out: torch.Tensor) -> torch.Tensor:
    pages, page, G, _ = k_pool.shape
    rows, H, _ = q.shape
    for b in range(table.shape[0]):
        r0 = min(max(int(starts[b]), 0), rows)
        count = max(min(int(starts[b + 1]), rows) - r0, 0)
        length = min(max(int(lengths[b]), 0), table.shape[1] * page)
        drafts = min(count, max_rows)
        where = [page_of(table, b, s, page, pages) for s in range(length + drafts)]
        for j in range(drafts):
            seen = [s for s, at in enumerate(where) if at >= 0 and (s < length or int(masks[r0 + j]) >> (s - length) & 1)]
            at = torch.tensor([where[s] for s in seen], dtype=torch.long), torch.tensor([s % page for s in seen], dtype=torch.long)
            k, v = (pool[at[0], at[1]].double().repeat_interleave(H // G, dim=1) for pool in (k_pool, v_pool))  # [keys, H, ..]
            w = torch.einsum("hd,khd->hk", q[r0 + j].double(), k) * scale
            if sink is not None:
                w = torch.cat([w, sink.double()[:, None]], 1)
            if w.shape[1] == 0:
                out[r0 + j] = 0
                continue
            out[r0 + j] = torch.einsum("hk,khd->hd", torch.softmax(w, 1)[:, : len(seen)], v).to(out.dtype)
    return out
