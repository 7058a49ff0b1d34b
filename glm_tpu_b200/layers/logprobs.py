"""Log probabilities of given tokens: scoring of prompts, the probability of an answer's tokens, checking drafted ones.

Per row of logits ``x`` and token ``k``: ``logprob = x_k - lse(x)``, ``entropy = - sum p log p`` (nats), ``best = max(x) - lse(x)`` (equal to ``logprob``
exactly where the token is a most likely one), and on request the ``top`` most likely tokens, ties to the lowest id.  Everything is fp32.  A token of -1
asks for nothing and gets NaN, and so does any other one outside the vocabulary (``status``: bad index).  Minus infinity is a masked token; a row of
nothing else has log probabilities of minus infinity and entropy 0.  A row with NaN or plus infinity gives NaN and ids of -1 (``status``: not finite).

``status``: an int32 tensor of one element on the same GPU into which these conditions are OR-ed; without one they only show in the numbers.
"""

from __future__ import annotations

import torch

from glm_tpu_b200.layers.contracts import TokenLogprobs
from glm_tpu_b200.ops import native
from glm_tpu_b200.oracle import scoring

MAX_TOP = 32


def _check_tokens(tokens: torch.Tensor, rows: int, device: int, status: torch.Tensor | None) -> None:
    if tokens.shape != (rows,) or tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tokens are int32 or int64, one for each of the {rows} rows")
    if tokens.get_device() != device:
        raise ValueError("tokens and rows lie on one device")
    if status is not None and (status.numel() != 1 or status.dtype is not torch.int32 or status.get_device() != device):
        raise ValueError("the status is one element of int32 on the device of the rows")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, status: torch.Tensor | None = None) -> TokenLogprobs:
    """``logits [rows, vocab]`` bf16 or fp32, contiguous along a row; ``tokens [rows]``; up to 32 alternatives a row.  One pass over the logits."""
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32) or not logits.shape[1]:
        raise ValueError("logits are [rows, vocab] in bf16 or fp32")
    rows, vocab = logits.shape
    _check_tokens(tokens, rows, logits.get_device(), status)
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"between 0 and {min(MAX_TOP, vocab)} alternatives")
    if not logits.is_cuda:
        return scoring.token_logprobs(logits, tokens, top)
    if logits.stride(1) != 1 and vocab > 1:
        raise ValueError("logits are contiguous along a row")
    with native.on_device(logits):
        sums = logits.new_empty((3, rows), dtype=torch.float32)
        ids = logits.new_empty((rows, top), dtype=torch.int32) if top else None
        alternatives = logits.new_empty((rows, top), dtype=torch.float32) if top else None
        native.token_logprobs(logits, tokens.contiguous(), sums, ids, alternatives, status=status)
    return TokenLogprobs(*sums.unbind(0), ids, alternatives)


def head_logprobs(hidden: torch.Tensor, head: torch.Tensor, tokens: torch.Tensor, *, vocab: int | None = None, status: torch.Tensor | None = None) -> TokenLogprobs:
    """The same, without alternatives, from ``hidden [rows, width]`` and the output table ``head [>= vocab, width]`` (both bf16 or both fp32): logits
    ``hidden @ head[:vocab].T`` with fp32 sums, which are not rounded and, in bf16 with many rows, never written.  On a GPU the width is a multiple of 8."""
    if hidden.dim() != 2 or head.dim() != 2 or hidden.dtype != head.dtype or hidden.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("hidden states and table are two-dimensional, both bf16 or both fp32")
    rows, width = hidden.shape
    vocab = head.shape[0] if vocab is None else int(vocab)
    if head.shape[1] != width or width < 1 or not 0 < vocab <= head.shape[0]:
        raise ValueError("the table has a row as wide as the hidden states for every token of the vocabulary")
    _check_tokens(tokens, rows, hidden.get_device(), status)
    if head.get_device() != hidden.get_device():
        raise ValueError("hidden states and table lie on one device")
    if not hidden.is_cuda:
        return scoring.head_logprobs(hidden, head[:vocab], tokens)
    if width % 8 or hidden.stride(1) != 1 or head.stride(1) != 1 or hidden.stride(0) % 8 or head.stride(0) % 8 or (hidden.data_ptr() | head.data_ptr()) % 16:
        raise ValueError("rows of hidden states and table are contiguous, 16-byte aligned and a multiple of 8 wide")
    with native.on_device(hidden):
        if rows > 1 and hidden.stride(0) < width:  # rows that share memory (``expand``): a tensor map holds rows that lie apart
            hidden = hidden.contiguous()
        if vocab > 1 and head.stride(0) < width:
            head = head[:vocab].contiguous()
        sums = hidden.new_empty((3, rows), dtype=torch.float32)
        native.head_logprobs(hidden, head, vocab, tokens.contiguous(), sums, status=status)
    return TokenLogprobs(*sums.unbind(0), None, None)
