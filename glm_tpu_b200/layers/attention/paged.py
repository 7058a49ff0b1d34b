"""Attention over a paged cache for a few drafted tokens per sequence, and the append that fills the cache.

A step over drafted tokens: ``append`` normalizes and rotates the rows of a fused ``q | k | v`` projection and writes keys and values into the slots behind
each sequence's committed ones; ``tree_attention`` lets every drafted token see the committed slots and its ancestors.  ``ancestor_masks`` makes the masks
of a tree.  Tokens that were accepted are appended once more, at consecutive slots (their position, and so their rotation, stays): rows of one call
are read from the projection and not from the cache, so no slot is moved within it.  A tree of one token is ordinary decoding, a chain a short prompt.

bf16, fp32 sums, one rounding of every result; in the attention a softmax weight meets the values with 16 bits.  Sequences, slots, pages and positions out of
range are never followed: they are OR-ed into ``status`` (an int32 tensor of one element on the same GPU) as a bad index, the row stores nothing and its queries
are zeros; in attention such a slot is not attended to.  What a row does not see may hold anything.  A committed value that is not finite leaves its channel so, as a
NaN or an infinity, in the rows of its sequence and in no other.
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from dataclasses import dataclass

import torch

from glm_tpu_b200.ops import native
from glm_tpu_b200.oracle import scoring

MAX_DRAFTS = 64
MAX_SLOTS = 1 << 30


@dataclass(frozen=True)
class PagedKV:
    """A pool of pages and the table that says which of them hold a sequence's slots: slot ``s`` of sequence ``b`` is row ``s % page`` of page
    ``table[b, s // page]``.  Entries behind a sequence's last page may hold anything."""

    k: torch.Tensor  # [pages, page, kv_heads, dim] bf16, a head's channels contiguous; page: a multiple of 8
    v: torch.Tensor  # [pages, page, kv_heads, vdim]
    table: torch.Tensor  # [sequences, pages of a sequence] int32


def ancestor_masks(parents: Sequence[int]) -> tuple[torch.Tensor, torch.Tensor]:
    """Masks (int64) and depths (int32) of a drafted tree on the CPU: ``parents[j] < j`` is the drafted token that token ``j`` follows, -1 the last
    committed one.  Bit ``i`` of ``masks[j]``: token ``i`` is ``j`` or one of its ancestors.  A token's position is the committed length + its depth."""
    if len(parents) > MAX_DRAFTS or any(not -1 <= p < j for j, p in enumerate(parents)):
        raise ValueError(f"up to {MAX_DRAFTS} drafted tokens, each behind its parent")
    masks, depths = [], []
    for j, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | 1 << j)
        depths.append(depths[p] + 1 if p >= 0 else 0)
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64), torch.tensor(depths, dtype=torch.int32)


def _shared(t: torch.Tensor) -> bool:
    """Whether rows of channels along an axis begin closer together than one is long (``expand``: all at one place)."""
    return any(n > 1 and step < t.shape[-1] for n, step in zip(t.shape[:-1], t.stride()))


def _checked(cache: PagedKV, device: int) -> tuple[int, ...]:
    """The cache as the kernels take it (the fields of ``native.PagedArgs``; the last seven: sequences, their pages, pages, slots of a page, heads, dim, vdim).
    ``device``: where the rows lie (-1: CPU)."""
    k, v, table = cache.k, cache.v, cache.table
    if k.dim() != 4 or v.dim() != 4 or table.dim() != 2:
        raise ValueError("pools have four axes, the table two")
    pages, page, G, dim = k.shape
    (*v_front, vdim), (seqs, per_seq) = v.shape, table.shape
    k_page, k_slot, k_head, k_last = k.stride()
    v_page, v_slot, v_head, v_last = v.stride()
    if v_front != [pages, page, G] or k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or not pages or not page or page % 8 or not G:
        raise ValueError("pools are [pages, page, kv_heads, dim] and [pages, page, kv_heads, vdim] in bf16, with a multiple of 8 slots a page")
    if table.dtype is not torch.int32 or (per_seq > 1 and table.stride(1) != 1) or per_seq * page > MAX_SLOTS:
        raise ValueError("the table is [sequences, pages of a sequence] in int32, of up to 2^30 slots a sequence")
    if k.get_device() != device or v.get_device() != device or table.get_device() != device:
        raise ValueError("rows, pools and table lie on one device")
    if not 16 <= dim <= 256 or not 16 <= vdim <= 256 or dim % 16 or vdim % 16:
        raise ValueError("heads are 16 to 256 channels wide, in multiples of 16")
    if (k_page < dim or k_slot < dim or k_head < dim or v_page < vdim or v_slot < vdim or v_head < vdim) and (_shared(k) or _shared(v)):
        raise ValueError("pages, slots and heads of the pools do not share memory")
    k_at, v_at = k.data_ptr(), v.data_ptr()
    if device >= 0 and (k_last != 1 or v_last != 1 or (k_page | k_slot | k_head | v_page | v_slot | v_head) % 8 or (k_at | v_at) % 16):
        raise ValueError("the channels of a head are contiguous and every head of the pools 16-byte aligned")
    return k_at, k_page, k_slot, k_head, v_at, v_page, v_slot, v_head, table.data_ptr(), table.stride(0), seqs, per_seq, pages, page, G, dim, vdim


def _check_index(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, device: int) -> None:
    if t.dtype is not dtype or t.shape != (n,) or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: {n} contiguous elements of {str(dtype)[6:]} on the device of the rows")


def append(qkv: torch.Tensor, cache: PagedKV, positions: torch.Tensor | None, seqs: torch.Tensor, slots: torch.Tensor, *, heads: int,
           rot: torch.Tensor | None = None, pairs: bool = False, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
           want_q: bool = True, status: torch.Tensor | None = None) -> torch.Tensor | None:
    """``qkv [rows, heads * dim + kv_heads * (dim + vdim)]`` bf16 -> queries ``[rows, heads, dim]``; keys and values into the cache.

    ``rot``: fp32 ``[positions, n, 2]`` (cos, sin) for the leading ``2 n`` channels of q and k, as halves ``(d, d + n)`` or, with ``pairs``, as neighbours
    ``(2j, 2j + 1)``; ``q_norm`` / ``k_norm``: bf16 ``[dim]``, RMS norm of every head before the rotation.  A negative slot stores nothing.  Rows of one call name different
    slots.  ``want_q=False``: keys and values only (returns ``None``)."""
    device = qkv.get_device()
    args = _checked(cache, device)
    G, dim, vdim = args[-3:]
    if qkv.dim() != 2 or qkv.dtype is not torch.bfloat16 or heads < 1 or qkv.shape[1] != heads * dim + G * (dim + vdim):
        raise ValueError("qkv is [rows, heads * dim + kv_heads * (dim + vdim)] in bf16")
    rows = qkv.shape[0]
    _check_index("seqs", seqs, rows, torch.int32, device)
    _check_index("slots", slots, rows, torch.int32, device)
    if rot is not None:
        if positions is None:
            raise ValueError("a rotation needs positions")
        _check_index("positions", positions, rows, torch.int32, device)
        if rot.dim() != 3 or not rot.shape[0] or rot.shape[2] != 2 or not 0 < 2 * rot.shape[1] <= dim or rot.dtype is not torch.float32 or not rot.is_contiguous() or rot.get_device() != device:
            raise ValueError("rot is [positions, n, 2] in fp32, contiguous, with 2 n channels at most as many as a head has")
    if status is not None:
        _check_index("status", status, 1, torch.int32, device)
    for weight in (q_norm, k_norm):
        if weight is not None:
            _check_index("norm", weight, dim, torch.bfloat16, device)
    if device < 0:
        q = scoring.append(qkv, cache.k, cache.v, cache.table, positions, seqs, slots, heads=heads, q_norm=q_norm, k_norm=k_norm, eps=eps, rot=rot, pairs=pairs)
        return q if want_q else None
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:
        raise ValueError("rows of qkv are contiguous and 16-byte aligned")
    if any(t is not None and t.data_ptr() % 16 for t in (rot, q_norm, k_norm)):
        raise ValueError("rot and the weights of the norms begin at a 16-byte boundary")
    with native.on_device(qkv):
        q = qkv.new_empty((rows, heads, dim)) if want_q else None
        native.paged_append(qkv, args, positions, seqs, slots, q, heads, rot, pairs, q_norm, k_norm, eps, status=status)
    return q


def tree_attention(q: torch.Tensor, cache: PagedKV, starts: torch.Tensor, lengths: torch.Tensor, masks: torch.Tensor, scale: float, *, max_rows: int,
                   sink: torch.Tensor | None = None, out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``q [rows, heads, dim]`` bf16 -> ``[rows, heads, vdim]``.

    Sequence ``b`` owns rows ``starts[b] .. starts[b + 1] - 1`` (int32, ascending), ``lengths[b]`` (int32) committed slots, and its drafted tokens lie in the slots behind
    those, one per row in order.  ``masks`` (int64): bit ``t`` lets a row see its sequence's drafted slot ``t``; bits of rows that the sequence does
    not have mean nothing.  ``max_rows`` (at most 64): rows of the largest sequence.  ``sink``: fp32 ``[heads]``, a score that takes weight and gives no value.  A row
    that sees nothing, without a sink, is zeros.  Rows that belong to no sequence stay as they are in ``out``, or are zeros where it is made here."""
    device = q.get_device()
    args = _checked(cache, device)
    seqs, _, _, _, G, dim, vdim = args[-7:]
    if q.dim() != 3 or q.dtype is not torch.bfloat16 or q.shape[2] != dim or not q.shape[1] or q.shape[1] % G:
        raise ValueError("q is [rows, heads, dim] in bf16, with a multiple of the cache's heads")
    rows, heads, _ = q.shape
    if seqs > 65535:
        raise ValueError("at most 65,535 sequences")
    _check_index("starts", starts, seqs + 1, torch.int32, device)
    _check_index("lengths", lengths, seqs, torch.int32, device)
    _check_index("masks", masks, rows, torch.int64, device)
    if not 1 <= max_rows <= MAX_DRAFTS:
        raise ValueError(f"between 1 and {MAX_DRAFTS} rows a sequence")
    if not 0.0 < scale < math.inf:
        raise ValueError("the scale is positive")
    if status is not None:
        _check_index("status", status, 1, torch.int32, device)
    if sink is not None:
        _check_index("sink", sink, heads, torch.float32, device)
    if out is not None and (out.shape != (rows, heads, vdim) or out.dtype is not torch.bfloat16 or out.get_device() != device):
        raise ValueError("out is [rows, heads, vdim] in bf16 on the device of q")
    if device < 0:
        out = torch.zeros((rows, heads, vdim), dtype=torch.bfloat16) if out is None else out
        return scoring.tree_attention(q, cache.k, cache.v, cache.table, starts, lengths, masks, scale, max_rows, sink, out)
    row, head, _ = q.stride()
    if (row < dim or head < dim) and _shared(q):  # a tensor map holds heads that lie apart
        q = q.contiguous()
    for t in (q,) if out is None else (q, out):
        row, head, last = t.stride()
        if t is out and (row < vdim or head < vdim) and _shared(out):
            raise ValueError("rows and heads of out do not share memory")
        if last != 1 or (row | head) % 8 or t.data_ptr() % 16:
            raise ValueError("the channels of a head are contiguous and every head of q and out 16-byte aligned")
    with native.on_device(q):
        made = out is None
        if made:
            out = (q.new_empty if seqs else q.new_zeros)((rows, heads, vdim))
        native.tree_attention(q, args, starts, lengths, masks, scale, max_rows, sink, out, clear_rest=made, status=status)
    return out
