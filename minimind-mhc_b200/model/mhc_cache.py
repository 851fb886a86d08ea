"""A paged cache of keys and values, the attention that reads it, and the moves of a step with drafted tokens.

    cache = PagedCache(layers=8, pages=1024, page_size=64, kv_heads=4, dim=96)
    step = CacheStep(page_table, lengths, cu_tokens)                     # what this step adds, and where
    q = append_kv(cache.keys[i], cache.values[i], step, k, v, q=q, rotary=rotary)
    out = cached_attention(q, cache.keys[i], cache.values[i], step)      # (T, heads, D)
    lengths += cu_tokens.diff()

This is the reference's decoding with past keys and values (``model/model_minimind.py:200-250``) over sequences of
different lengths without copies of the past.  With drafted tokens ``mask`` says which new tokens a new token sees
(``tree_mask``), ``positions`` where they stand, and after the verification (``model/mhc_verify.py``) ``keep_drafts``
moves the kept ones up.  CUDA tensors only.  No gradients.  The checks and allocations are in
``csrc/host/mhc_torch.cpp``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat
from .mhc_rotary import Rotary


class PagedCache:
    """Keys and values of all layers in pages of ``page_size`` tokens: ``keys`` and ``values`` are (layers, pages,
    page_size, kv_heads, dim).  Which page belongs to whom is the caller's bookkeeping.  The functions below take any
    tensors of that shape (one layer: without the first dimension), whatever their strides, with contiguous heads; those
    that write to them no expanded ones."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, dim: int, dtype=torch.bfloat16, device="cuda"):
        shape = (layers, pages, page_size, kv_heads, dim)
        self.keys = torch.zeros(shape, dtype=dtype, device=device)
        self.values = torch.zeros(shape, dtype=dtype, device=device)


class CacheStep(NamedTuple):
    """What one step adds to the cache, all on the device and only read there (a captured step can be replayed with
    other numbers in them).  Sequence b has ``lengths[b]`` tokens in the cache; its new ones are the rows
    ``[cu_tokens[b], cu_tokens[b + 1])`` of the step's tokens, and place p of a sequence is slot ``p % page_size`` of page
    ``page_table[b, p // page_size]``.  Places behind the table and pages that the cache does not have do not exist:
    nothing is written there, and what is read there is not seen."""
    page_table: torch.Tensor  # (B, most pages of a sequence) int32
    lengths: torch.Tensor     # (B,) int32
    cu_tokens: torch.Tensor   # (B + 1,) int32, not decreasing


def append_kv(keys: torch.Tensor, values: torch.Tensor, step: CacheStep, k: torch.Tensor, v: torch.Tensor,
              q: torch.Tensor | None = None, rotary: Rotary | None = None,
              positions: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes the new tokens' k and v (T, kv_heads, D) to their places in one layer's ``keys`` and ``values``.

    With ``rotary`` the keys are rotated on the way, and so are the queries q (T, heads, D), which are returned (rows of no
    sequence are 0).  A token's position is its place, or ``positions[t]`` (int32 or int64): drafted tokens stand at
    ``lengths[b]`` plus their depth in the tree.  All tensors have the cache's type.
    """
    if rotary is None:
        turns, interleaved, gain = None, False, 1.0
    else:
        turns = rotary.turns(k.device) if k.is_cuda else rotary._host
        interleaved, gain = rotary.interleaved, rotary.gain
    return nat.host().append_kv(keys, values, *step, k, v, q, positions, turns, interleaved, gain)


def cached_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, step: CacheStep,
                     mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of the new tokens' queries q (T, H, D) over their sequences' cache, the new tokens included.

    A token sees all of its sequence's ``lengths[b]`` earlier tokens and, of the new ones, itself and those before it or,
    with ``mask`` (T,) int64, new token c where bit c is set (the first 64 of a sequence can be seen).  H is a multiple of
    the cache's heads; D at most 128; ``scale`` defaults to ``D ** -0.5``.  A token that sees nothing gets 0, rows of no
    sequence too.  What a token does not see, NaN and infinities included, does not touch it.  The same bits every time.
    """
    return nat.host().cached_attention(q, keys, values, *step, mask, scale)


def keep_drafts(keys: torch.Tensor, values: torch.Tensor, step: CacheStep, path: torch.Tensor, kept: torch.Tensor) -> None:
    """Moves the kept tokens' keys and values to the places right behind the context, in all layers of ``keys`` and
    ``values`` at once: the i-th of ``kept[b]`` is new token ``path[cu_tokens[b] + i]`` of its sequence, ascending, as
    ``verify_drafts`` returns them.  The sequence's new length is ``lengths[b] + kept[b]``.
    """
    nat.host().keep_drafts(keys, values, *step, path, kept)


def tree_mask(parents: torch.Tensor, cu_tokens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(mask, depth) of drafted trees: for every row the bits of itself and its ancestors, and how many ancestors it has.

    ``parents`` (T,) is the index of a row's parent within its sequence, below its own; -1 for the first.  (A row whose
    parent is none of that is taken for a first one, and so are all rows of no sequence.)  Trees of up to 64 rows.  Plain
    torch operations, on the tensors' device and without waiting for it: a tree that stays the same is done once.
    """
    if parents.dim() != 1 or cu_tokens.dim() != 1 or cu_tokens.numel() < 1:
        raise ValueError(f"tree_mask: parents (T,) and cu_tokens (B + 1,) are wanted, got {tuple(parents.shape)}, {tuple(cu_tokens.shape)}")
    t = parents.shape[0]
    at = torch.arange(t, device=parents.device)
    start = cu_tokens.long()[torch.searchsorted(cu_tokens[1:].long().contiguous(), at, right=True).clamp(max=cu_tokens.numel() - 2)]
    start = torch.where(at < cu_tokens[-1], start, at)  # rows behind the last sequence are their own first ones
    child = (parents >= 0) & (parents < at - start) & (start >= 0)
    up = torch.where(child, start + parents.long(), at)  # a root is its own parent
    mask = torch.ones_like(at) << (at - start).clamp(0, 63)
    depth = child.long()
    for _ in range(6):  # the ancestors at twice the distance
        mask, depth, up = mask | mask[up], depth + depth[up], up[up]
    return mask, depth
