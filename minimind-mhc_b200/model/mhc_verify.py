"""Verification of drafted tokens against the target's probabilities.

    path, kept, following = verify_drafts(tokens, parents, cu_tokens, target, draft, random)

decides which of a step's drafted tokens are kept, so that the answer is distributed as if the target had drawn every
token itself, and draws the next one.  The random numbers are the caller's.  CUDA tensors only.

That holds where the children of a row are drawn from its row of ``draft`` independently of each other, with replacement
(the same token may come twice), or, without ``draft``, are chosen without chance.  Children drawn without replacement, as
``torch.multinomial`` draws several unless told otherwise, give another distribution.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat


class Verified(NamedTuple):
    path: torch.Tensor  # (T,) int32: from cu_tokens[b] on the kept rows within the sequence, row 0 first, then -1
    kept: torch.Tensor  # (B,) int32: how many, row 0 included
    next: torch.Tensor  # (B,) int64: the token behind the last kept one


def verify_drafts(tokens: torch.Tensor, parents: torch.Tensor, cu_tokens: torch.Tensor, target: torch.Tensor,
                  draft: torch.Tensor | None, random: torch.Tensor) -> Verified:
    """Walks every sequence's drafted tree from its first row and keeps what passes.

    Sequence b's rows are ``[cu_tokens[b], cu_tokens[b + 1])``: its last token, then the drafted ones, each behind its
    parent; ``parents`` (T,) int32 index within the sequence, -1 for the first row.  ``tokens`` (T,) int64.  Row t of
    ``target`` (T, V) holds the target's probabilities of the token behind row t, row t of ``draft`` those that the
    children of t were drawn from, each by itself; ``None`` where they were not drawn (the draft's best, for one).  Both fp32, bf16 or
    fp16, alike, rows that sum to one.  ``random`` (T,) fp32 in [0, 1).

    The children x of the last kept row are tested in their order.  With rest the target's row and mass 1 at first, x is
    kept if ``random * mass * draft(x) < rest(x)`` (draft(x) = 1 without a draft).  If not, rest becomes
    max(rest - mass * draft, 0), mass its sum; without a draft mass loses rest(x), down to 0, and rest(x) becomes 0.  The next token
    is the first whose cumulative sum of rest exceeds the first row's random number times the sum.  Where nothing of
    rest is left it is drawn from the target's row; -1 if that has no positive finite sum, and for empty sequences.
    Sums are fp64.  NaN and negative probabilities count as 0; tokens outside the vocabulary, parents that do not come
    before their row and rows behind a sequence's first 1024 are not kept.
    """
    return Verified(*nat.host().verify_drafts(tokens, parents, cu_tokens, target, draft, random))
