"""Causal attention over packed sequences, with grouped heads.

    out = packed_attention(q, k, v, cu_seqlens)     # (T, H, D): sequences back to back
    out = packed_attention(q, k, v)                 # (B, L, H, D): B rows of L tokens

computes what the reference's ``Attention.forward`` asks of
``scaled_dot_product_attention`` (``model/model_minimind.py:220-250``: causal,
the query heads of a group sharing a key / value head), and the same over
sequences of different lengths packed into one row, where a token sees the
tokens up to itself of its own sequence only.  CUDA tensors only.  The checks,
the allocations and the autograd node are in ``csrc/host/mhc_torch.cpp``.
"""

from __future__ import annotations

import torch

from . import _native as nat


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Causal attention of every sequence over itself.

    q (T, H, D) with k, v (T, Hk, D) and ``cu_seqlens`` (B + 1) int32 on the
    device, the sequences' offsets; or q (B, L, H, D) with k, v (B, L, Hk, D)
    and no ``cu_seqlens``.  H is a multiple of Hk, D at most 128; fp32, bf16 or
    fp16, all three alike; rows may lie at any strides (slices of one
    projection's output are read in place).  Under autocast all three are cast
    to its type, as ``scaled_dot_product_attention`` does.  ``scale`` defaults
    to ``D ** -0.5``.  Second and forward-mode derivatives are refused, as are
    tracers (``torch.jit.trace``, ``make_fx``).

    Sequences may be empty.  Tokens before ``cu_seqlens[0]`` or from
    ``cu_seqlens[-1]`` on belong to none: their output and gradients are 0, and
    nothing they hold reaches another token.  The offsets are read on the
    device: they are not checked beyond their type.  A NaN or infinity reaches
    what sees it by the formula, and neither another sequence nor an earlier
    token.
    """
    return nat.host().packed_attention(q, k, v, cu_seqlens, scale)
