"""Top-k router of a mixture of experts with its balance loss, in one pass over
the logits in each direction.

    weights, experts, counts, aux_loss = route_topk(gate(x), k, aux_coef=5e-4)

computes what the reference's ``MOEFeedForward`` computes around its gate
(``model/model_minimind.py:262-293``): the softmax over the experts, the k
largest of each token, their weights renormalised to one, and the balance loss
``coef * E * sum_e load_e * mean_t p_te``; and the experts' counts, which a
caller that groups tokens by expert needs next.  CUDA tensors only.  The
checks, the allocations and the autograd node are in
``csrc/host/mhc_torch.cpp``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat


class Routing(NamedTuple):
    weights: torch.Tensor   # (..., k) fp32, summing to one over the k
    experts: torch.Tensor   # (..., k) int64
    counts: torch.Tensor    # (E,) int64
    aux_loss: torch.Tensor  # () fp32


def route_topk(logits: torch.Tensor, k: int, aux_coef: float = 0.0) -> Routing:
    """Routes every row of ``logits`` (..., E) to its ``k`` largest experts.

    logits: fp32 / bf16 / fp16, E <= 512; the softmax and everything after it
    are fp32.  Among equal logits the lower expert index wins; NaN is above
    everything; a row of ``-inf`` has weights 0.  The gradient flows through
    ``weights`` and ``aux_loss``; the counts are constants of the loss.  Second
    and forward-mode derivatives and tracers are refused.
    """
    return Routing(*nat.host().route_topk(logits, int(k), float(aux_coef)))
