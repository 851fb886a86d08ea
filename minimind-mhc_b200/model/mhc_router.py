"""Top-k router of a mixture of experts with its balance loss, in one pass over
the logits in each direction.

    weights, experts, counts, aux_loss = route_topk(gate(x), k, aux_coef=5e-4)

computes what the reference's ``MOEFeedForward`` computes around its gate
(``model/model_minimind.py:262-293``): the softmax over the experts, the k
largest of each token, their weights renormalised to one, and the balance loss
``coef * E * sum_e load_e * mean_t p_te``; and the experts' counts, which a
caller that groups tokens by expert needs next.  CUDA tensors only.
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


class _RouteFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, k, coef):
        t, e = logits.shape
        z = logits if t == 0 or (logits.stride(1) == 1 and logits.stride(0) >= e) else logits.contiguous()
        rs = z.stride(0) if t > 1 else e
        index = z.get_device()
        weights = z.new_empty((t, k), dtype=torch.float32)
        experts = z.new_empty((t, k), dtype=torch.int64)
        counts = z.new_empty((e,), dtype=torch.int64)
        loss = z.new_empty((), dtype=torch.float32)
        need = nat.lib().mhc_route_fwd_workspace(t, e)
        ws = z.new_empty((need,), dtype=torch.uint8) if need else None
        nat.call_on(index, "mhc_route_fwd", z.data_ptr(), nat.dtype_code(z.dtype), t, e, rs, k, coef,
                    weights.data_ptr(), experts.data_ptr(), counts.data_ptr(), loss.data_ptr(), nat.ptr(ws), need)
        ctx.save_for_backward(z, weights, experts, counts)
        ctx.meta = (k, coef, rs)
        ctx.mark_non_differentiable(experts, counts)
        ctx.set_materialize_grads(False)
        return weights, experts, counts, loss

    @staticmethod
    def backward(ctx, dw, _experts, _counts, dloss):
        nat.refuse_double_backward("route_topk")
        if dw is None and dloss is None:
            return None, None, None
        z, weights, experts, counts = ctx.saved_tensors
        k, coef, rs = ctx.meta
        t, e = z.shape
        if dw is not None:
            dw = dw.to(torch.float32).contiguous()
        if dloss is not None:
            dloss = dloss.to(torch.float32)
        dz = z.new_empty((t, e))
        nat.call_on(z.get_device(), "mhc_route_bwd", z.data_ptr(), nat.dtype_code(z.dtype), t, e, rs, k, coef,
                    weights.data_ptr(), experts.data_ptr(), counts.data_ptr(), nat.ptr(dw), nat.ptr(dloss),
                    dz.data_ptr())
        return dz, None, None


def route_topk(logits: torch.Tensor, k: int, aux_coef: float = 0.0) -> Routing:
    """Routes every row of ``logits`` (..., E) to its ``k`` largest experts.

    logits: fp32 / bf16 / fp16, E <= 512; the softmax and everything after it
    are fp32.  Among equal logits the lower expert index wins; NaN is above
    everything; a row of ``-inf`` has weights 0.  The gradient flows through
    ``weights`` and ``aux_loss``; the counts are constants of the loss.
    """
    nat.require_cuda(logits)
    if logits.dim() < 1:
        raise ValueError("route_topk: logits must have at least one dimension")
    nat.dtype_code(logits.dtype)
    e, k = logits.shape[-1], int(k)
    if not 1 <= e <= 512:
        raise ValueError(f"route_topk: 1 to 512 experts are supported, got {e}")
    if not 1 <= k <= e:
        raise ValueError(f"route_topk: k must be in [1, {e}], got {k}")
    flat = logits if logits.dim() == 2 else logits.reshape(-1, e)
    w, idx, counts, loss = _RouteFn.apply(flat, k, float(aux_coef))
    if logits.dim() != 2:
        w, idx = w.view(*logits.shape[:-1], k), idx.view(*logits.shape[:-1], k)
    return Routing(w, idx, counts, loss)
