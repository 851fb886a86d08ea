"""Causal attention over packed sequences, with grouped heads.

    out = packed_attention(q, k, v, cu_seqlens)     # (T, H, D): sequences back to back
    out = packed_attention(q, k, v)                 # (B, L, H, D): B rows of L tokens

computes what the reference's ``Attention.forward`` asks of
``scaled_dot_product_attention`` (``model/model_minimind.py:220-250``: causal,
the query heads of a group sharing a key / value head), and the same over
sequences of different lengths packed into one row, where a token sees the
tokens up to itself of its own sequence only.  CUDA tensors only.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as nat


def _rows(x):
    """x (T, heads, D) as the kernels read it: any token and head strides, but contiguous rows, and for 16-bit types
    what TMA can address (rows that begin at multiples of 16 bytes, heads that do not overlap), where a copy costs less
    than the kernels that do without."""
    st, sh, sd = x.stride()
    t, h, d = x.shape
    if sd != 1 and d != 1:
        return x.contiguous()
    if x.element_size() == 2 and d % 8 == 0 and (st % 8 or sh % 8 or x.data_ptr() % 16 or (h > 1 and sh < d)):
        return x.contiguous()
    return x


def _forward(q, k, v, cu, seqlen, scale, for_grad):
    """out, and what the backward needs beside it."""
    t, h, d = q.shape
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = q.new_empty((t, h, d))
    # the backward's row sums use out before its rounding to 16 bits
    out_lo = q.new_empty((t, h, d)) if for_grad and q.dtype != torch.float32 else None
    lib = nat.lib()
    lse = q.new_empty((h, lib.mhc_attn_lse_pitch(t)), dtype=torch.float32)
    strides = (ctypes.c_int64 * 6)(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2])
    batch = 0 if cu is None else cu.numel() - 1
    need = lib.mhc_attn_fwd_workspace(t)
    ws = q.new_empty((need,), dtype=torch.uint8)
    nat.call_on(q.get_device(), "mhc_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), nat.dtype_code(q.dtype), t,
                h, k.shape[1], d, strides, nat.ptr(cu), batch, seqlen, scale, out.data_ptr(), nat.ptr(out_lo),
                lse.data_ptr(), ws.data_ptr(), need)
    return out, (q, k, v, cu, out, out_lo, lse), (strides, batch, seqlen, scale)


class _PackedAttentionFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, cu, seqlen, scale):
        out, saved, ctx.meta = _forward(q, k, v, cu, seqlen, scale, True)
        ctx.save_for_backward(*saved)
        return out

    @staticmethod
    def backward(ctx, dout):
        nat.refuse_double_backward("packed_attention")
        q, k, v, cu, out, out_lo, lse = ctx.saved_tensors
        strides, batch, seqlen, scale = ctx.meta
        t, h, d = q.shape
        hk = k.shape[1]
        dout = dout.contiguous()
        dq, dk, dv = q.new_empty((t, h, d)), q.new_empty((t, hk, d)), q.new_empty((t, hk, d))
        need = nat.lib().mhc_attn_bwd_workspace(t, h, hk, d)
        ws = q.new_empty((need,), dtype=torch.uint8)
        nat.call_on(q.get_device(), "mhc_attn_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                    nat.ptr(out_lo), dout.data_ptr(), lse.data_ptr(), nat.dtype_code(q.dtype), t, h, hk, d, strides,
                    nat.ptr(cu), batch, seqlen, scale, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(),
                    need)
        return dq, dk, dv, None, None, None


def _attend(q, k, v, cu, seqlen, scale):
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttentionFn.apply(q, k, v, cu, seqlen, scale)
    return _forward(q, k, v, cu, seqlen, scale, False)[0]


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Causal attention of every sequence over itself.

    q (T, H, D) with k, v (T, Hk, D) and ``cu_seqlens`` (B + 1) int32 on the
    device, the sequences' offsets; or q (B, L, H, D) with k, v (B, L, Hk, D)
    and no ``cu_seqlens``.  H is a multiple of Hk, D at most 128; fp32, bf16 or
    fp16, all three alike; rows may lie at any strides (slices of one
    projection's output are read in place).  ``scale`` defaults to
    ``D ** -0.5``.

    Sequences may be empty.  Tokens before ``cu_seqlens[0]`` or from
    ``cu_seqlens[-1]`` on belong to none: their output and gradients are 0, and
    nothing they hold reaches another token.  The offsets are read on the
    device: they are not checked beyond their type.
    """
    nat.require_cuda(q, k, v, cu_seqlens)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"packed_attention: q, k and v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    nat.dtype_code(q.dtype)
    if not (q.device == k.device == v.device) or (cu_seqlens is not None and cu_seqlens.device != q.device):
        raise ValueError("packed_attention: q, k, v and cu_seqlens must be on one device")
    want = 4 if cu_seqlens is None else 3
    if q.dim() != want or k.dim() != want or v.dim() != want:
        raise ValueError("packed_attention: (T, heads, D) tensors with cu_seqlens or (B, L, heads, D) tensors without "
                         f"are wanted, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape != v.shape or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"packed_attention: shapes do not match: {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    h, d = q.shape[-2:]
    hk = k.shape[-2]
    if hk < 1 or h < 1 or h % hk:
        raise ValueError(f"packed_attention: {h} query heads cannot share {hk} key heads")
    if not 1 <= d <= 128:
        raise ValueError(f"packed_attention: head sizes up to 128 are supported, got {d}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"packed_attention: scale must be positive and finite, got {scale}")
    if cu_seqlens is None:
        b, l = q.shape[:2]
        return _attend(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), None, l, scale).view(b, l, h, d)
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError("packed_attention: cu_seqlens must be int32 with one offset more than there are sequences, "
                         f"got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)}")
    return _attend(q, k, v, cu_seqlens.contiguous(), 0, scale)
