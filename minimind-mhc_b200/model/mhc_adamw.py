"""AdamW over many tensors in one launch, with moments in fp32 or in 8 bits.

``adamw_step`` / ``adamw_step_8bit`` are the step itself on lists of tensors, in
place; :class:`AdamW` is a ``torch.optim.Optimizer`` around them.  The update is
``torch.optim.AdamW``'s (decoupled weight decay, bias correction), which the
reference's trainers use (``trainer/train_pretrain.py:146``), with the gradient
clipping of the line before the step (``:45-52``) as an argument: the norm is
taken on the device, scales the gradients inside the step and is never read by
the host.  CUDA tensors only.

8-bit moments: 256 consecutive values of a tensor share one fp32 scale, the
largest magnitude among them.  The first moment is int8, ``(c/127)^2 * sign *
scale``, the second uint8, ``(c/255)^4 * scale``; a parameter's optimizer state
is 2.03 bytes a value instead of 8.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat

QUANT_BLOCK = 256  # values that share a scale


class Moment8(NamedTuple):
    """One tensor's moment in 8 bits: ``codes`` int8 (first moment) or uint8
    (second), ``scales`` fp32, one for every 256 values."""
    codes: torch.Tensor
    scales: torch.Tensor


def zero_moment(p: torch.Tensor, signed: bool) -> Moment8:
    """The 8-bit moment of ``p`` before the first step."""
    n = p.numel()
    return Moment8(torch.zeros(p.shape, dtype=torch.int8 if signed else torch.uint8, device=p.device),
                   torch.zeros(-(-n // QUANT_BLOCK), dtype=torch.float32, device=p.device))


def unpack_moment(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values that an 8-bit moment stands for, in the codes' shape."""
    nat.require_cuda(codes, scales)
    n = codes.numel()
    if codes.dtype not in (torch.int8, torch.uint8) or scales.dtype != torch.float32:
        raise TypeError(f"unpack_moment: int8 / uint8 codes and fp32 scales are wanted, got {codes.dtype} and "
                        f"{scales.dtype}")
    if scales.numel() != -(-n // QUANT_BLOCK):
        raise ValueError(f"unpack_moment: {n} codes have {-(-n // QUANT_BLOCK)} scales, got {scales.numel()}")
    if scales.device != codes.device:
        raise ValueError("unpack_moment: codes and scales are on different devices")
    codes, scales = codes.contiguous(), scales.contiguous()
    with torch.cuda.device(codes.device):
        out = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
        nat.call("mhc_adamw_unpack", codes.data_ptr(), int(codes.dtype == torch.int8), scales.data_ptr(),
                 out.data_ptr(), n, nat.stream_of(codes))
    return out


def _group(params, grads, ms, vs, steps, bits, lr, betas, eps, weight_decay):
    """One group of tensors as the host module takes it."""
    mscales = vscales = []
    if bits == 8:
        ms, mscales = zip(*ms) if ms else ([], [])
        vs, vscales = zip(*vs) if vs else ([], [])
    return params, grads, ms, vs, mscales, vscales, steps, lr, betas[0], betas[1], eps, weight_decay


def _step(params, grads, ms, vs, bits, step, lr, betas, eps, weight_decay, max_grad_norm):
    steps = list(step) if isinstance(step, (list, tuple)) else [int(step)]
    return nat.host().adamw([_group(params, grads, ms, vs, steps, bits, lr, betas, eps, weight_decay)], bits,
                            max_grad_norm)


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               max_grad_norm=None):
    """One step of AdamW, in place, over lists of contiguous tensors: parameters
    and gradients fp32 / bf16 / fp16, moments fp32.

    ``step`` counts the updates, this one included, from 1: one number, or one
    for every tensor.  ``max_grad_norm`` scales the gradients to a norm (over
    all of them) of at most that; the gradients themselves are left alone.
    Returns that norm as a device scalar, or ``None`` without clipping.
    """
    return _step(params, grads, exp_avgs, exp_avg_sqs, 32, step, lr, betas, eps, weight_decay, max_grad_norm)


@torch.no_grad()
def adamw_step_8bit(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps=1e-8,
                    weight_decay=1e-2, max_grad_norm=None):
    """:func:`adamw_step` with the moments as lists of (codes, scales)
    (:class:`Moment8`).  The step itself uses the moments before they are
    rounded to 8 bits again."""
    return _step(params, grads, exp_avgs, exp_avg_sqs, 8, step, lr, betas, eps, weight_decay, max_grad_norm)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on the kernels above.

    ``state_bits`` 32 or 8 chooses how the moments are held.  ``max_grad_norm``
    scales the gradients of all parameter groups to that norm as part of the
    step; the norm before scaling is kept in ``grad_norm`` (a device scalar).
    A parameter without a gradient is left out of a step and keeps its own step
    count, as in torch.  All parameters are on one device.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 max_grad_norm=None):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {state_bits}")
        if not lr >= 0 or not eps >= 0 or not weight_decay >= 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("AdamW: lr, eps, weight_decay >= 0 and betas in [0, 1) are wanted")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"AdamW: max_grad_norm must be positive or None, got {max_grad_norm}")
        self.state_bits = state_bits
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        """For copies and pickles: torch's has the groups and the state only."""
        return super().__getstate__() | {k: getattr(self, k) for k in ("state_bits", "max_grad_norm", "grad_norm")}

    def _state_of(self, p):
        s = self.state[p]
        if not s:
            s["step"] = 0
            if self.state_bits == 32:
                s["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            else:
                s["exp_avg"], s["exp_avg_scale"] = zero_moment(p, True)
                s["exp_avg_sq"], s["exp_avg_sq_scale"] = zero_moment(p, False)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, states = [], []
        for group in self.param_groups:
            live = [p for p in group["params"] if p.grad is not None]
            if not live:
                continue
            mine = [self._state_of(p) for p in live]
            grads = [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in live]
            if self.state_bits == 32:
                ms, vs = [s["exp_avg"] for s in mine], [s["exp_avg_sq"] for s in mine]
            else:
                ms = [(s["exp_avg"], s["exp_avg_scale"]) for s in mine]
                vs = [(s["exp_avg_sq"], s["exp_avg_sq_scale"]) for s in mine]
            work.append(_group(live, grads, ms, vs, [s["step"] + 1 for s in mine], self.state_bits, group["lr"],
                               group["betas"], group["eps"], group["weight_decay"]))
            states += mine
        if not work:
            return loss
        self.grad_norm = nat.host().adamw(work, self.state_bits, self.max_grad_norm)
        for s in states:
            s["step"] += 1
        return loss

    def _converted(self, saved, p):
        """One parameter's saved state in this optimizer's own form, on its device."""
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else \
                ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
        if not saved:
            return {}
        held = 8 if "exp_avg_scale" in saved else 32
        if held != self.state_bits:
            raise ValueError(f"AdamW: the saved moments are held in {held} bits, this optimizer's in {self.state_bits}")
        if "step" not in saved or any(n not in saved for n in names):
            raise ValueError(f"AdamW: a parameter's saved state must have step, {', '.join(names)}; got {', '.join(saved)}")
        own = {"step": int(saved["step"])}  # torch's is a tensor, on the device in its fused form
        for name in names:
            t = saved[name].detach()
            scale = name.endswith("_scale")
            want = (-(-p.numel() // QUANT_BLOCK),) if scale else p.shape
            dtype = torch.float32 if scale or held == 32 else torch.int8 if name == "exp_avg" else torch.uint8
            if t.shape != want:
                raise ValueError(f"AdamW: {name} of a parameter {tuple(p.shape)} is saved as {tuple(t.shape)}")
            if t.dtype != dtype and not (held == 32 and t.is_floating_point()):
                raise ValueError(f"AdamW: {name} is saved as {t.dtype}, {dtype} is wanted")
            own[name] = t.to(device=p.device, dtype=dtype, copy=True).contiguous()
        return own

    # torch.optim.AdamW's options that change what a step computes, with the value this class computes
    _ONLY = dict(amsgrad=False, maximize=False, differentiable=False, decoupled_weight_decay=True)

    def load_state_dict(self, state_dict):
        """Takes checkpoints of this class and of ``torch.optim.AdamW`` (for
        ``state_bits=32``; moments of any floating type become fp32).  What it
        cannot go on from is a ``ValueError`` and changes nothing: moments held in
        another number of bits, ``amsgrad``, ``maximize``, another optimizer's
        weight decay."""
        groups = state_dict["param_groups"]
        for g in groups:
            if any(name not in g for name in self.defaults):
                raise ValueError(f"AdamW: a checkpoint's groups must have {', '.join(self.defaults)}; got {', '.join(g)}")
            for name, value in self._ONLY.items():
                if g.get(name, value) != value:
                    raise ValueError(f"AdamW: a checkpoint with {name}={g[name]} cannot be continued")
        saved = [i for g in groups for i in g["params"]]
        here = [p for g in self.param_groups for p in g["params"]]
        states = [self._converted(state_dict["state"].get(i, {}), p) for i, p in zip(saved, here)]
        super().load_state_dict(state_dict)  # torch casts an optimizer's state to its parameter's type
        for p, own in zip(here, states):
            self.state.pop(p, None)
            if own:
                self.state[p] = own
        for g in self.param_groups:
            for name in (*self._ONLY, "foreach", "capturable", "fused"):
                g.pop(name, None)
            g["lr"] = float(g["lr"])  # a device tensor in torch's capturable form
