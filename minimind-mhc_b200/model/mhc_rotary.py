"""Rotary positions of queries and keys, with their gradient, in one launch.

    rotary = Rotary(96, theta=1e6)
    q, k = rotate(rotary, q, k)                  # (B, L, heads, D): positions 0 .. L - 1 in every row
    q, k = rotate(rotary, q, k, positions)       # any positions, packed rows (T, heads, D) among them

computes what the reference's ``precompute_freqs_cis`` and ``apply_rotary_pos_emb`` compute
(``model/model_minimind.py:132-159``), without tables of cosines: an angle is formed where it is used, from a frequency
in 64-bit fixed point, exactly at any distance.  CUDA tensors only.  The checks, the allocations and the autograd node
are in ``csrc/host/mhc_torch.cpp``.
"""

from __future__ import annotations

import math

import torch

from . import _native as nat

# 2^192 / (2 pi): a frequency's turns need the bits behind a double's last
_TURNS = (159154943091895335768883763372514362034459645740456448747667344058896797634226535090113802766253085956072842726757958
          << 192) // 10 ** 117


def _turns_of(f: float) -> int:
    """round(f / (2 pi) * 2^64) modulo 2^64."""
    n, d = f.as_integer_ratio()
    shift = 127 + d.bit_length()  # d is a power of two
    return ((n * _TURNS + (1 << (shift - 1))) >> shift) & 0xFFFFFFFFFFFFFFFF


class Rotary:
    """The frequencies of a rotation by position.

    ``dim`` (even): how many elements at the front of a head are rotated, element i with i + dim / 2 or, ``interleaved``,
    2 i with 2 i + 1.  Pair i turns by ``theta ** (-2 i / dim)`` radians a position.  ``factor`` above 1 stretches the
    positions for longer contexts: by itself all frequencies are divided by it; with ``original_length``, the trained
    length, only the slow ones: those that turn less than ``slow`` times within it are divided, those that turn more than
    ``fast`` times left, with a ramp over the pairs between.  Cosines and sines are multiplied by ``gain``: with
    ``original_length`` and a factor above 1 it is 0.1 log(factor) + 1 if it is not given, else 1.  It belongs to the
    weights like the frequencies do: a model whose scaled positions leave cosines and sines as they are (an attention
    factor of 1) needs ``gain=1.0``.  ``inv_freq`` sets the dim / 2 frequencies (radians a position) in place of all that.

    The frequencies lie on ``device`` (the current CUDA device) and are copied to another device at the first call
    there, which a CUDA graph cannot capture."""

    def __init__(self, dim: int, theta: float = 10000.0, *, interleaved: bool = False, factor: float = 1.0,
                 original_length: int | None = None, fast: float = 32.0, slow: float = 1.0, gain: float | None = None,
                 inv_freq=None, device=None):
        if dim < 2 or dim % 2:
            raise ValueError(f"Rotary: dim must be even and positive, got {dim}")
        half = dim // 2
        if inv_freq is None:
            if not (theta > 0 and math.isfinite(theta) and theta != 1.0):
                raise ValueError(f"Rotary: theta must be positive, finite and not 1, got {theta}")
            if not (factor >= 1 and math.isfinite(factor)):
                raise ValueError(f"Rotary: factor must be at least 1 and finite, got {factor}")
            inv = [theta ** (-2 * i / dim) for i in range(half)]
            if original_length is None:
                inv = [f / factor for f in inv]
            elif factor != 1:
                if original_length < 1 or not (fast > 0 and slow > 0):
                    raise ValueError(f"Rotary: original_length {original_length}, fast {fast} and slow {slow} must be positive")

                def pair_of(turns):  # the pair that turns so often within the trained length
                    return dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

                lo, hi = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), half - 1)
                ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(half)]
                inv = [f * (1 - r + r / factor) for f, r in zip(inv, ramp)]
                if gain is None:
                    gain = 0.1 * math.log(factor) + 1.0
        else:
            inv = [float(f) for f in (inv_freq.detach().double().cpu().tolist() if torch.is_tensor(inv_freq) else inv_freq)]
            if len(inv) != half or not all(math.isfinite(f) for f in inv):
                raise ValueError(f"Rotary: {half} finite frequencies are wanted, got {len(inv)}")
        self.dim, self.interleaved, self.gain = dim, bool(interleaved), 1.0 if gain is None else float(gain)
        if not math.isfinite(self.gain):
            raise ValueError(f"Rotary: gain must be finite, got {gain}")
        turns = [_turns_of(f) for f in inv]
        with torch.inference_mode(False):  # a later training step keeps them for its backward pass
            self.inv_freq = torch.tensor(inv, dtype=torch.float64, device="cpu")
            self._host = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device="cpu")
        self._on = {}
        if device is not None or torch.cuda.is_available():
            self.turns(torch.device("cuda" if device is None else device))

    def turns(self, device) -> torch.Tensor:
        """The frequencies as 2^-64ths of a turn (int64), on ``device``."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        got = self._on.get(device)
        if got is None:
            with torch.inference_mode(False):
                got = self._on[device] = self._host.to(device)
        return got


def rotate(rotary: Rotary, q: torch.Tensor, k: torch.Tensor,
           positions: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotates every head of q and k by its token's position.

    q (T, H, D) and k (T, Hk, D), or (B, L, H, D) and (B, L, Hk, D); fp32, bf16 or fp16, both alike; D up to 256 and
    at least ``rotary.dim``, elements behind it are copied; any strides.  ``positions`` (int32 or int64, on the device):
    one for every token, (T,) or (B, L), or (L,) for every row alike; without it a token's index in its row.  Computed in
    fp32 and rounded once.  New contiguous tensors are returned; the gradients of q and k are the opposite rotation.
    Second and forward-mode derivatives are refused, as are tracers.
    """
    return nat.host().rotate(q, k, positions, rotary.turns(q.device) if q.is_cuda else rotary._host, rotary.interleaved,
                             rotary.gain)
