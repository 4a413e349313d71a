"""Rotary positions for the query and key heads of an attention layer, with autograd.

``rotary_frequencies`` makes the plan a model keeps (one per head size and length), ``axs_rotary_unified`` turns q and k in
one kernel launch.  (No counterpart in the reference, whose models learn absolute positions.)
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from .. import ops


@dataclass(frozen=True)
class RotaryFrequencies:
    """The frequencies of ``rotated // 2`` pairs on one device: ``turns`` holds, for each pair, the fraction of a full turn it
    makes per position as a 64-bit fixed-point number (int64 bits), ``gain`` the factor on cos and sin."""
    turns: torch.Tensor
    gain: float

    @property
    def rotated(self) -> int:
        return 2 * self.turns.numel()

    def to(self, device) -> "RotaryFrequencies":
        return RotaryFrequencies(self.turns.to(device), self.gain)


def rotary_frequencies(rotated: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0, gain: float | None = None,
                       device="cuda") -> RotaryFrequencies:
    """Pair ``i`` of ``rotated // 2`` turns by ``base ** (-2 i / rotated)`` radians per position.  ``scaling`` stretches the
    positions a model was trained on by ``factor``:

    * ``"none"``
    * ``"linear"``: every frequency divided by ``factor``
    * ``"ntk"``: ``base`` raised to ``base * factor ** (rotated / (rotated - 2))``, so that the slowest pair is slowed by ``factor``
      and the fastest not at all
    * ``"yarn"``: pairs that make more than ``fast_turns`` turns over ``original_length`` positions keep their frequency, those
      that make fewer than ``slow_turns`` are divided by ``factor``, linear in the pair's number in between (the numbers of the two
      borders rounded outwards to whole pairs); cos and sin are multiplied by ``0.1 ln(factor) + 1``

    ``gain`` replaces the factor on cos and sin.  Computed in 64 bits on the host."""
    if rotated < 0 or rotated % 2:
        raise ValueError(f"rotated must be an even number of values, got {rotated}")
    if not (base > 0 and math.isfinite(base)) or not (factor > 0 and math.isfinite(factor)):
        raise ValueError("base and factor must be positive")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"Unknown scaling: {scaling}")
    if scaling == "ntk" and rotated > 2:
        base = base * factor ** (rotated / (rotated - 2))
    freq = [base ** (-2.0 * i / rotated) for i in range(rotated // 2)]
    own_gain = 1.0
    if scaling == "linear":
        freq = [w / factor for w in freq]
    elif scaling == "yarn" and rotated:
        if not (original_length > 0 and fast_turns > slow_turns > 0 and base > 1):
            raise ValueError("yarn needs original_length > 0, fast_turns > slow_turns > 0 and base > 1")

        def pair_with(turns: float) -> float:
            return rotated * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(pair_with(fast_turns)), 0)
        high = min(math.ceil(pair_with(slow_turns)), rotated // 2 - 1)
        slowed = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(rotated // 2)]
        freq = [w * (1 - s) + w / factor * s for w, s in zip(freq, slowed)]
        own_gain = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    fixed = [round(w / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for w in freq]
    turns = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in fixed], dtype=torch.int64, device=device)
    return RotaryFrequencies(turns, float(own_gain if gain is None else gain))


class _Rotary(torch.autograd.Function):
    """Forward: rotate; backward: the transposed rotation (angles negated, same factor) of the gradients."""

    @staticmethod
    def forward(ctx, q, k, positions, turns, gain, interleaved):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, turns)
        ctx.gain, ctx.interleaved = gain, interleaved
        return ops.rotary(q, k, positions, turns, gain, interleaved, False, who="axs_rotary_unified")

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, turns = ctx.saved_tensors
        if dq is None and dk is None:
            return None, None, None, None, None, None
        dq, dk = ops.rotary(dq, dk, positions, turns, ctx.gain, ctx.interleaved, True, who="axs_rotary_unified")
        return dq, dk, None, None, None, None


def axs_rotary_unified(q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor, frequencies: RotaryFrequencies,
                       layout: str = "half") -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Rotate ``q`` (batch, query heads, tokens, size) and ``k`` (batch, key heads, tokens, size), either of which may be None;
    fp32 or bf16, any strides with a unit innermost one (other tensors are copied).  ``positions``: int32 or int64, (tokens,) or
    (batch, tokens), any sign.  The first ``frequencies.rotated`` values of every head are rotated, the others copied; ``layout``
    "half" pairs value i with value i + rotated / 2, "interleaved" value 2 i with 2 i + 1.  Returns new tensors; the arithmetic is
    fp32, rounded once at the end."""
    if layout not in ("half", "interleaved"):
        raise ValueError(f"Unknown layout: {layout}")
    if not isinstance(frequencies, RotaryFrequencies):
        raise TypeError("frequencies must come from rotary_frequencies")
    return _Rotary.apply(q, k, positions, frequencies.turns, frequencies.gain, layout == "interleaved")
