"""Attention that never writes its scores to memory, with a backward pass that recomputes the probabilities.

``AXSMultiheadAttentionUnified`` quantises the normalised attention weights and therefore materialises them; with
``quantize_weights=False`` it calls this operator instead.  (The reference has only the materialised form,
``axs/unified/modules_unified.py:229-264``.)
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops


class _Attention(torch.autograd.Function):
    """Forward: one pass over the keys with a running maximum and sum; saved: the operands, the output and two fp32 numbers a
    row.  Backward: probabilities recomputed from them, gradients in fp32 rounded once."""

    @staticmethod
    def forward(ctx, q, k, v, key_lengths, mask, scale, causal, window, want_lse):
        o, stats, lse, q, k, v, low = ops.attention_fwd(q, k, v, key_lengths, mask, scale, causal, window, want_lse, any(ctx.needs_input_grad))
        ctx.save_for_backward(q, k, v, o, low, stats, key_lengths, mask)
        ctx.call = (scale, causal, window)
        if lse is None:
            return o
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, *unused):
        q, k, v, o, low, stats, key_lengths, mask = ctx.saved_tensors
        dq, dk, dv = ops.attention_bwd(d_o, q, k, v, o, low, stats, key_lengths, mask, *ctx.call)
        return dq, dk, dv, None, None, None, None, None, None


def axs_attention_unified(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False, window: int | None = None,
                          key_lengths: torch.Tensor | None = None, mask: torch.Tensor | None = None, scale: float | None = None,
                          return_lse: bool = False):
    """``softmax(scale * q @ k^T + mask) @ v`` for ``q`` (batch, heads, queries, size) and ``k``, ``v`` (batch, key heads, keys, size),
    all fp32 or all bf16, ``size`` up to 128; the query heads are split evenly over the key heads in order.  ``scale`` defaults to
    ``size ** -0.5``.

    * ``causal``: query i stands at key ``i + keys - queries`` and sees no later key; ``window`` (with causal): only the last
      ``window`` keys up to its own.
    * ``key_lengths`` int32 (batch,): keys from there on are hidden, whatever the memory holds.
    * ``mask``: broadcastable to (batch, heads, queries, keys); bool (False hides) or fp32 / bf16 values added to the scaled scores
      (-inf hides; no gradient).  A key that only some queries see must hold finite values.

    A query that sees no key gives zeros and takes no part in the gradients.  Statistics, sums and scores are fp32; with bf16 tensors the
    products run on the tensor cores, for which the probabilities and, in the backward pass, the scores' gradients are rounded to
    bf16.  Returns the output in q's shape and type, with ``return_lse`` also log-sum-exp of each row's scores (fp32, -inf for a row
    without keys, not differentiable)."""
    mask, scale, window = ops.attention_check(q, k, v, key_lengths, mask, scale, causal, window, "axs_attention_unified")
    return _Attention.apply(q, k, v, key_lengths, mask, scale, bool(causal), window, bool(return_lse))
