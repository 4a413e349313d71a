"""Distillation loss of a (quantised) student from the top logits of a full-precision teacher, with its gradient.

A teacher's top ``k`` logits per position are what a training set can store (the reference trains on labels only; no counterpart
there).  ``axs_distillation_unified`` is the loss, ``AXSDistillationLoss`` the form that
``AXSTrainingPipelineUnified.training_step`` takes as its ``loss_fn``.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


class _Distillation(torch.autograd.Function):
    """Forward: one pass over the logits (online softmax), each row's maximum and sum saved; backward: one more pass
    that recomputes the student's probabilities and writes the gradient."""

    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_index, temperature, reduction):
        loss, z, t, index, stats, count = ops.distill_fwd(logits, teacher_logits, teacher_index, temperature, reduction)
        ctx.save_for_backward(z, t, index, stats, count)
        ctx.temperature, ctx.shape, ctx.dtype = temperature, logits.shape, logits.dtype
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        z, t, index, stats, count = ctx.saved_tensors
        grad = ops.distill_bwd(z, t, index, stats, upstream, count, ctx.temperature)
        return grad.reshape(ctx.shape).to(ctx.dtype), None, None, None, None


def axs_distillation_unified(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor, temperature: float = 1.0,
                             reduction: str = "mean") -> torch.Tensor:
    """``temperature ** 2 * KL(teacher || student)`` per position: the teacher's distribution is the softmax of its logits over the
    position's used slots, the student's the softmax of ``logits`` (..., vocabulary) over the whole vocabulary, both at
    ``temperature``.  ``teacher_logits`` (..., k) fp32 or bf16 and ``teacher_index`` (..., k) integers with k from 1 to 1024; a slot whose
    index is outside the vocabulary (-1 by custom) or whose logit is -inf is unused, two slots of one position that name the same
    index add up, and a position without a used slot is left out: loss and gradient 0.  ``reduction``: "none" (one fp32 value per
    position), "sum", or "mean" over the positions that are not left out (0 if there is none).  fp32 results; gradients reach
    ``logits`` only, in their type.  Logits are fp32 or bf16 (others are converted to fp32)."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"Unknown reduction: {reduction}")
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return _Distillation.apply(logits, teacher_logits, teacher_index, temperature, _REDUCTIONS[reduction])


class AXSDistillationLoss:
    """``loss_fn`` for the training pipeline: ``loss_fn(model_output, inputs) -> loss``, the teacher's top logits taken from the batch
    by ``teacher(inputs) -> (teacher_logits, teacher_index)``."""

    def __init__(self, teacher, temperature: float = 1.0, reduction: str = "mean") -> None:
        self.teacher, self.temperature, self.reduction = teacher, temperature, reduction

    def __call__(self, model_output: torch.Tensor, inputs) -> torch.Tensor:
        teacher_logits, teacher_index = self.teacher(inputs)
        return axs_distillation_unified(model_output, teacher_logits, teacher_index, self.temperature, self.reduction)
