"""Distillation of a move (or any class) distribution from a teacher's top logits.

A teacher's whole distribution is rarely kept: a record holds its k best classes
and their logits.  With p = softmax(student / T) over all V classes and q =
softmax(teacher / T) over the row's filled slots,

    loss      = T^2 sum_j q_j (log q_j - log p_{i_j})          (per row)
    d loss/ds = T (p_v - q of class v)

Slots with an index outside [0, V) are empty, and a class may be named twice.  Classes
the student excludes hold -inf: they get no probability and no gradient, unless the
teacher names one with q > 0 (the loss is then infinite).  A row without a
filled slot, or whose classes are all excluded, has loss 0 and no gradient.

distill_loss is differentiable in the student's logits and reads them once more
in its backward; distill_loss_and_grad makes both in one pass, for loops that
know each row's weight in the total loss beforehand: logits.backward(grad).
"""

from __future__ import annotations

import math

import torch
from torch import Tensor, autograd

from sft_amd import _native

from .ops import calls
from .rows import dense_rows

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class DistillFunction(autograd.Function):
    """apply(student [R, V], teacher [R, k], indices [R, k], temperature) -> loss [R]."""

    @staticmethod
    def forward(ctx, student, teacher, indices, temperature):
        ctx.save_for_backward(student, teacher, indices)
        ctx.temperature = temperature
        return calls().distill_loss(student, teacher, indices, temperature)

    @staticmethod
    @autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        student, teacher, indices = ctx.saved_tensors
        return calls().distill_grad(student, teacher, indices, ctx.temperature,
                                          grad_loss.float().contiguous()), None, None, None


def _checked(student, teacher_logits, teacher_indices, temperature):
    assert student.is_cuda and student.dim() == 2 and student.shape[1] >= 1
    assert student.dtype in _FLOATS and teacher_logits.dtype in _FLOATS
    assert teacher_indices.dtype in (torch.int32, torch.int64)
    assert teacher_logits.dim() == 2 and teacher_logits.shape == teacher_indices.shape
    assert teacher_logits.shape[0] == student.shape[0]
    assert 1 <= teacher_logits.shape[1] <= _native.SFT_DISTILL_MAX_K
    assert teacher_logits.device == student.device and teacher_indices.device == student.device
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    return dense_rows(student), teacher_logits.detach().contiguous(), teacher_indices.contiguous()


def distill_loss(student_logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor,
                 temperature: float = 1.0) -> Tensor:
    """Per-row loss (float32 [R]) of student logits [R, V] against a teacher's k top logits [R, k] of the
    classes in teacher_indices (int32 or int64; outside [0, V): an empty slot)."""
    student, teacher, indices = _checked(student_logits, teacher_logits, teacher_indices, temperature)
    return DistillFunction.apply(student, teacher, indices, float(temperature))


def distill_loss_and_grad(student_logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor,
                          row_weight: Tensor | None = None, temperature: float = 1.0) -> tuple[Tensor, Tensor]:
    """(loss [R], row_weight * d loss / d student [R, V]) in one pass over the logits, outside autograd;
    row_weight float32 [R] (None: 1) is each row's share of the total loss, loss scaling included."""
    student, teacher, indices = _checked(student_logits, teacher_logits, teacher_indices, temperature)
    if row_weight is not None:
        assert row_weight.shape == (student.shape[0],) and row_weight.dtype == torch.float32
        assert row_weight.device == student.device
        row_weight = row_weight.detach().contiguous()
    return calls().distill_loss_and_grad(student.detach(), teacher, indices, float(temperature), row_weight)
