"""Distillation of a move (or any class) distribution from a teacher's top logits.

A teacher's whole distribution is rarely kept: a record holds its k best classes
and their logits.  With p = softmax(student / T) over all V classes and q =
softmax(teacher / T) over the row's filled slots,

    loss      = T^2 sum_j q_j (log q_j - log p_{i_j})          (per row)
    d loss/ds = T (p_v - q of class v)

Slots with an index outside [0, V) are empty, and a class may be named twice.  Classes
the student excludes hold -inf: they get no probability and no gradient, unless the
teacher names one with q > 0 (the loss is then infinite).  A row without a
filled slot, or whose classes are all excluded, has loss 0 and no gradient; a NaN
in any other row makes its loss and gradient NaN.

distill_loss is differentiable in the student's logits and reads them once more
in its backward; distill_loss_and_grad makes both in one pass, for loops that
know each row's weight in the total loss beforehand: logits.backward(grad).
"""

from __future__ import annotations

import torch
from torch import Tensor, autograd

from sft_amd import _native

from . import ops  # noqa: F401  (registers torch.ops.sft.*)
from .rows import dense_rows

class DistillFunction(autograd.Function):
    """The operator in programs that are being compiled; eager ones record the binding's node.

    apply(student [R, V], teacher [R, k], indices [R, k], temperature) -> loss [R]."""

    @staticmethod
    def forward(ctx, student, teacher, indices, temperature):
        ctx.save_for_backward(student, teacher, indices)
        ctx.temperature = temperature
        return torch.ops.sft.distill_loss(student, teacher, indices, temperature)

    @staticmethod
    @autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        student, teacher, indices = ctx.saved_tensors
        return torch.ops.sft.distill_grad(student, teacher, indices, ctx.temperature,
                                          grad_loss.float().contiguous()), None, None, None


def distill_loss(student_logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor,
                 temperature: float = 1.0) -> Tensor:
    """Per-row loss (float32 [R]) of student logits [R, V] against a teacher's k top logits [R, k] of the
    classes in teacher_indices (int32 or int64; outside [0, V): an empty slot)."""
    if not torch.compiler.is_compiling():
        return _native.dense_binding().distill_loss(student_logits, teacher_logits, teacher_indices, temperature)
    return DistillFunction.apply(dense_rows(student_logits), teacher_logits.detach().contiguous(),
                                 teacher_indices.contiguous(), float(temperature))


def distill_loss_and_grad(student_logits: Tensor, teacher_logits: Tensor, teacher_indices: Tensor,
                          row_weight: Tensor | None = None, temperature: float = 1.0) -> tuple[Tensor, Tensor]:
    """(loss [R], row_weight * d loss / d student [R, V]) in one pass over the logits, outside autograd;
    row_weight float32 [R] (None: 1) is each row's share of the total loss, loss scaling included."""
    if not torch.compiler.is_compiling():
        return _native.dense_binding().distill_loss_and_grad(student_logits, teacher_logits, teacher_indices,
                                                             row_weight, temperature)
    row_weight = None if row_weight is None else row_weight.detach().contiguous()
    return torch.ops.sft.distill_loss_and_grad(dense_rows(student_logits.detach()),
                                               teacher_logits.detach().contiguous(), teacher_indices.contiguous(),
                                               float(temperature), row_weight)
