"""The dense head's library calls as torch custom operators, for programs that are
being compiled: opaque to Dynamo and Inductor, with known output shapes, as the
feature transformer's are.  Every op allocates and returns its outputs and mutates
nothing.  Eager programs take the same calls through the binding module
(sft_amd/_native.py, dense_binding), whose dispatch costs less than a small
call's kernels.
"""

from __future__ import annotations

import torch
from torch import Tensor

from sft_amd import _native


# ---- FusedLinearFunction ----
@torch.library.custom_op("sft::linear_fwd", mutates_args=(), device_types="cuda")
def linear_fwd(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, act: int,
               keep: bool) -> tuple[Tensor, Tensor]:
    """(y, act' of every output for the backward; empty where it is not kept or is 1)."""
    M, N = x.shape[0], weight.shape[0]
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    kept = keep and act != _native.SFT_ACT_NONE
    deriv = torch.empty((M, N) if kept else (0,), dtype=_native.deriv_dtype(x.dtype), device=x.device)
    _native.linear_fwd(x, weight, bias, residual, y, deriv if kept else None, act)
    return y, deriv


@linear_fwd.register_fake
def _(x, weight, bias, residual, act, keep):
    shape = (x.shape[0], weight.shape[0])
    kept = keep and act != _native.SFT_ACT_NONE
    return x.new_empty(shape), x.new_empty(shape if kept else (0,), dtype=_native.deriv_dtype(x.dtype))


@torch.library.custom_op("sft::linear_bwd", mutates_args=(), device_types="cuda")
def linear_bwd(grad_y: Tensor, deriv: Tensor, x: Tensor, weight: Tensor, act: int, need_x: bool, need_weight: bool,
               need_bias: bool) -> tuple[Tensor, Tensor, Tensor]:
    """Grads of x, weight and bias; empty where not needed."""
    (M, K), N = x.shape, weight.shape[0]
    dx, dw, db = (torch.empty(shape if need else (0,), dtype=x.dtype, device=x.device)
                  for need, shape in ((need_x, (M, K)), (need_weight, (N, K)), (need_bias, (N,))))
    _native.linear_bwd(grad_y, None if act == _native.SFT_ACT_NONE else deriv, x, weight, dx if need_x else None,
                       dw if need_weight else None, db if need_bias else None, act)
    return dx, dw, db


@linear_bwd.register_fake
def _(grad_y, deriv, x, weight, act, need_x, need_weight, need_bias):
    (M, K), N = x.shape, weight.shape[0]
    return tuple(x.new_empty(shape if need else (0,))
                 for need, shape in ((need_x, (M, K)), (need_weight, (N, K)), (need_bias, (N,))))


# ---- ExpertBalanceFunction ----
@torch.library.custom_op("sft::balance_fwd", mutates_args=(), device_types="cuda")
def balance_fwd(logits: Tensor, mask: Tensor | None, top_k: int) -> tuple[Tensor, Tensor, Tensor]:
    """(loss, counts [E], number of kept positions)."""
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    counts = torch.empty(logits.shape[1], dtype=torch.int64, device=logits.device)
    kept = torch.empty((), dtype=torch.int64, device=logits.device)
    _native.balance_fwd(logits, mask, top_k, loss, counts, kept)
    return loss, counts, kept


@balance_fwd.register_fake
def _(logits, mask, top_k):
    return (logits.new_empty((), dtype=torch.float32), logits.new_empty((logits.shape[1],), dtype=torch.int64),
            logits.new_empty((), dtype=torch.int64))


@torch.library.custom_op("sft::balance_bwd", mutates_args=(), device_types="cuda")
def balance_bwd(logits: Tensor, mask: Tensor | None, top_k: int, counts: Tensor, kept: Tensor,
                grad_loss: Tensor) -> Tensor:
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _native.balance_bwd(logits, mask, top_k, counts, kept, grad_loss, grad)
    return grad


@balance_bwd.register_fake
def _(logits, mask, top_k, counts, kept, grad_loss):
    return logits.new_empty(logits.shape)


# ---- DistillFunction ----
@torch.library.custom_op("sft::distill_loss", mutates_args=(), device_types="cuda")
def distill_loss(student: Tensor, teacher: Tensor, indices: Tensor, temperature: float) -> Tensor:
    loss = torch.empty(student.shape[0], dtype=torch.float32, device=student.device)
    _native.distill(student, teacher, indices, temperature, None, loss, None)
    return loss


@distill_loss.register_fake
def _(student, teacher, indices, temperature):
    return student.new_empty((student.shape[0],), dtype=torch.float32)


@torch.library.custom_op("sft::distill_grad", mutates_args=(), device_types="cuda")
def distill_grad(student: Tensor, teacher: Tensor, indices: Tensor, temperature: float, row_weight: Tensor) -> Tensor:
    grad = torch.empty(student.shape, dtype=student.dtype, device=student.device)
    _native.distill(student, teacher, indices, temperature, row_weight, None, grad)
    return grad


@distill_grad.register_fake
def _(student, teacher, indices, temperature, row_weight):
    return student.new_empty(student.shape)


@torch.library.custom_op("sft::distill_loss_and_grad", mutates_args=(), device_types="cuda")
def distill_loss_and_grad(student: Tensor, teacher: Tensor, indices: Tensor, temperature: float,
                          row_weight: Tensor | None) -> tuple[Tensor, Tensor]:
    loss = torch.empty(student.shape[0], dtype=torch.float32, device=student.device)
    grad = torch.empty(student.shape, dtype=student.dtype, device=student.device)
    _native.distill(student, teacher, indices, temperature, row_weight, loss, grad)
    return loss, grad


@distill_loss_and_grad.register_fake
def _(student, teacher, indices, temperature, row_weight):
    return student.new_empty((student.shape[0],), dtype=torch.float32), student.new_empty(student.shape)
