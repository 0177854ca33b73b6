"""The dense head's library calls as torch custom operators, as the feature
transformer's are: opaque to Dynamo and Inductor, with known output shapes.
Every op allocates and returns its outputs and mutates nothing."""

from __future__ import annotations

import torch
from torch import Tensor

from sft_amd import _native


def _deriv_dtype(dtype: torch.dtype) -> torch.dtype:
    return torch.float32 if dtype == torch.float32 else torch.int16


# ---- FusedLinearFunction ----
@torch.library.custom_op("sft::linear_fwd", mutates_args=(), device_types="cuda")
def linear_fwd(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, act: int,
               keep: bool) -> tuple[Tensor, Tensor]:
    """(y, act' of every output for the backward; empty where it is not kept or is 1)."""
    M, N = x.shape[0], weight.shape[0]
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    kept = keep and act != _native.SFT_ACT_NONE
    deriv = torch.empty((M, N) if kept else (0,), dtype=_deriv_dtype(x.dtype), device=x.device)
    _native.linear_fwd(x, weight, bias, residual, y, deriv if kept else None, act)
    return y, deriv


@linear_fwd.register_fake
def _(x, weight, bias, residual, act, keep):
    shape = (x.shape[0], weight.shape[0])
    kept = keep and act != _native.SFT_ACT_NONE
    return x.new_empty(shape), x.new_empty(shape if kept else (0,), dtype=_deriv_dtype(x.dtype))


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
