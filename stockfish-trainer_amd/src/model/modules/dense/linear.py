"""Linear layers with their bias, activation and residual in the product's
epilogue: y = residual + act(x w^T + bias) as one kernel (the dense layers
behind the feature transformer, reference src/model/modules/layer_stacks.py,
stacked_linear.py and moe_stacks.py, run on torch's products).

fused_linear(x, weight, bias, residual, activation) takes float32, float16 or
bfloat16 CUDA tensors of one type, sums in 32 bits and rounds once.  x and
residual may have any leading dimensions; their rows, weight's and an incoming
gradient's are read in place where the last dimension is dense (slices of wider
rows are), and copied otherwise.  Under autograd it is differentiable in all
four tensors; the backward keeps act' of every output (16-bit fixed point
beside 16-bit layers), not the pre-activations, and does not vary from run to
run.  Derivatives at the kinks are those of torch.clamp.
"""

from __future__ import annotations

import torch
from torch import Tensor, autograd

from sft_amd import _native

from . import ops  # noqa: F401  (registers torch.ops.sft.*)
from .rows import dense_rows

ACTIVATIONS = {
    "none": _native.SFT_ACT_NONE,
    "relu": _native.SFT_ACT_RELU,
    "crelu": _native.SFT_ACT_CRELU,
    "screlu": _native.SFT_ACT_SCRELU,
    "silu": _native.SFT_ACT_SILU,
    "gelu": _native.SFT_ACT_GELU,
}


class FusedLinearFunction(autograd.Function):
    """The operator in programs that are being compiled; eager ones record the binding's node.

    apply(x [M, K], weight [N, K], bias [N] or None, residual [M, N] or None, act code) -> y [M, N]."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x, weight, residual = dense_rows(x), dense_rows(weight), dense_rows(residual)
        bias = None if bias is None else bias.contiguous()
        y, deriv = torch.ops.sft.linear_fwd(x, weight, bias, residual, act, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, deriv)
        ctx.act = act
        return y

    @staticmethod
    @autograd.function.once_differentiable
    def backward(ctx, grad_y):
        x, weight, deriv = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = torch.ops.sft.linear_bwd(dense_rows(grad_y), deriv, x, weight, ctx.act, *need[:3])
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None,
                grad_y if need[3] else None, None)


def fused_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, residual: Tensor | None = None,
                 activation: str = "none") -> Tensor:
    """residual + act(x @ weight.T + bias); x [..., K], weight [N, K], bias [N], residual [..., N]."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if not torch.compiler.is_compiling():
        return _native.dense_binding().linear(x, weight, bias, residual, act)
    N, K = weight.shape
    lead = x.shape[:-1]
    if x.shape[-1] != K or (residual is not None and residual.shape != (*lead, N)):
        raise ValueError("x must be [..., K] and residual [..., N]")
    x = x.reshape(-1, K)
    residual = None if residual is None else residual.reshape(-1, N)
    return FusedLinearFunction.apply(x, weight, bias, residual, act).view(*lead, N)
