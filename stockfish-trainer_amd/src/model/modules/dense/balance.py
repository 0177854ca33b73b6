"""The balance loss of a router over expert stacks, and how often each expert is
chosen (for routers such as the reference's MoELayerStacks,
src/model/modules/moe_stacks.py).

With p = softmax of a position's logits over the E experts and S its top_k ones,
over the n positions that count:

    counts_e = positions with e in S        f_e = counts_e / (n top_k)
    loss     = E sum_e f_e mean(p_e)

which is 1 for a balanced router and E / top_k at worst.  The counts are whole
numbers without a gradient; the loss's flows through p.  Positions whose mask is
False count nowhere, whatever their logits hold, and so do positions whose
experts are all at -inf.  A NaN in a position that counts makes the loss NaN.
"""

from __future__ import annotations

import torch
from torch import Tensor, autograd

from sft_amd import _native

from . import ops  # noqa: F401  (registers torch.ops.sft.*)
from .rows import dense_rows


class ExpertBalanceFunction(autograd.Function):
    """The operator in programs that are being compiled; eager ones record the binding's node.

    apply(logits [T, E], mask [T] or None, top_k) -> (loss, counts)."""

    @staticmethod
    def forward(ctx, logits, mask, top_k):
        logits = dense_rows(logits)
        loss, counts, kept = torch.ops.sft.balance_fwd(logits, mask, top_k)
        ctx.save_for_backward(logits, mask, counts, kept)
        ctx.top_k = top_k
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @autograd.function.once_differentiable
    def backward(ctx, grad_loss, _):
        logits, mask, counts, kept = ctx.saved_tensors
        return torch.ops.sft.balance_bwd(logits, mask, ctx.top_k, counts, kept, grad_loss.float()), None, None


def expert_balance(logits: Tensor, top_k: int = 1, mask: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(loss, a float32 scalar; counts, int64 [E]) of router logits [..., E] and a bool mask [...] of the
    positions that count (None: all)."""
    if not torch.compiler.is_compiling():
        return _native.dense_binding().balance(logits, top_k, mask)
    if mask is not None and mask.shape != logits.shape[:-1]:
        raise ValueError("mask must be logits' shape without the last")
    mask = None if mask is None else mask.reshape(-1).contiguous()
    return ExpertBalanceFunction.apply(logits.reshape(-1, logits.shape[-1]), mask, top_k)
