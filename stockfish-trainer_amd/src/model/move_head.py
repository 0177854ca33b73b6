"""A head that predicts moves, on the dense operators: what a network trained on a
stronger one's move choices puts behind the feature transformer.

    x       l0 of transform_inputs, [B, L1]
    router  g = softmax(x Wr^T + br) over the experts
    experts e = crelu(x We^T + be), all experts' layers in one product; h = sum_k g_k e_k
    blocks  h = h + gelu(h Wb^T + bb), as often as asked
    moves   logits = h Wm^T + bm over 64 x 64 from- and to-squares

(The reference's MoELayerStacks, src/model/modules/moe_stacks.py, likewise computes
all experts and mixes them by the router.)  The loss is the mean divergence from
the teacher's top moves plus `balance_weight` times the router's balance loss.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

from .modules.dense import distill_loss, expert_balance, fused_linear

MOVES = 64 * 64


class MoveHead(nn.Module):
    def __init__(self, L1: int, width: int = 128, experts: int = 8, blocks: int = 2, moves: int = MOVES, top_k: int = 1,
                 balance_weight: float = 0.01, device=None, dtype=None):
        super().__init__()
        made = {"device": device, "dtype": dtype}
        self.experts, self.width, self.top_k, self.balance_weight = experts, width, top_k, balance_weight
        self.router = nn.Linear(L1, experts, **made)
        self.expert = nn.Linear(L1, experts * width, **made)
        self.blocks = nn.ModuleList(nn.Linear(width, width, **made) for _ in range(blocks))
        self.moves = nn.Linear(width, moves, **made)

    def forward(self, x: Tensor, legal: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """(move logits [B, moves], -inf where a bool `legal` is False; router logits [B, experts])."""
        routes = fused_linear(x, self.router.weight, self.router.bias)
        gate = torch.softmax(routes.float(), dim=1).to(x.dtype)
        each = fused_linear(x, self.expert.weight, self.expert.bias, activation="crelu")
        h = (each.view(-1, self.experts, self.width) * gate.unsqueeze(2)).sum(1)
        for block in self.blocks:
            h = fused_linear(h, block.weight, block.bias, h, "gelu")
        logits = fused_linear(h, self.moves.weight, self.moves.bias)
        return (logits if legal is None else logits.masked_fill(~legal, float("-inf"))), routes

    def loss(self, x: Tensor, teacher_logits: Tensor, teacher_moves: Tensor, legal: Tensor | None = None,
             temperature: float = 1.0) -> tuple[Tensor, Tensor]:
        """(loss, counts): the training loss of a batch, and how often each expert was chosen.  Positions without
        a teacher move (all of teacher_moves outside the moves) are left out of both of its parts."""
        logits, routes = self(x, legal)
        taught = ((teacher_moves >= 0) & (teacher_moves < logits.shape[1])).any(1)
        each = distill_loss(logits, teacher_logits, teacher_moves, temperature)
        balance, counts = expert_balance(routes, self.top_k, taught)
        return each.sum() / taught.sum().clamp(min=1) + self.balance_weight * balance, counts
