from .balance import ExpertBalanceFunction, expert_balance
from .distill import DistillFunction, distill_loss, distill_loss_and_grad
from .linear import FusedLinearFunction, fused_linear

__all__ = [
    "DistillFunction",
    "ExpertBalanceFunction",
    "FusedLinearFunction",
    "distill_loss",
    "distill_loss_and_grad",
    "expert_balance",
    "fused_linear",
]
