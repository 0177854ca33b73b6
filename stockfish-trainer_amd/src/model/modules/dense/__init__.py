from .linear import FusedLinearFunction, fused_linear

__all__ = ["FusedLinearFunction", "fused_linear"]
