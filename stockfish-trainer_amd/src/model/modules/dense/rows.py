"""Row layouts the dense head's kernels read in place."""

from __future__ import annotations

from torch import Tensor


def dense_rows(t: Tensor | None) -> Tensor | None:
    """A 2-D t, or a copy of it where its rows are not dense, overlap or lie in descending order."""
    if t is None or t.is_contiguous():
        return t
    rows, cols = t.shape
    if (cols == 1 or t.stride(1) == 1) and (rows == 1 or t.stride(0) >= cols):
        return t
    return t.contiguous()
