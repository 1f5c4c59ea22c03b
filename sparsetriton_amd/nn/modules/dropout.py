"""Dropout on sparse features (no counterpart in the reference)."""

from typing import Optional

from torch import nn

from sparsetriton_amd.nn.functional.dropout import sparse_dropout
from sparsetriton_amd.tensor import SparseTensor

__all__ = ["SparseDropout"]


class SparseDropout(nn.Module):
    """``sparse_dropout`` in training, the identity in evaluation; ``residual`` is added in the same pass.

    The mask's numbers come from torch's generator of the device, fresh for each call.
    """

    def __init__(self, p: float = 0.5) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout needs a probability (got p = {p})")
        self.p = p

    def extra_repr(self) -> str:
        return f"p={self.p}"

    def forward(self, input, residual: Optional[SparseTensor] = None):
        return sparse_dropout(input, self.p, training=self.training, residual=residual)
