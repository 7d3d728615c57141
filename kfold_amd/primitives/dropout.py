"""Dropout with a mask that is never stored, ``hip`` backend.

Counterpart of the reference's dropout of the pair track's updates (primitives/dropout.py:65: the
identity in eval mode), with one mask value per element or shared along a dimension (row- / column-wise
dropout of ``[B, N, N, C]``).
"""

from __future__ import annotations

import torch
from torch import nn

from .. import functional


class Dropout(nn.Module):
    """``(residual or 0) + dropout(x)``.  ``shared_dim``: the dimension one mask value covers.  A call
    takes the mask's ``seed`` (and ``offset``) or, without one, draws a seed from torch's CPU generator
    (``torch.manual_seed`` makes it repeatable).  A call recorded into a HIP graph needs a seed in device
    memory: a drawn one would be the same in every replay."""

    def __init__(self, p: float, shared_dim: int | None = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout: p={p} is no probability")
        self.p = p
        self.shared_dim = shared_dim

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, seed=None, offset: int = 0) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        if seed is None:
            seed = int(torch.randint(0, 2 ** 62, (), device="cpu"))       # whatever torch's default device is
        return functional.dropout(x, self.p, seed, offset, self.shared_dim, residual)
