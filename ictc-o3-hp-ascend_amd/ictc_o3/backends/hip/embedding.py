"""Rows of a table by token on HIP kernels, and the table's gradient in a fixed order
(``ictc_hip_embedding_*``; the reference's species embedding is a product with one-hot rows,
``mace_ictc/models/pure_cartesian_ictd_fix.py:3008-3011``).

The lookup and the table's gradient are linear and each other's adjoint: their autograd nodes
(``csrc/host_layers.cpp``) call each other from their backward, and every derivative order stays on the kernels.
"""
from __future__ import annotations

import torch

from ictc_o3 import _lib

from .runtime import require_ordinary_autograd


def embedding(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """scale * table[tokens] for int32 or int64 tokens of any shape and a table [rows, width]: [..., width].  Tokens
    outside [0, rows) (padding) give rows of zeros and have no gradient.  The table's gradient is dense and
    bit-identical from run to run."""
    require_ordinary_autograd()
    return _lib.layers().embedding(tokens, table, scale)
