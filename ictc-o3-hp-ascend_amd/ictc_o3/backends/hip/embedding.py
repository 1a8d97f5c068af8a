"""Rows of a table by token on HIP kernels, and the table's gradient in a fixed order
(``ictc_hip_embedding_*``; the reference's species embedding is a product with one-hot rows,
``mace_ictc/models/pure_cartesian_ictd_fix.py:3008-3011``).

The lookup and the table's gradient are linear and each other's adjoint: ``_Lookup`` and ``_TableGrad`` call each
other from their backward, and every derivative order stays on the kernels.
"""
from __future__ import annotations

import math

import torch

from ictc_o3 import _lib

from .runtime import require_gpu_fp32


def _lookup(table, tokens, scale):
    out = torch.empty(tokens.shape[0], table.shape[1], device=table.device, dtype=torch.float32)
    if tokens.shape[0]:     # (tensors without elements have no address)
        _lib.check(_lib.lib().ictc_hip_embedding_forward(
            tokens.data_ptr(), tokens.element_size(), table.data_ptr(), out.data_ptr(), *table.shape, scale,
            tokens.shape[0], _lib.stream_of(table.device)), "ictc_hip_embedding_forward")
    return out


def _table_grad(grad, tokens, rows, scale):
    count, width = grad.shape
    if count == 0:
        return torch.zeros(rows, width, device=grad.device, dtype=torch.float32)
    lib = _lib.lib()
    units = int(lib.ictc_hip_embedding_workspace(rows, width, count))
    if units < 0:
        _lib.check(-units, "ictc_hip_embedding_workspace")
    out = torch.empty(rows, width, device=grad.device, dtype=torch.float32)
    ws = torch.empty(units, device=grad.device, dtype=torch.int32)
    _lib.check(lib.ictc_hip_embedding_table_grad(
        tokens.data_ptr(), tokens.element_size(), grad.data_ptr(), out.data_ptr(), rows, width, scale, count,
        ws.data_ptr(), units, _lib.stream_of(grad.device)), "ictc_hip_embedding_table_grad")
    return out


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale):
        ctx.rows, ctx.scale = table.shape[0], scale
        ctx.save_for_backward(tokens)
        return _lookup(table, tokens, scale)

    @staticmethod
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        grad = grad.contiguous()
        if not torch.is_grad_enabled():
            return _table_grad(grad, tokens, ctx.rows, ctx.scale), None, None
        return _TableGrad.apply(grad, tokens, ctx.rows, ctx.scale), None, None


class _TableGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, tokens, rows, scale):
        ctx.scale = scale
        ctx.save_for_backward(tokens)
        return _table_grad(grad, tokens, rows, scale)

    @staticmethod
    def backward(ctx, cot):
        tokens, = ctx.saved_tensors
        return _Lookup.apply(cot.contiguous(), tokens, ctx.scale), None, None, None


def embedding(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """scale * table[tokens] for int32 or int64 tokens of any shape and a table [rows, width]: [..., width].  Tokens
    outside [0, rows) (padding) give rows of zeros and have no gradient.  The table's gradient is dense and
    bit-identical from run to run."""
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError("the table must have shape [rows, width]")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("tokens must be int32 or int64")
    if isinstance(scale, bool) or not isinstance(scale, (int, float)) or not math.isfinite(scale):
        raise ValueError("scale must be a finite number")
    require_gpu_fp32(table)
    if tokens.device != table.device:
        raise ValueError("All operands must be on the same GPU")
    out = _Lookup.apply(table.contiguous(), tokens.reshape(-1).contiguous(), float(scale))
    return out.view(*tokens.shape, table.shape[1])
