"""Layer norm of rows, alone or with SiLU behind it (``ictc_hip_layer_norm_*``; no counterpart in the
reference, whose radial network has none).  Formulas stand in ``ictc_hip.h``.

Forward, gradients and the gradients of those (training on forces) each run as one kernel; beyond, where the
second ones are recorded, and for cotangents of weight gradients, the gradients' formulas are composed of torch
operations in 64 bits and differentiated, so every order stays available.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from ictc_o3 import _lib

from .norms import _cont, _weights_run
from .runtime import require_gpu_fp32

MAX_WIDTH = 8192
ACTIVATIONS = {None: 0, "silu": 1}


def _workspace(rows: int, width: int, device) -> torch.Tensor:
    floats = int(_lib.lib().ictc_hip_layer_norm_workspace(width, rows))
    if floats < 0:
        _lib.check(-floats, "ictc_hip_layer_norm_workspace")
    return torch.empty(floats, device=device, dtype=torch.float32)


def _forward(spec, x, weight, bias):
    p = _lib.ptr
    y = torch.empty_like(x)
    if x.shape[0] == 0:     # (tensors without elements have no address)
        return y
    _lib.check(_lib.lib().ictc_hip_layer_norm_forward(p(x), p(weight), p(bias), p(y), x.shape[1], *spec, x.shape[0],
                                                      _lib.stream_of(x.device)), "ictc_hip_layer_norm_forward")
    return y


def _outputs(rows, weights, need):
    """Uninitialised gradients of rows and weights, None where not needed; zeros for weights without rows."""
    make = torch.empty_like if rows.shape[0] else torch.zeros_like
    return [make(t) if n else None for t, n in zip(weights, need)]


def _backward(spec, x, weight, bias, dy, need):
    """Gradients to (x, weight, bias), None where not needed."""
    p = _lib.ptr
    dx = torch.empty_like(x) if need[0] else None
    dw, db = _outputs(x, (weight, bias), need[1:])
    if x.shape[0] == 0:
        return dx, dw, db
    ws = _workspace(*x.shape, x.device) if need[1] or need[2] else None
    _lib.check(_lib.lib().ictc_hip_layer_norm_backward(
        p(x), p(weight), p(bias), p(dy), p(dx), p(dw), p(db), p(ws), 0 if ws is None else ws.numel(), x.shape[1], *spec,
        x.shape[0], _lib.stream_of(x.device)), "ictc_hip_layer_norm_backward")
    return dx, dw, db


def _second(spec, x, weight, bias, dy, cx, need):
    """Gradients to (x, weight, bias, dy), None where not needed."""
    p = _lib.ptr
    gx = torch.empty_like(x) if need[0] else None
    gdy = torch.empty_like(dy) if need[3] else None
    gw, gb = _outputs(x, (weight, bias), need[1:3])
    if x.shape[0] == 0:
        return gx, gw, gb, gdy
    ws = _workspace(*x.shape, x.device) if need[1] or need[2] else None
    _lib.check(_lib.lib().ictc_hip_layer_norm_second(
        p(x), p(weight), p(bias), p(dy), p(cx), p(gx), p(gdy), p(gw), p(gb), p(ws), 0 if ws is None else ws.numel(),
        x.shape[1], *spec, x.shape[0], _lib.stream_of(x.device)), "ictc_hip_layer_norm_second")
    return gx, gw, gb, gdy


def gradient_formula(spec, x, weight, bias, dy):
    """(dx, dweight, dbias) of torch operations: what ``ictc_hip_layer_norm_backward`` computes.  In 64 bits, as
    the kernels' sums and projections are; the results are rounded once."""
    activation, eps = spec
    dtype = x.dtype
    x, weight, bias, dy = (None if t is None else t.double() for t in (x, weight, bias, dy))
    xc = x - x.mean(1, keepdim=True)
    rho = (xc.square().mean(1, keepdim=True) + eps).rsqrt()
    xh = xc * rho
    dz = dy
    if activation:
        z = weight * xh if bias is None else weight * xh + bias
        open_ = torch.sigmoid(z)
        dz = dy * open_ * (1.0 + z * torch.sigmoid(-z))
    e = weight * dz
    dx = rho * (e - e.mean(1, keepdim=True) - xh * (e * xh).mean(1, keepdim=True))
    results = dx, (dz * xh).sum(0), None if bias is None else dz.sum(0)
    return tuple(None if t is None else t.to(dtype) for t in results)


class _Gradient(torch.autograd.Function):
    """The gradients as a function of (x, weight, bias, dy)."""

    @staticmethod
    def forward(ctx, spec, need, *inputs):
        ctx.set_materialize_grads(False)
        ctx.spec = spec
        ctx.save_for_backward(*inputs)
        return _backward(spec, *inputs, need)

    @staticmethod
    def backward(ctx, *cots):
        inputs = ctx.saved_tensors
        x, weight, bias, dy = inputs
        need = list(ctx.needs_input_grad[2:])
        if not _weights_run(weight, bias, need[1:3], x):
            need[1] = need[2] = False
        if not any(need) or all(c is None for c in cots):
            return (None,) * 6
        graph = torch.is_grad_enabled()
        if graph or cots[1] is not None or cots[2] is not None:
            with torch.enable_grad():
                own = [None if t is None else t.view_as(t) if t.requires_grad else t for t in inputs]
                heads = [(o, c) for o, c in zip(gradient_formula(ctx.spec, *own), cots)
                         if o is not None and c is not None and o.requires_grad]
                leaves = [t for t, n in zip(own, need) if n]
                grads = [None] * len(leaves)
                if heads:
                    grads = torch.autograd.grad([o for o, _ in heads], leaves, [c for _, c in heads],
                                                create_graph=graph, allow_unused=True)
            grads = iter(grads)
            return (None, None, *[next(grads) if n else None for n in need])
        if not ctx.spec[0]:          # without an activation the bias is in none of the gradients
            need[2] = False
        return (None, None, *_second(ctx.spec, *inputs, cots[0].contiguous(), need))


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, spec, x, weight, bias):
        ctx.spec = spec
        ctx.save_for_backward(x, weight, bias)
        return _forward(spec, x, weight, bias)

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        need = list(ctx.needs_input_grad[1:])
        if not _weights_run(weight, bias, need[1:], x):
            need[1] = need[2] = False
        if not any(need):
            return (None,) * 4
        dy = dy.contiguous()
        if torch.is_grad_enabled():       # recorded (a function of its own costs 15 us a call)
            return (None, *_Gradient.apply(ctx.spec, tuple(need), x, weight, bias, dy))
        return (None, *_backward(ctx.spec, x, weight, bias, dy, need))


def layer_norm(features: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               activation: Optional[str] = None) -> torch.Tensor:
    """Norm over the last axis (mean and variance of each row), times a weight and plus a bias for each column,
    with SiLU behind it where ``activation`` is "silu", for features [..., W], weight [W] and bias [W] or None."""
    if activation not in ACTIVATIONS:
        raise ValueError('activation must be None or "silu"')
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not eps > 0.0 or not math.isfinite(eps):
        raise ValueError("eps must be a positive number")
    if features.dim() < 1 or not 1 <= features.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"features must have between 1 and {MAX_WIDTH} columns")
    width = features.shape[-1]
    if weight.shape != (width,) or (bias is not None and bias.shape != (width,)):
        raise ValueError(f"weight and bias must have shape [{width}]")
    require_gpu_fp32(*[t for t in (features, weight, bias) if t is not None])
    y = _LayerNorm.apply((ACTIVATIONS[activation], float(eps)), features.reshape(-1, width).contiguous(),
                         weight.contiguous(), _cont(bias))
    return y.view(features.shape)
