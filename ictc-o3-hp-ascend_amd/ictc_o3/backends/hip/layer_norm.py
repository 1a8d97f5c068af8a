"""Layer norm of rows, alone or with SiLU behind it (``ictc_hip_layer_norm_*``; no counterpart in the
reference, whose radial network has none).  Formulas stand in ``ictc_hip.h``.

Forward, gradients and the gradients of those (training on forces) each run as one kernel, called from autograd
nodes in ``csrc/host_layers.cpp``; beyond, where the second ones are recorded, and for cotangents of weight
gradients, the gradients' formulas are composed of torch operations in 64 bits and differentiated, so every order
stays available.
"""
from __future__ import annotations

from typing import Optional

import torch

from ictc_o3 import _lib

from .runtime import require_ordinary_autograd

ACTIVATIONS = {None: 0, "silu": 1}


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
        dz = dy * torch.sigmoid(z) * (1.0 + z * torch.sigmoid(-z))
    e = weight * dz
    dx = rho * (e - e.mean(1, keepdim=True) - xh * (e * xh).mean(1, keepdim=True))
    results = dx, (dz * xh).sum(0), None if bias is None else dz.sum(0)
    return tuple(None if t is None else t.to(dtype) for t in results)


def composed_gradients(spec, inputs, need, cots):
    """Gradients of <cots, gradient_formula(inputs)> to the inputs that need them (None for the others), recorded
    where grad mode is on."""
    graph = torch.is_grad_enabled()
    with torch.enable_grad():
        own = [None if t is None else t.view_as(t) if t.requires_grad else t for t in inputs]
        heads = [(o, c) for o, c in zip(gradient_formula(spec, *own), cots)
                 if o is not None and c is not None and o.requires_grad]
        leaves = [t for t, n in zip(own, need) if n]
        grads = [None] * len(leaves)
        if heads and leaves:
            grads = torch.autograd.grad([o for o, _ in heads], leaves, [c for _, c in heads], create_graph=graph,
                                        allow_unused=True)
    grads = iter(grads)
    return tuple(next(grads) if n else None for n in need)


def layer_norm(features: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               activation: Optional[str] = None) -> torch.Tensor:
    """Norm over the last axis (mean and variance of each row), times a weight and plus a bias for each column,
    with SiLU behind it where ``activation`` is "silu", for features [..., W], weight [W] and bias [W] or None."""
    if activation not in ACTIVATIONS:
        raise ValueError('activation must be None or "silu"')
    require_ordinary_autograd()
    return _lib.layers().layer_norm(features, weight, bias, ACTIVATIONS[activation], eps)
