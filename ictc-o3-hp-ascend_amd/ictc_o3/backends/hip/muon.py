"""Orthogonalised updates of many matrices on ``libictc_hip.so`` (``ictc_hip_orthogonalize``,
``ictc_hip_muon_step``; no counterpart in the reference, whose training loop uses torch's optimizers).  Formulas
stand in ``ictc_hip.h``.

Nothing here reads from the device or copies to it: the tensors' addresses are kernel arguments, and clipping
coefficient and (where it is a tensor) the learning rate stay on the device, so a step can be captured into a
HIP graph.  ``ictc_o3.optim.Muon`` is the optimizer on top.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ictc_o3 import _lib

from .optimizer import _number, _on

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_STEPS = 64
SHORT = 128           # shorter sides that the kernels do in chunks of columns
ADJUST = {"original": 0, "match_rms_adamw": 1}


def _desc(*, steps, coefficients, eps, beta=0.0, nesterov=False, weight_decay=0.0, lr=0.0, adjust="original"):
    if isinstance(steps, bool) or not isinstance(steps, int) or not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"steps must be an integer in [1, {MAX_STEPS}]")
    if len(coefficients) != 3 or not all(isinstance(c, (int, float)) and math.isfinite(c) for c in coefficients):
        raise ValueError("coefficients must be three finite numbers")
    if not _number(eps, "eps") > 0.0:
        raise ValueError("eps must be positive")
    if adjust not in ADJUST:
        raise ValueError(f"adjust must be one of {sorted(ADJUST)}")
    return _lib.MuonDesc(_number(beta, "beta", 1.0), _number(weight_decay, "weight_decay"), float(eps),
                         (ctypes.c_double * 3)(*coefficients), _number(lr, "lr"), bool(nesterov), steps, ADJUST[adjust])


def _workspace(shapes, count: int, device) -> torch.Tensor:
    needed = int(_lib.lib().ictc_hip_muon_workspace(*shapes, count))
    if needed < 0:
        _lib.check(-needed, "ictc_hip_muon_workspace")
    # (torch's allocations begin at multiples of 512 bytes)
    return torch.empty(needed, device=device, dtype=torch.uint8)


_SIDE_STREAMS = {}


def _side_stream(device: torch.device):
    """One default-priority side stream per device, created once, and another one for captures: work that is issued
    elsewhere meanwhile must not end up in a graph."""
    key = device.index, torch.cuda.is_current_stream_capturing()
    stream = _SIDE_STREAMS.get(key)
    if stream is None:
        stream = _SIDE_STREAMS[key] = torch.cuda.Stream(device=device)
    return stream


def _both_kinds(shapes, device, run) -> None:
    """run(places) for the matrices whose shorter side is up to SHORT, which have launches of their own, and for the
    others; where there are both, on two streams side by side (both are bound by the latency of their launches: 12
    matrices of 1 to 1,501 rows and columns 188 us against 257 one after the other)."""
    rows, columns = (memoryview(b).cast("q") for b in shapes[:2])
    kinds = ([], [])
    for k, (r, c) in enumerate(zip(rows, columns)):
        kinds[min(r, c) <= SHORT].append(k)
    if not kinds[0] or not kinds[1]:
        run(None)
        return
    here, side = torch.cuda.current_stream(device), _side_stream(device)
    side.wait_stream(here)
    try:
        with torch.cuda.stream(side):
            run(kinds[1])
        run(kinds[0])
    finally:
        here.wait_stream(side)


def _at(values, places):
    return values if places is None else [values[k] for k in places]


def orthogonalize(matrices, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
    """Each matrix of a list (tensors [..., rows, columns], leading axes counting matrices) scaled to Frobenius norm
    1 and brought near an orthogonal one by ``steps`` Newton-Schulz products, as a list of new tensors.  Without
    gradients.  The coefficients have to keep singular values below 5 (beyond, a result may not be a number)."""
    with torch.no_grad():
        matrices = list(matrices)
        if not matrices:
            return []
        host = _lib.host()
        _, _, *shapes, contiguous = host.matrices(matrices, "matrices")
        if not contiguous:
            matrices = [m.contiguous() for m in matrices]
        desc = _desc(steps=steps, coefficients=coefficients, eps=eps)
        device = matrices[0].device

        def run(places):
            own = _at(matrices, places)
            _, at, *sizes, _ = host.matrices(own, "matrices")
            _, to, *_ = host.matrices(_at(out, places), "matrices")
            ws = _workspace(sizes, len(own), device)
            _lib.check(_lib.lib().ictc_hip_orthogonalize(at, to, *sizes, len(own), ctypes.byref(desc), ws.data_ptr(),
                                                         ws.numel(), _lib.stream_of(device)), "ictc_hip_orthogonalize")

        with _on(device):
            out = host.alike(matrices)
            _both_kinds(shapes, device, run)
        return out


def muon_step(params, grads, momentum, *, lr, beta: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
              steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7, adjust: str = "original", clip=None) -> None:
    """One step of every parameter with a gradient, in place (a None gradient leaves its parameter and momentum as
    they are): a moving average of the gradient, orthogonalised as ``orthogonalize`` does, as the update.  The
    parameters are matrices (or have leading axes that count them).  What is written, parameters and momentum, must
    not overlap each other or a gradient.

    momentum: a list of float32 tensors of the parameters' shapes (zeros before the first step).  lr: a number, or a
    one-element float32 tensor on the device.  adjust: the update's size, "original" for sqrt(max(1, rows / columns))
    or "match_rms_adamw" for 0.2 sqrt(max(rows, columns)), which gives entries of AdamW's usual size.  clip:
    ``gradient_norm``'s result, whose coefficient scales the gradients (not a number: nothing changes)."""
    params, grads, momentum = list(params), list(grads), list(momentum)
    host = _lib.host()
    _, _, _, _, _, contiguous = host.pairs(params, grads, 1)
    if not contiguous:
        grads = [g if g is None else g.contiguous() for g in grads]
    n, device = len(params), params[0].device
    _, _, *shapes, _ = host.matrices(params, "parameters")
    m_device, _, *m_shapes, contiguous = host.matrices(momentum, "momentum")
    if len(momentum) != n or not contiguous or m_device != device.index or m_shapes != shapes:
        raise ValueError("momentum must hold a contiguous tensor of each parameter's shape beside the parameters")
    if clip is not None and (clip.dtype is not torch.float32 or clip.shape != (2,) or clip.device != device
                             or not clip.is_contiguous()):
        raise ValueError("clip must be gradient_norm's result")
    lr_device = None
    if isinstance(lr, torch.Tensor):
        if lr.dtype is not torch.float32 or lr.numel() != 1 or lr.device != device:
            raise ValueError("a learning rate tensor must hold one FP32 value beside the parameters")
        lr_device, lr = lr.data_ptr(), 0.0
    host.apart(params, momentum, grads)
    desc = _desc(steps=steps, coefficients=coefficients, eps=eps, beta=beta, nesterov=nesterov,
                 weight_decay=weight_decay, lr=lr, adjust=adjust)
    if all(g is None for g in grads):
        return

    def run(places):
        own = _at(params, places)
        _, p_at, g_at, _, _, _ = host.pairs(own, _at(grads, places), 1)
        _, m_at, *sizes, _ = host.matrices(_at(momentum, places), "momentum")
        ws = _workspace(sizes, len(own), device)
        _lib.check(_lib.lib().ictc_hip_muon_step(p_at, g_at, m_at, *sizes, len(own), ctypes.byref(desc), _lib.ptr(clip),
                                                 lr_device, _lib.ptr(ws), ws.numel(), _lib.stream_of(device)),
                   "ictc_hip_muon_step")

    with _on(device):
        _both_kinds(shapes, device, run)
    # the kernels write through addresses: tell autograd (and caches keyed on versions) of the change
    host.written(params, grads)
    host.written(momentum, grads)
