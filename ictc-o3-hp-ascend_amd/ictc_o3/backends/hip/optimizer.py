"""The optimizer step on ``libictc_hip.so``: the norm of all gradients and one AdamW update of many
tensors (``ictc_hip_gradient_norm``, ``ictc_hip_adamw_step``; no counterpart in the reference, whose
training loop uses torch's optimizers).  Formulas and the 8-bit format stand in ``ictc_hip.h``.

Nothing here reads from the device or copies to it: the tensors' addresses are kernel arguments, and
steps, clipping coefficient and (where it is a tensor) the learning rate stay on the device, so a step
can be captured into a HIP graph.  ``ictc_o3.optim.AdamW`` is the optimizer on top.
"""
from __future__ import annotations

import ctypes
import math
from contextlib import nullcontext

import torch

from ictc_o3 import _lib

MOMENT_BLOCK = 256
_HERE = nullcontext()


def _on(device: torch.device):
    """The launch's device made current where it is not (streams belong to a device)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def state_values(sizes) -> int:
    """Values of the flat moments for tensors of these sizes (each padded to whole blocks)."""
    return sum(-(-n // MOMENT_BLOCK) for n in sizes) * MOMENT_BLOCK


def new_state(params, moment_bits: int = 32):
    """(exp_avg, exp_avg_sq, progress) before the first step: zeros, and no steps for each tensor.
    8-bit moments are (codes, block exponents) pairs."""
    params = list(params)
    if not params:
        raise ValueError("expected at least one parameter")
    device = torch.device("cuda", _lib.host().addresses(params, "parameters")[0])
    total = state_values([p.numel() for p in params])
    if moment_bits == 32:
        moments = [torch.zeros(total, device=device) for _ in range(2)]
    elif moment_bits == 8:
        moments = [(torch.zeros(total, device=device, dtype=torch.uint8),
                    torch.zeros(total // MOMENT_BLOCK, device=device, dtype=torch.uint8)) for _ in range(2)]
    else:
        raise ValueError("moment_bits must be 32 or 8")
    progress = torch.ones(len(params), 3, device=device, dtype=torch.float64)
    progress[:, 0] = 0.0
    return moments[0], moments[1], progress


def gradient_norm(grads, max_norm=None) -> torch.Tensor:
    """[norm, coefficient] on the device: the 2-norm of all gradients together and min(1, max_norm /
    norm) (1 without max_norm; not-a-number for a norm that is not finite, with which ``adamw_step``
    leaves everything as it is).  The gradients are not changed; entries that are None are left out."""
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("expected at least one gradient")
    if max_norm is not None and not float(max_norm) > 0.0:
        raise ValueError("max_norm must be positive, or None for no limit")
    # (as a float32: one that rounds to zero would mean no limit)
    limit = 0.0 if max_norm is None or math.isinf(max_norm) else max(float(max_norm), 2.0 ** -149)
    _, at, sizes, contiguous = _lib.host().addresses(grads, "gradients")
    if not contiguous:
        grads = [g.contiguous() for g in grads]
        _, at, sizes, _ = _lib.host().addresses(grads, "gradients")
    n, device = len(grads), grads[0].device
    out = torch.empty(2, device=device)
    lib = _lib.lib()
    doubles = lib.ictc_hip_gradient_norm_workspace(n)
    workspace = torch.empty(doubles, device=device, dtype=torch.float64)
    with _on(device):
        _lib.check(lib.ictc_hip_gradient_norm(
            at, sizes, n, limit, workspace.data_ptr(), doubles, out.data_ptr(), _lib.stream_of(device)),
            "ictc_hip_gradient_norm")
    return out


def _moments(state, values: int, device, what: str):
    """(address of the values or codes, address of the exponents or None, bits)."""
    if isinstance(state, torch.Tensor):
        if state.dtype is not torch.float32 or state.numel() != values or not state.is_contiguous() \
                or state.device != device:
            raise ValueError(f"{what} must be a contiguous FP32 tensor of {values} values beside the parameters")
        return state.data_ptr(), None, 32
    codes, top = state
    if (codes.dtype is not torch.uint8 or top.dtype is not torch.uint8 or codes.numel() != values
            or top.numel() * MOMENT_BLOCK != values or not codes.is_contiguous() or not top.is_contiguous()
            or codes.device != device or top.device != device):
        raise ValueError(f"{what} must be contiguous uint8 codes ({values}) and exponents "
                         f"({values // MOMENT_BLOCK}) beside the parameters")
    return codes.data_ptr(), top.data_ptr(), 8


def _number(value, name: str, below: float = math.inf) -> float:
    if isinstance(value, bool) or not isinstance(value, (int, float)) or not 0.0 <= value < below:
        raise ValueError(f"{name} must be a number in [0, {below})")
    return float(value)


def adamw_step(params, grads, exp_avg, exp_avg_sq, progress, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               clip=None, seed=0) -> None:
    """One AdamW step of every parameter with a gradient, in place (a None gradient leaves its
    parameter, moments and steps as they are).  One launch updates many tensors side by side: no two of
    them may overlap.

    exp_avg, exp_avg_sq, progress: as ``new_state`` makes them (float32 moments, or pairs of 8-bit codes
    and block exponents; for each parameter its steps t, beta1^t and beta2^t, further rows are left alone).
    lr: a number, or a one-element float32 tensor on the device.  clip: ``gradient_norm``'s result, whose
    coefficient scales the gradients.  seed: of the 8-bit rounding."""
    params, grads = list(params), list(grads)
    _, p_at, g_at, sizes, values, contiguous = _lib.host().pairs(params, grads, MOMENT_BLOCK)
    if not contiguous:
        grads = [g if g is None else g.contiguous() for g in grads]
        _, p_at, g_at, sizes, values, _ = _lib.host().pairs(params, grads, MOMENT_BLOCK)
    n, device = len(params), params[0].device
    m, m_top, bits = _moments(exp_avg, values, device, "exp_avg")
    v, v_top, v_bits = _moments(exp_avg_sq, values, device, "exp_avg_sq")
    if bits != v_bits:
        raise ValueError("exp_avg and exp_avg_sq must have the same number of bits")
    if (progress.dim() != 2 or progress.shape[0] < n or progress.shape[1] != 3 or progress.dtype is not torch.float64
            or not progress.is_contiguous() or progress.device != device):
        raise ValueError(f"progress must be a contiguous float64 tensor of at least {n} rows of 3 beside the "
                         "parameters")
    if clip is not None and (clip.dtype is not torch.float32 or clip.shape != (2,) or clip.device != device
                             or not clip.is_contiguous()):
        raise ValueError("clip must be gradient_norm's result")
    lr_device = None
    if isinstance(lr, torch.Tensor):
        if lr.dtype is not torch.float32 or lr.numel() != 1 or lr.device != device:
            raise ValueError("a learning rate tensor must hold one FP32 value beside the parameters")
        lr_device, lr = lr.data_ptr(), 0.0
    desc = _lib.AdamwDesc(_number(betas[0], "beta1", 1.0), _number(betas[1], "beta2", 1.0),
                          _number(weight_decay, "weight_decay"), _number(lr, "lr"), _number(eps, "eps"),
                          int(seed) & 0xFFFFFFFF, bits)
    with _on(device):
        _lib.check(_lib.lib().ictc_hip_adamw_step(
            p_at, g_at, sizes, n, ctypes.byref(desc), m, v, m_top, v_top, progress.data_ptr(),
            _lib.ptr(clip), lr_device, _lib.stream_of(device)), "ictc_hip_adamw_step")
    # the kernel writes through addresses: tell autograd (and caches keyed on versions) of the change
    _lib.host().written(params, grads)


def moment_values(exp_avg, exp_avg_sq):
    """8-bit moments as the values they stand for, bfloat16 (which holds them exactly)."""
    codes = exp_avg[0]
    values, device = codes.numel(), codes.device
    if not codes.is_cuda or values % MOMENT_BLOCK:
        raise ValueError("expected 8-bit moments on a ROCm GPU")
    m, m_top, _ = _moments(exp_avg, values, device, "exp_avg")
    v, v_top, _ = _moments(exp_avg_sq, values, device, "exp_avg_sq")
    out = [torch.empty(values, device=device, dtype=torch.bfloat16) for _ in range(2)]
    with _on(device):
        _lib.check(_lib.lib().ictc_hip_moment_values(m, m_top, v, v_top, out[0].data_ptr(), out[1].data_ptr(), values,
                                                     _lib.stream_of(device)), "ictc_hip_moment_values")
    return out[0], out[1]
