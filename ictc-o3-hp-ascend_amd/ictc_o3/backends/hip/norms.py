"""Norms of a residual block on equivariant node features (``ictc_hip_norm_*``; no counterpart in the
reference, whose layers have none): the norm before the first block, and a block's end in one kernel
(norm of the block's output, gate, residual sum, norm before the next block).  Formulas stand in
``ictc_hip.h``.

Forward, gradients and the gradients of those (training on forces) each run as one kernel; beyond, where the
second ones are recorded, and for cotangents of weight gradients, the gradients' formulas are composed of torch
operations in 64 bits and differentiated, so every order stays available.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from ictc_o3 import _lib
from ictc_o3.autograd.adjoint_requirements import required_gradients

from .runtime import require_gpu_fp32

MAX_CHANNELS, MAX_LMAX = 1024, 3


def _degrees(width: int, channels: int, what: str) -> int:
    lmax = math.isqrt(width // channels) - 1
    if lmax < 0 or channels * (lmax + 1) ** 2 != width:
        raise ValueError(f"{what} must have channels * (lmax + 1)^2 columns, got {width} for {channels} channels")
    return lmax


def _cont(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


def _workspace(desc, rows: int, device) -> torch.Tensor:
    floats = int(_lib.lib().ictc_hip_norm_workspace(ctypes.byref(desc), rows))
    if floats < 0:
        _lib.check(-floats, "ictc_hip_norm_workspace")
    return torch.empty(floats, device=device, dtype=torch.float32)


def _forward(desc, x, block, gate, post, pre):
    p = _lib.ptr
    like = x if block is None else block
    h = None if block is None else torch.empty_like(like)
    y = None if pre is None else torch.empty_like(like)
    if x.shape[0] == 0:     # (tensors without elements have no address)
        return h, y
    _lib.check(_lib.lib().ictc_hip_norm_forward(ctypes.byref(desc), p(x), p(block), p(gate), p(post), p(pre), p(h),
                                                p(y), x.shape[0], _lib.stream_of(x.device)), "ictc_hip_norm_forward")
    return h, y


def _backward(desc, h, block, gate, post, pre, dh, dy, need):
    """Gradients to (x, block, gate, post, pre), None where not needed."""
    p = _lib.ptr
    like = h if block is None else block
    rows, device = like.shape[0], like.device
    dx = torch.empty(rows, desc.channels * (desc.input_lmax + 1) ** 2, device=device) if need[0] else None
    db = torch.empty_like(block) if need[1] else None
    dg = torch.empty_like(gate) if need[2] else None
    dpost = torch.empty_like(post) if need[3] else None
    dpre = torch.empty_like(pre) if need[4] else None
    if rows == 0:
        for w in (dpost, dpre):
            if w is not None:
                w.zero_()
        return dx, db, dg, dpost, dpre
    ws = _workspace(desc, rows, device) if need[3] or need[4] else None
    _lib.check(_lib.lib().ictc_hip_norm_backward(
        ctypes.byref(desc), p(h), p(block), p(gate), p(post), p(pre), p(dh), p(dy), p(dx), p(db), p(dg), p(dpost),
        p(dpre), p(ws), 0 if ws is None else ws.numel(), rows, _lib.stream_of(device)), "ictc_hip_norm_backward")
    return dx, db, dg, dpost, dpre


def _second(desc, x, h, block, gate, post, pre, dh, dy, cx, cb, cg, need):
    """Gradients to (x, block, gate, post, pre, dh, dy), None where not needed."""
    p = _lib.ptr
    rows, device = x.shape[0], x.device
    out = [torch.empty_like(t) if n else None for t, n in zip((x, block, gate, post, pre, dh, dy), need)]
    if rows == 0:
        for w in out[3:5]:
            if w is not None:
                w.zero_()
        return out
    ws = _workspace(desc, rows, device) if need[3] or need[4] else None
    gx, gb, gg, gpost, gpre, gdh, gdy = out
    _lib.check(_lib.lib().ictc_hip_norm_second(
        ctypes.byref(desc), p(h), p(block), p(gate), p(post), p(pre), p(dh), p(dy), p(cx), p(cb), p(cg), p(gx), p(gb),
        p(gg), p(gdh), p(gdy), p(gpost), p(gpre), p(ws), 0 if ws is None else ws.numel(), rows,
        _lib.stream_of(device)), "ictc_hip_norm_second")
    return out


ASK_FROM = 1 << 25   # values of a row operand


def _weights_run(post, pre, declared, rows) -> bool:
    """Whether the engine will use a weight's gradient (not so where forces are taken from positions).  One
    answer decides for both, rows are not asked about, and small calls ask nothing: a question takes the host 14
    to 20 us, the weights' gradients 5 us for 2,048 rows of 2,048 values, 9 for 8,192 and 35 for 32,768."""
    if rows.numel() < ASK_FROM:
        return any(declared)
    return any(n and required_gradients((w,), (True,))[0] for w, n in zip((post, pre), declared))


class _Layout:
    """Index of each column's degree and (degree, channel) place, and its share in the mean."""

    def __init__(self, channels: int, lmax: int, device):
        degree = torch.cat([torch.full((channels * (2 * l + 1),), l) for l in range(lmax + 1)])
        self.places = (lmax + 1) * channels
        self.place = (degree * channels + torch.cat([torch.arange(channels).repeat_interleave(2 * l + 1)
                                                     for l in range(lmax + 1)])).to(device)
        self.share = (1.0 / ((lmax + 1) * channels * (2 * degree + 1).double())).to(device)

    def spread(self, w):
        return w.reshape(-1, self.places)[:, self.place]

    def gather(self, v):
        """Sums over the components: [N, columns] -> [N, places]."""
        return v.new_zeros(v.shape[0], self.places).index_add(1, self.place, v)


def gradient_formula(desc, x, block, gate, post, pre, dh, dy):
    """(dx, dblock, dgate, dpost, dpre) of torch operations: what ``ictc_hip_norm_backward`` computes, from the
    forward pass's arguments.  In 64 bits, as the kernels' sums and projections are: what is left of a cotangent
    along its row (eps / (q + eps) of it for a row with one large entry) is a difference, and in 32 bits its
    rounding was all that came out (800 times the result at an entry of 300).  The results are rounded once."""
    dtype = x.dtype
    x, block, gate, post, pre, dh, dy = (None if t is None else t.double() for t in (x, block, gate, post, pre, dh, dy))
    lay = _Layout(desc.channels, desc.lmax, x.device)
    width, wide = desc.channels * (desc.lmax + 1) ** 2, x.shape[1]

    def fit(v, columns):
        return v[:, :columns] if columns <= v.shape[1] else torch.nn.functional.pad(v, (0, columns - v.shape[1]))

    def root(v):
        return ((v * v * lay.share).sum(1, keepdim=True) + desc.eps).rsqrt()

    def adjoint(v, rho, e):
        return rho * e - rho ** 3 * lay.share * v * (e * v).sum(1, keepdim=True)

    if block is not None:
        open_ = torch.ones_like(block[:, :1]) if gate is None else torch.sigmoid(gate)
        k, rho_b = desc.residual_scale * post.reshape(1, -1) * open_, root(block)
    r, dpre = dh, None
    if dy is not None:
        h = x if block is None else fit(x, width) + lay.spread(k.expand(x.shape[0], -1)) * rho_b * block
        rho = root(h)
        through = adjoint(h, rho, lay.spread(pre) * dy)
        r = through if dh is None else dh + through
        dpre = lay.gather(rho * dy * h).sum(0).view_as(pre)
    dx = fit(r, wide)
    if block is None:
        return dx.to(dtype), None, None, None, dpre.to(dtype)
    db = adjoint(block, rho_b, lay.spread(k.expand(x.shape[0], -1)) * r)
    along = rho_b * lay.gather(r * block) * desc.residual_scale
    dgate = None if gate is None else along * open_ * (1.0 - open_) * post.reshape(1, -1)
    results = dx, db, dgate, (along * open_).sum(0).view_as(post), dpre
    return tuple(None if t is None else t.to(dtype) for t in results)


class _Gradient(torch.autograd.Function):
    """The gradients as a function of (x, block, gate, post, pre, dh, dy); h is the forward pass's result."""

    @staticmethod
    def forward(ctx, desc, need, h, *inputs):
        ctx.set_materialize_grads(False)
        ctx.desc = desc
        ctx.save_for_backward(h, *inputs)
        return _backward(desc, h, *inputs[1:], need)

    @staticmethod
    def backward(ctx, *cots):
        h, *inputs = ctx.saved_tensors
        desc = ctx.desc
        x, block, gate, post, pre, dh, dy = inputs
        need = list(ctx.needs_input_grad[3:])
        if not _weights_run(post, pre, need[3:5], h):
            need[3] = need[4] = False
        if not any(need) or all(c is None for c in cots):
            return (None,) * 10
        graph = torch.is_grad_enabled()
        if graph or cots[3] is not None or cots[4] is not None:
            with torch.enable_grad():
                own = [None if t is None else t.view_as(t) if t.requires_grad else t for t in inputs]
                heads = [(o, c) for o, c in zip(gradient_formula(desc, *own), cots) if o is not None and c is not None
                         and o.requires_grad]
                leaves = [t for t, n in zip(own, need) if n]
                grads = [None] * len(leaves)
                if heads:
                    grads = torch.autograd.grad([o for o, _ in heads], leaves, [c for _, c in heads],
                                                create_graph=graph, allow_unused=True)
            grads = iter(grads)
            return (None, None, None, *[next(grads) if n else None for n in need])
        # x, dy and pre take part through the norm behind the block
        follows = dy is not None
        need = [n and (follows or i not in (0, 4, 6)) for i, n in enumerate(need)]
        if block is None:
            need[5] = False
        cx, cb, cg = (_cont(c) for c in cots[:3])
        return (None, None, None, *_second(desc, x, h, *inputs[1:], cx, cb, cg, need))


def _gradients(desc, need, h, x, *inputs):
    """The gradients, recorded where a graph is (a function of its own costs 15 us a call)."""
    if torch.is_grad_enabled():
        return _Gradient.apply(desc, need, h.detach(), x, *inputs)
    return _backward(desc, h, *inputs, need)


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, desc, x, pre):
        ctx.desc = desc
        ctx.save_for_backward(x, pre)
        return _forward(desc, x, None, None, None, pre)[1]

    @staticmethod
    def backward(ctx, dy):
        x, pre = ctx.saved_tensors
        need = (ctx.needs_input_grad[1], _weights_run(None, pre, (False, ctx.needs_input_grad[2]), x))
        if not any(need):
            return None, None, None
        dx, _, _, _, dpre = _gradients(ctx.desc, (need[0], False, False, False, need[1]), x, x, None, None, None,
                                       pre, None, dy.contiguous())
        return None, dx, dpre


class _BlockEnd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, desc, x, block, gate, post, pre):
        ctx.set_materialize_grads(False)
        ctx.desc = desc
        h, y = _forward(desc, x, block, gate, post, pre)
        ctx.save_for_backward(x, h, block, gate, post, pre)
        return h, y

    @staticmethod
    def backward(ctx, dh, dy):
        x, h, block, gate, post, pre = ctx.saved_tensors
        if dh is None and dy is None:
            return (None,) * 6
        need = list(ctx.needs_input_grad[1:])
        if not _weights_run(post, pre, need[3:5], h):
            need[3] = need[4] = False
        dx = None
        if dy is None:
            need[4] = False
            if need[0] and ctx.desc.input_lmax == ctx.desc.lmax:    # the sum passes its cotangent on
                dx, need[0] = dh, False
        if not any(need):
            return None, dx, None, None, None, None
        grads = _gradients(ctx.desc, tuple(need), h, x, block, gate, post, pre, _cont(dh), _cont(dy))
        return (None, grads[0] if dx is None else dx, *grads[1:])


def _weight(w: torch.Tensor, channels: int, lmax: int, what: str) -> torch.Tensor:
    if w.numel() != channels * (lmax + 1) or w.dim() not in (1, 2) or (w.dim() == 2 and w.shape[1] != channels):
        raise ValueError(f"{what} must have lmax + 1 = {lmax + 1} rows of {channels} channels (or be that, flat)")
    return w.contiguous()


def _sizes(rows: torch.Tensor, channels: int, eps: float, what: str) -> int:
    if not isinstance(channels, int) or isinstance(channels, bool) or not 1 <= channels <= MAX_CHANNELS:
        raise ValueError(f"channels must be an integer in [1, {MAX_CHANNELS}]")
    if not eps > 0.0 or not math.isfinite(eps):
        raise ValueError("eps must be positive")
    if rows.dim() != 2:
        raise ValueError(f"{what} must be two-dimensional")
    lmax = _degrees(rows.shape[1], channels, what)
    if lmax > MAX_LMAX:
        raise ValueError(f"the norms are compiled for lmax <= {MAX_LMAX}")
    return lmax


def equivariant_norm(features: torch.Tensor, weight: torch.Tensor, *, channels: int, eps: float = 1e-5):
    """Root-mean-square norm of node features [N, C (L+1)^2] in mul_ir order, every degree with the same
    weight in the mean, times a weight for each degree and channel ([L+1, C])."""
    lmax = _sizes(features, channels, eps, "features")
    weight = _weight(weight, channels, lmax, "the weight")
    require_gpu_fp32(features, weight)
    desc = _lib.NormDesc(channels, lmax, lmax, 1.0, eps)
    return _Norm.apply(desc, features.contiguous(), weight)


def gated_residual_norm(features: torch.Tensor, block: torch.Tensor, gate: Optional[torch.Tensor],
                        post_weight: torch.Tensor, pre_weight: Optional[torch.Tensor], *, channels: int,
                        residual_scale: float = 1.0, eps: float = 1e-5):
    """A block's end in one pass: (h, y) with

        h = features + residual_scale * sigmoid(gate) * norm(block; post_weight)      y = norm(h; pre_weight)

    block [N, C (L+1)^2] and features (its degrees may be fewer: the missing ones are zero; or more: those
    are left out) in mul_ir order; gate [N, (L+1) C], or None for none; weights [L+1, C]; pre_weight None:
    no norm behind the block (y is None).  norm is ``equivariant_norm``'s."""
    lmax = _sizes(block, channels, eps, "block")
    if features.dim() != 2 or features.shape[0] != block.shape[0]:
        raise ValueError("features must be two-dimensional, with a row for each of the block's")
    input_lmax = _degrees(features.shape[1], channels, "features")
    if gate is not None and gate.shape != (block.shape[0], (lmax + 1) * channels):
        raise ValueError(f"gate must have shape [{block.shape[0]}, {(lmax + 1) * channels}]")
    if isinstance(residual_scale, bool) or not isinstance(residual_scale, (int, float)) \
            or not math.isfinite(residual_scale):
        raise ValueError("residual_scale must be a finite number")
    post_weight = _weight(post_weight, channels, lmax, "post_weight")
    if pre_weight is not None:
        pre_weight = _weight(pre_weight, channels, lmax, "pre_weight")
    require_gpu_fp32(*[t for t in (features, block, gate, post_weight, pre_weight) if t is not None])
    desc = _lib.NormDesc(channels, lmax, input_lmax, float(residual_scale), eps)
    return _BlockEnd.apply(desc, features.contiguous(), block.contiguous(), _cont(gate), post_weight, pre_weight)
