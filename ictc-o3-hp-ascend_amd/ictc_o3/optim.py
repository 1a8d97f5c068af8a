"""AdamW on the HIP kernels: one update launch for all of a model's tensors, moments in float32 or in
8 bits, gradients clipped by their global norm on the way (``ictc_o3.backends.hip.optimizer``).

    optimizer = ictc_o3.optim.AdamW(model.parameters(), lr=1e-3, moment_bits=8, max_grad_norm=10.0)
    mace_hip.training_step(model, optimizer, graph)
    mace_hip.CapturedTrainingStep(model, optimizer, graph)

The step reads nothing back and keeps its state on the device, so it can be captured as it is (a learning
rate that changes between replays is given as a one-element float32 tensor; the first step of a group makes
its moments and is taken outside of the capture).
"""
from __future__ import annotations

import torch

from ictc_o3.backends.hip.optimizer import MOMENT_BLOCK, adamw_step, gradient_norm, moment_values, new_state


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with torch.optim's interface, for contiguous float32 parameters on a GPU.
    Moments are kept for whole groups (``moments`` gives one parameter's; ``state`` stays empty).

    moment_bits: 32 or 8 bits a value (8: blocks of 256 values with a power of two as scale, rounded at
    random from ``seed``).  max_grad_norm: the global norm of all groups' gradients is limited to it
    before the step; a norm that is not finite leaves parameters, moments and steps as they are (and is
    seen in ``grad_norm``, the last step's [norm, coefficient] on the device)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, moment_bits=32,
                 max_grad_norm=None, seed=0):
        if moment_bits not in (32, 8):
            raise ValueError("moment_bits must be 32 or 8")
        if max_grad_norm is not None and not float(max_grad_norm) > 0.0:
            raise ValueError("max_grad_norm must be positive or None")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError("lr must not be negative")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("betas must lie in [0, 1)")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("eps and weight_decay must not be negative")
        self.moment_bits, self.max_grad_norm, self.seed = moment_bits, max_grad_norm, int(seed)
        self.grad_norm = None
        self._moments = []           # for each group (exp_avg, exp_avg_sq, progress), or None before its first step
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, capturable=True))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        if not all(p.is_contiguous() for p in params) or len({id(p) for p in params}) != len(params):
            self.param_groups.pop()
            raise ValueError("parameters must be contiguous, and each in its group once")
        self._moments.append(None)

    def __getstate__(self):
        """For copies and pickles: torch's own part and what this class adds to it."""
        own = ("moment_bits", "max_grad_norm", "seed", "grad_norm", "_moments")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in own}}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grads = [[p.grad for p in group["params"]] for group in self.param_groups]
        first = any(state is None and any(g is not None for g in gs) for state, gs in zip(self._moments, grads))
        if first and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a group's first step makes its moments and cannot be captured: every replay would be a "
                               "first step (take a step, or load a state, before the capture)")
        clip = None
        if self.max_grad_norm is not None and any(g is not None for gs in grads for g in gs):
            clip = self.grad_norm = gradient_norm([g for gs in grads for g in gs], self.max_grad_norm)
        for i, (group, gs) in enumerate(zip(self.param_groups, grads)):
            if all(g is None for g in gs):
                continue
            if self._moments[i] is None:
                self._moments[i] = new_state(group["params"], self.moment_bits)
            adamw_step(group["params"], gs, *self._moments[i], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], clip=clip, seed=self.seed + i)
        return loss

    def moments(self, param: torch.Tensor):
        """(exp_avg, exp_avg_sq, steps) of one parameter: the values its moments stand for (float32, or
        bfloat16 for 8-bit moments) and its number of steps (a device scalar); None before the first step."""
        for group, state in zip(self.param_groups, self._moments):
            at = 0
            for row, p in enumerate(group["params"]):
                if p is param:
                    if state is None:
                        return None
                    m, v = state[:2] if self.moment_bits == 32 else moment_values(*state[:2])
                    part = slice(at, at + p.numel())
                    return m[part].view(p.shape), v[part].view(p.shape), state[2][row, 0]
                at += -(-p.numel() // MOMENT_BLOCK) * MOMENT_BLOCK
        raise ValueError("not a parameter of this optimizer")

    def state_dict(self):
        out = super().state_dict()
        out["moment_bits"], out["seed"], out["moments"] = self.moment_bits, self.seed, list(self._moments)
        return out

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Restores hyperparameters, moments and steps.  Moments and learning rate tensors that exist are
        overwritten in place, so a captured step goes on from what was loaded (numbers among its
        hyperparameters are part of the graph: a rate that has to follow is a tensor)."""
        if state_dict.get("moment_bits") != self.moment_bits or len(state_dict["moments"]) != len(self.param_groups):
            raise ValueError("the state has another number of moment bits or of parameter groups")
        new = []
        for group, saved in zip(self.param_groups, state_dict["moments"]):
            own = None
            if saved is not None:
                own = new_state(group["params"], self.moment_bits)
                for a, b in zip(_tensors(own), _tensors(saved)):
                    if a.shape != b.shape or a.dtype != b.dtype:
                        raise ValueError("the state belongs to parameters of other sizes")
                    a.copy_(b)
            new.append(own)
        rates = [group["lr"] for group in self.param_groups]
        loaded = {}                  # groups may share a tensor (the default's): one value for all of them
        for rate, group in zip(rates, state_dict["param_groups"]):
            if isinstance(rate, torch.Tensor) and loaded.setdefault(id(rate), float(group["lr"])) != float(group["lr"]):
                raise ValueError("groups that share a learning rate tensor cannot take different learning rates")
        super().load_state_dict({k: state_dict[k] for k in ("state", "param_groups")})
        for rate, group in zip(rates, self.param_groups):
            if isinstance(rate, torch.Tensor):
                rate.copy_(torch.as_tensor(group["lr"]).reshape(rate.shape))
                group["lr"] = rate
            elif isinstance(group["lr"], torch.Tensor):
                group["lr"] = group["lr"].to(group["params"][0].device)
        self.seed = int(state_dict["seed"])
        for i, own in enumerate(new):
            if self._moments[i] is None:
                self._moments[i] = own
                continue
            if own is None:
                own = new_state(self.param_groups[i]["params"], self.moment_bits)
            for a, b in zip(_tensors(self._moments[i]), _tensors(own)):
                a.copy_(b)


def _tensors(state):
    """The tensors of one group's state, in order."""
    return [t for part in state for t in ((part,) if isinstance(part, torch.Tensor) else part)]
