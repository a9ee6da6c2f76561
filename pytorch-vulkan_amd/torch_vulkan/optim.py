"""Opt-in fused AdamW and Muon for ``"vulkan"`` parameters.

``Muon`` keeps the constructor keywords and the state key (``momentum_buffer``)
of ``torch.optim.Muon``; every parameter group is one call of
``torch.ops.torch_vulkan.muon_step_``, in FP32 throughout.

AdamW: interface of the reference's ``torch_vulkan.optim.AdamW``
(torch_vulkan/optim.py:13-75 there): the constructor keywords ``lr``,
``betas``, ``eps``, ``weight_decay``, ``batched`` and ``amsgrad``, and per
parameter the state keys of ``torch.optim.AdamW`` (``step``, ``exp_avg``,
``exp_avg_sq``, ``max_exp_avg_sq``), so checkpoints move between this
optimizer and torch's.

How it runs here: each parameter group becomes one ``_GroupStep`` -- the
parameters that have gradients, their moment buffers and their host step
counts -- which is handed to the backend's custom ops
(``torch.ops.torch_vulkan.adamw_step_batch_`` / ``adamw_amsgrad_step_batch_``,
schemas of csrc/ops/adamw.cpp:307-317).  The backend turns one batch call into
one multi-tensor launch over every tensor of the group (a new launch only where
two entries alias).  ``batched=False`` issues one call per parameter instead
(``adamw_step_`` for plain AdamW; the AMSGrad variant has no single-tensor op,
so it gets a one-entry batch).  ``torch.optim.AdamW(fused=True)`` also runs on
the device, through ``aten::_fused_adamw_``.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

_ops = None


def _backend_ops():
    global _ops
    if _ops is None:
        _ops = torch.ops.torch_vulkan
    return _ops


def _check_hyperparameters(lr, betas, eps, weight_decay):
    beta1, beta2 = betas
    problems = [name for name, ok in (("lr", lr >= 0), ("eps", eps >= 0), ("weight_decay", weight_decay >= 0),
                                      ("beta1", 0 <= beta1 < 1), ("beta2", 0 <= beta2 < 1)) if not ok]
    if problems:
        raise ValueError(f"AdamW: out-of-range hyperparameter(s) {', '.join(problems)} "
                         f"(lr={lr}, betas={betas}, eps={eps}, weight_decay={weight_decay})")


def _host_step(value) -> int:
    """A step count as a Python int (torch.optim checkpoints store a tensor)."""
    return int(value.item()) if isinstance(value, torch.Tensor) else int(value)


@dataclass
class _GroupStep:
    """The tensors of one parameter group that take part in this step."""
    amsgrad: bool
    params: list = field(default_factory=list)
    grads: list = field(default_factory=list)
    exp_avgs: list = field(default_factory=list)
    exp_avg_sqs: list = field(default_factory=list)
    max_exp_avg_sqs: list = field(default_factory=list)
    steps: list = field(default_factory=list)

    def lists(self, sl=slice(None)):
        out = [self.params[sl], self.grads[sl], self.exp_avgs[sl], self.exp_avg_sqs[sl]]
        if self.amsgrad:
            out.append(self.max_exp_avg_sqs[sl])
        return out

    def launch(self, hyper, batched):
        ops = _backend_ops()
        batch_op = ops.adamw_amsgrad_step_batch_ if self.amsgrad else ops.adamw_step_batch_
        if batched:
            batch_op(*self.lists(), *hyper, self.steps)
            return
        for i in range(len(self.params)):
            if self.amsgrad:
                batch_op(*self.lists(slice(i, i + 1)), *hyper, self.steps[i:i + 1])
            else:
                ops.adamw_step_(*(lst[i] for lst in self.lists()), *hyper, self.steps[i])


class AdamW(torch.optim.Optimizer):
    """Decoupled-weight-decay Adam whose update runs as multi-tensor gfx950
    launches (see the module docstring)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, batched=True,
                 amsgrad=False):
        _check_hyperparameters(lr, betas, eps, weight_decay)
        defaults = {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay, "batched": batched,
                    "amsgrad": amsgrad}
        super().__init__(params, defaults)

    @staticmethod
    def _fill_state(p, state, keys):
        """Missing entries of a parameter's state: a fresh parameter's, or the
        buffer of a checkpoint written without AMSGrad that is resumed with it."""
        state.setdefault("step", 0)
        for key in keys:
            if key not in state:
                state[key] = torch.zeros_like(p, memory_format=torch.preserve_format)

    def _collect(self, group) -> _GroupStep:
        # One pass over the group, with the steps advanced by one.  It runs
        # ahead of the launch on every step, so the common parameter (state
        # present, an int step, the device of the one before) takes no call
        # into a method and no device-type string.  With the library's cheaper
        # alias check and step factors, issuing a step of 161 parameters takes
        # 130 us in place of 202 (its kernel: 126).
        batch = _GroupStep(amsgrad=bool(group["amsgrad"]))
        keys = ("exp_avg", "exp_avg_sq") + (("max_exp_avg_sq",) if batch.amsgrad else ())
        params, grads, exp_avgs, exp_avg_sqs = batch.params, batch.grads, batch.exp_avgs, batch.exp_avg_sqs
        max_exp_avg_sqs, steps = batch.max_exp_avg_sqs, batch.steps
        states, device = self.state, None
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            if g.is_sparse:
                raise RuntimeError("torch_vulkan AdamW: sparse gradients are not supported")
            if p.device != device:
                if p.device.type != "vulkan":
                    raise RuntimeError(f"torch_vulkan AdamW: parameter on {p.device}, expected a vulkan tensor")
                device = p.device
            state = states[p]
            try:
                step, exp_avg, exp_avg_sq = state["step"], state["exp_avg"], state["exp_avg_sq"]
                if batch.amsgrad:
                    max_exp_avg_sqs.append(state["max_exp_avg_sq"])
            except KeyError:
                self._fill_state(p, state, keys)
                step, exp_avg, exp_avg_sq = state["step"], state["exp_avg"], state["exp_avg_sq"]
                if batch.amsgrad:
                    max_exp_avg_sqs.append(state["max_exp_avg_sq"])
            step = step + 1 if type(step) is int else _host_step(step) + 1
            state["step"] = step
            params.append(p)
            grads.append(g)
            exp_avgs.append(exp_avg)
            exp_avg_sqs.append(exp_avg_sq)
            steps.append(step)
        return batch

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            batch = self._collect(group)
            if not batch.params:
                continue
            beta1, beta2 = group["betas"]
            hyper = (group["lr"], beta1, beta2, group["eps"], group["weight_decay"])
            batch.launch(hyper, group.get("batched", True))
        return loss


class Muon(torch.optim.Optimizer):
    """Orthogonalised momentum for matrices (two-dimensional FP32 parameters):
    matrices of one shape go through the Newton-Schulz products together."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True,
                 ns_coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, ns_steps=5, adjust_lr_fn=None):
        problems = [name for name, ok in (("lr", lr >= 0), ("weight_decay", weight_decay >= 0),
                                          ("momentum", 0 <= momentum <= 1), ("eps", eps > 0), ("ns_steps", ns_steps >= 0),
                                          ("ns_coefficients", len(ns_coefficients) == 3),
                                          ("adjust_lr_fn", adjust_lr_fn in (None, "original", "match_rms_adamw"))) if not ok]
        if problems:
            raise ValueError(f"Muon: out-of-range hyperparameter(s) {', '.join(problems)}")
        super().__init__(params, {"lr": lr, "weight_decay": weight_decay, "momentum": momentum, "nesterov": nesterov,
                                  "ns_coefficients": tuple(ns_coefficients), "eps": eps, "ns_steps": ns_steps,
                                  "adjust_lr_fn": adjust_lr_fn})
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon: only matrices are supported, got a parameter of shape {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params, grads, buffers = [], [], []
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("torch_vulkan Muon: sparse gradients are not supported")
                if p.device.type != "vulkan":
                    raise RuntimeError(f"torch_vulkan Muon: parameter on {p.device}, expected a vulkan tensor")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p.grad, memory_format=torch.contiguous_format)
                params.append(p)
                grads.append(p.grad)
                buffers.append(state["momentum_buffer"])
            if params:
                _backend_ops().muon_step_(params, grads, buffers, group["lr"], group["weight_decay"], group["momentum"],
                                          group["nesterov"], list(group["ns_coefficients"]), group["ns_steps"],
                                          group["eps"], group["adjust_lr_fn"] or "original")
        return loss
