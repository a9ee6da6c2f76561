"""Linear layers whose bias, activation and residual ride in the product's
epilogue, for ``"vulkan"`` tensors.

``linear(x, weight, bias, activation, residual)`` computes
``act(x @ weight.T + bias) + residual`` in one call and its gradients in
another; ``Linear`` is ``torch.nn.Linear`` with that call (same parameters and
state dict).  ``torch.nn.LayerNorm`` runs on the device as it is.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, keep):
        y, z = torch.ops.torch_vulkan.linear_act(x, weight, bias, residual, activation, keep)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, z if keep else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx = dw = db = None
        if any(want[:3]):
            got = torch.ops.torch_vulkan.linear_act_backward(dy, x, weight, z, ctx.activation, list(want[:3]))
            dx, dw, db = (g if w else None for g, w in zip(got, want))
        return dx, dw, db, dy if want[3] else None, None, None


def linear(x, weight, bias=None, activation="none", residual=None):
    """``act(x @ weight.T + bias) + residual``; x [..., k], weight [n, k], bias
    [n], residual broadcastable to [..., n].  activation: one of ACTIVATIONS."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: activation must be one of {ACTIVATIONS}, got {activation!r}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: input {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    shape = (*x.shape[:-1], weight.shape[0])
    flat = x.reshape(math.prod(shape[:-1]), x.shape[-1])
    if residual is not None:
        residual = residual.expand(shape).reshape(flat.shape[0], shape[-1])
    # The activation's input is kept only where a gradient will ask for it.  Within
    # the function a parameter needs its gradient under no_grad too, and the mode is
    # off whatever the caller's.
    keep = activation != "none" and torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (flat, weight, bias))
    return _Linear.apply(flat, weight, bias, residual, activation, keep).view(shape)


class Linear(torch.nn.Linear):
    """``torch.nn.Linear`` with the activation in its epilogue; ``forward(x,
    residual=None)``."""

    def __init__(self, in_features, out_features, bias=True, activation="none", device=None, dtype=None):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        if activation not in ACTIVATIONS:
            raise ValueError(f"Linear: activation must be one of {ACTIVATIONS}, got {activation!r}")
        self.activation = activation

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self):
        return super().extra_repr() + f", activation={self.activation}"
