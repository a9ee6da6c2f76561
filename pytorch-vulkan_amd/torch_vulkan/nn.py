"""Linear layers whose bias, activation and residual ride in the product's
epilogue, and attention layers, for ``"vulkan"`` tensors.

``linear(x, weight, bias, activation, residual)`` computes
``act(x @ weight.T + bias) + residual`` in one call and its gradients in
another; ``Linear`` is ``torch.nn.Linear`` with that call (same parameters and
state dict).  ``torch.nn.LayerNorm`` runs on the device as it is.

``qk_norm_rotary``, ``attention`` and ``KVCache`` are the parts of an attention
layer on packed sequences [tokens, heads, head_dim], ``Attention`` is the layer.
Gradients once, FP32, on the device alone; ``rotary_frequencies`` gives the
rotation's frequencies, stretched for contexts longer than a model was trained on.
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


def rotary_frequencies(rotary_dim, base=10000.0, factor=1.0, trained=None, turns=(1.0, 32.0)):
    """Angles a position of a rotation's pairs: ``base ** (-2 i / rotary_dim)``.

    factor > 1 stretches them for a context that many times as long as the one
    trained on: all of them alike (every position divided by factor), or, where
    ``trained`` names that context's length, by parts: a pair that makes more
    than turns[1] turns within it keeps its frequency, one that makes fewer
    than turns[0] is divided by factor, and those between are mixed in
    proportion to their turns."""
    if rotary_dim % 2 or rotary_dim < 0:
        raise ValueError(f"rotary_frequencies: rotary_dim must be even, got {rotary_dim}")
    if not base > 0 or not factor > 0 or (trained is not None and not (trained > 0 and turns[0] < turns[1])):
        raise ValueError("rotary_frequencies: base, factor and trained must be positive, turns ascend")
    out = []
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        keep = 0.0
        if trained is not None:
            keep = min(1.0, max(0.0, (trained * f / (2 * math.pi) - turns[0]) / (turns[1] - turns[0])))
        out.append(f * keep + f / factor * (1 - keep))
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, form):
        ctx.form = form
        ctx.save_for_backward(q if form[3] is not None else None, k if form[3] is not None else None, q_weight, k_weight, positions)
        frequencies, interleaved, magnitude, eps = form
        return torch.ops.torch_vulkan.qk_norm_rotary(q, k, positions, frequencies, interleaved, magnitude, q_weight, k_weight, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        frequencies, interleaved, magnitude, eps = ctx.form
        want = ctx.needs_input_grad[:4]
        got = torch.ops.torch_vulkan.qk_norm_rotary_backward(dq, dk, q, k, positions, frequencies, interleaved, magnitude,
                                                             q_weight, k_weight, eps, list(want))
        return *(g if w else None for g, w in zip(got, want)), None, None


def qk_norm_rotary(q, k, positions, frequencies, interleaved=False, magnitude=1.0, q_weight=None, k_weight=None, eps=None):
    """Norm of each head of q and k (``x / sqrt(mean(x ** 2) + eps) * weight``; eps
    None: none) and rotation of the first 2 len(frequencies) elements by
    ``positions * frequencies``, in pairs of neighbours (interleaved) or of halves.
    q and k are [tokens, heads, head_dim], positions int64 [tokens]."""
    return _Rotary.apply(q, k, q_weight, k_weight, positions, (list(frequencies), interleaved, magnitude, eps))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, form):
        out, lse = torch.ops.torch_vulkan.attention(q, k, v, starts, *form)
        ctx.form = form
        ctx.save_for_backward(q, k, v, out, lse, starts)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, starts = ctx.saved_tensors
        want = ctx.needs_input_grad[:3]
        got = torch.ops.torch_vulkan.attention_backward(dout, q, k, v, out, lse, starts, *ctx.form, list(want))
        return *(g if w else None for g, w in zip(got, want)), None, None


def attention(q, k, v, starts=None, sequences=1, window=0, sinks=0, scale=None):
    """Causal attention of packed sequences: q [tokens, heads, head_dim], k and v
    [tokens, kv_heads, head_dim], kv_heads a divisor of heads.  starts: int32
    [sequences + 1], every sequence's first row and the last one's end (rows outside
    get zeros), or None for ``sequences`` of equal length.  A row sees the last
    ``window`` tokens, itself among them (0: all), and the first ``sinks``.  scale
    None: head_dim ** -0.5."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    return _Attention.apply(q, k, v, starts, (sequences, window, sinks, scale))


class KVCache:
    """Keys and values of many sequences in pages of ``page_size`` tokens: int8 with a
    scale to a token and head, or float32.

    A batch names new tokens and their sequences: ``table`` int32 [sequences,
    pages], the pages of each in order (-1: released), ``lengths`` int32
    [sequences], tokens with the new ones, and ``starts`` as in attention(), None
    for as many new tokens of each."""

    def __init__(self, pages, heads, page_size, head_dim, dtype=torch.int8, device="vulkan"):
        if dtype not in (torch.int8, torch.float32):
            raise ValueError(f"KVCache: dtype must be int8 or float32, got {dtype}")
        if page_size < 16 or page_size % 16 or head_dim < 16 or head_dim % 16 or head_dim > 128:
            raise ValueError(f"KVCache: page_size and head_dim must be multiples of 16, head_dim at most 128, got {page_size} "
                             f"and {head_dim}")
        new = lambda *shape, dtype: torch.zeros(*shape, dtype=dtype, device=device)
        self.k, self.v = new(pages, heads, page_size, head_dim, dtype=dtype), new(pages, heads, head_dim, page_size, dtype=dtype)
        scales = dtype == torch.int8
        self.k_scale, self.v_scale = (new(pages, heads, page_size, dtype=torch.float32) if scales else None for _ in range(2))

    def _held(self):
        return self.k, self.v, self.k_scale, self.v_scale

    def write(self, k, v, table, lengths, starts=None):
        """Writes the new tokens' k and v [tokens, heads, head_dim]."""
        torch.ops.torch_vulkan.kv_cache_write_(*self._held(), table, lengths, starts, k, v)

    def read(self, tokens, table, lengths, starts=None):
        """The last tokens of every sequence (as many as starts names), as float32 k and v."""
        return torch.ops.torch_vulkan.kv_cache_read(*self._held(), table, lengths, starts, tokens)

    def attention(self, q, table, lengths, starts=None, window=0, sinks=0, scale=None):
        """Attention of the new tokens, written before, over their sequences; no gradients."""
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        return torch.ops.torch_vulkan.attention_paged(*self._held(), table, lengths, starts, q, window, sinks, scale)


class Attention(torch.nn.Module):
    """An attention layer: projections, norm and rotation of queries and keys, causal
    attention, projection back.  x is [tokens, width], packed sequences.

    ``forward(x, positions, starts=None, sequences=1, residual=None)`` trains;
    with ``cache`` (a KVCache) and its batch's ``table`` and ``lengths`` the new
    tokens are written to it and attend over it."""

    def __init__(self, width, heads, kv_heads=None, head_dim=None, window=0, sinks=0, qk_norm=True, frequencies=None,
                 eps=1e-6, bias=False, device=None, dtype=None):
        super().__init__()
        kv_heads, head_dim = kv_heads or heads, head_dim or width // heads
        if heads % kv_heads:
            raise ValueError(f"Attention: {heads} heads do not share {kv_heads} key heads evenly")
        self.heads, self.kv_heads, self.head_dim, self.window, self.sinks = heads, kv_heads, head_dim, window, sinks
        self.frequencies = rotary_frequencies(head_dim // 2 * 2) if frequencies is None else list(frequencies)
        self.eps = eps if qk_norm else None
        made = dict(device=device, dtype=dtype)
        self.q = Linear(width, heads * head_dim, bias=bias, **made)
        self.k = Linear(width, kv_heads * head_dim, bias=bias, **made)
        self.v = Linear(width, kv_heads * head_dim, bias=bias, **made)
        self.out = Linear(heads * head_dim, width, bias=bias, **made)
        for name in ("q_weight", "k_weight"):
            self.register_parameter(name, torch.nn.Parameter(torch.ones(head_dim, **made)) if qk_norm else None)

    def forward(self, x, positions, starts=None, sequences=1, residual=None, cache=None, table=None, lengths=None):
        split = lambda t, heads: t.view(x.shape[0], heads, self.head_dim)
        q, k = qk_norm_rotary(split(self.q(x), self.heads), split(self.k(x), self.kv_heads), positions, self.frequencies,
                              q_weight=self.q_weight, k_weight=self.k_weight, eps=self.eps)
        v = split(self.v(x), self.kv_heads)
        if cache is None:
            mixed = attention(q, k, v, starts, sequences, self.window, self.sinks)
        else:
            cache.write(k, v, table, lengths, starts)
            mixed = cache.attention(q, table, lengths, starts, self.window, self.sinks)
        return self.out(mixed.view(x.shape[0], self.heads * self.head_dim), residual)
