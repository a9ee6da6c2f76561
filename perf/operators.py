"""The residual feed-forward block of a language model and its optimizer step, as cases that can be timed.

Three operators of FP32 training and serving: layer normalisation, a linear
layer whose bias, activation and residual ride in the product's epilogue, and
the orthogonalised momentum step (Muon) of the block's matrices.  ``listed()``
names twelve pieces of such work, ``draw()`` gives others of the same ranges,
``run()`` passes one of them through elementary torch operations or, where
``own`` is true, through this backend's kernels (``torch_vulkan.mx`` on the
tensors' own device pointers), and ``exact()`` restates it in float64.

Case fields: ``kind`` selects the operator, the others are its sizes.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-vulkan_amd")

EPS = 1e-5                              # layer norm
STEPS, NS_EPS = 5, 1e-7                 # orthogonalisation: iterations, smallest norm divided by
NS = (3.4445, -4.7750, 2.0315)          # its polynomial a x + b x^3 + c x^5
LR, DECAY, MOMENTUM = 0.02, 0.1, 0.95   # optimizer step


def listed():
    return [
        # A served token through the norm in front of a block: latency alone.
        dict(name="norm_token", kind="norm", rows=1, cols=1024, train=False),
        # A prompt of 2,048 tokens through the same norm.
        dict(name="norm_prompt", kind="norm", rows=2048, cols=1024, train=False),
        # A training micro-batch, forward and all gradients.
        dict(name="norm_train", kind="norm", rows=8192, cols=1024, train=True),
        # Odd sizes: rows that start at no 16-byte boundary.
        dict(name="norm_odd_train", kind="norm", rows=5001, cols=1447, train=True),
        # Wide rows of a large model, forward and all gradients.
        dict(name="norm_wide_train", kind="norm", rows=8192, cols=4096, train=True),
        # Four tokens decoded together through the up-projection: the weight is
        # read once for almost no arithmetic.
        dict(name="linear_tokens", kind="linear", m=4, k=1024, n=4096, act="gelu", residual=False, train=False),
        # Training, up-projection of a block: GELU in the epilogue.
        dict(name="linear_up_train", kind="linear", m=4096, k=1024, n=4096, act="gelu", residual=False, train=True),
        # Training, down-projection back onto the residual stream.
        dict(name="linear_down_train", kind="linear", m=4096, k=4096, n=1024, act="none", residual=True, train=True),
        # Odd sizes in every direction, everything in the epilogue at once.
        dict(name="linear_odd_train", kind="linear", m=1537, k=765, n=2050, act="silu", residual=True, train=True),
        # Orthogonalising one matrix of a large layer.
        dict(name="orthogonalize_large", kind="orthogonalize", count=1, rows=4096, cols=4096),
        # Optimizer step over the square matrices of four attention layers.
        dict(name="muon_square", kind="muon", count=16, rows=1024, cols=1024),
        # Optimizer step over the output projections of a small convolution or
        # feed-forward net: odd, tall matrices, where launches count.
        dict(name="muon_tall_odd", kind="muon", count=6, rows=1000, cols=513),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "linear", "linear", "linear", "orthogonalize", "muon", "muon"])
    if kind == "norm":
        cols = _log(rng, 64, 8192)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        return dict(kind=kind, rows=min(_log(rng, 1, 16384), 8192 * 4096 // cols), cols=cols, train=rng.random() < 0.7)
    if kind == "linear":
        m, k, n = _log(rng, 1, 8192), _log(rng, 64, 4096), _log(rng, 64, 4096)
        if rng.random() < 0.5:
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        m = max(1, min(m, int(4096 * 1024 * 4096 / (k * n))))
        return dict(kind=kind, m=m, k=k, n=n, act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    residual=rng.random() < 0.5, train=rng.random() < 0.7)
    rows, cols = _log(rng, 32, 4096), _log(rng, 32, 4096)
    if rng.random() < 0.5:
        rows, cols = max(64, rows // 64 * 64), max(64, cols // 64 * 64)
    count = _log(rng, 1, 16)
    while count > 1 and count * _ns_flops(rows, cols) > _ns_flops(2048, 2048):
        count -= 1
    return dict(kind=kind, count=count, rows=rows, cols=cols)


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Named float32 tensors of one case, made on the GPU from the seed alone."""
    g, c = torch.Generator(device="cuda").manual_seed(seed), case

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=g) * scale + mean

    if c["kind"] == "norm":
        # Activations of a residual stream: every row has a level and a spread of its own.
        x = normal(c["rows"], c["cols"]) * (normal(c["rows"], 1).abs() + 0.2) + normal(c["rows"], 1, scale=0.3)
        return dict(x=x, gamma=normal(c["cols"], scale=0.2, mean=1.0), beta=normal(c["cols"], scale=0.2),
                    dy=normal(c["rows"], c["cols"], scale=0.05) if c["train"] else None)
    if c["kind"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        return dict(x=normal(m, k), w=normal(n, k, scale=k ** -0.5), b=normal(n, scale=0.1),
                    res=normal(m, n) if c["residual"] else None, dy=normal(m, n, scale=0.05) if c["train"] else None)
    shape = (c["count"], c["rows"], c["cols"])
    # Gradients of matrices: a few strong directions over noise.
    grad = normal(*shape, scale=1e-3) + 3e-3 * torch.matmul(normal(*shape[:2], 4), normal(shape[0], 4, shape[2]))
    if c["kind"] == "orthogonalize":
        return dict(grad=grad)
    return dict(grad=grad, momentum=normal(*shape, scale=1e-3), param=normal(*shape, scale=shape[2] ** -0.5))


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# --------------------------------------------------------------- operators
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state, state["case"])
    with torch.no_grad():
        return _PLAIN[kind](state, state["case"])


def _plain_norm(t, c):
    x, gamma = t["x"], t["gamma"]
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = (d * d).mean(1, keepdim=True).add(EPS).rsqrt()
    xhat = d * rstd
    y = xhat * gamma + t["beta"]
    if not c["train"]:
        return [y]
    dy = t["dy"]
    g = dy * gamma
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return [y, dx, (dy * xhat).sum(0), dy.sum(0)]


def _act(name, z):
    """The activation of z and its derivative there."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    r = math.sqrt(2 / math.pi)
    h = torch.tanh(r * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + h), 0.5 * (1 + h) + 0.5 * z * (1 - h * h) * r * (1 + 3 * 0.044715 * z * z)


def _plain_linear(t, c):
    z = torch.matmul(t["x"], t["w"].t()) + t["b"]
    y, slope = _act(c["act"], z)
    if c["residual"]:
        y = y + t["res"]
    if not c["train"]:
        return [y]
    dz = t["dy"] * slope
    return [y, torch.matmul(dz, t["w"]), torch.matmul(dz.t(), t["x"]), dz.sum(0)]


def _orthogonal(u):
    """Newton-Schulz iterations on a stack of matrices (float32; the norm in float64)."""
    a, b, c = NS
    norm = (u.double() * u.double()).sum((1, 2), keepdim=True).sqrt().clamp_min(NS_EPS)
    x = (u.double() / norm).to(u.dtype)
    if x.shape[1] > x.shape[2]:
        x = x.transpose(1, 2).contiguous()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(1, 2).contiguous() if u.shape[1] > u.shape[2] else x


def _plain_orthogonalize(t, c):
    return [_orthogonal(t["grad"])]


def _plain_muon(t, c):
    m, g, p = t["momentum"], t["grad"], t["param"]
    m.copy_(m + (1 - MOMENTUM) * (g - m))
    o = _orthogonal(g + MOMENTUM * (m - g))
    p.copy_(p * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, c["rows"] / c["cols"])) * o)
    return [p, m]


_PLAIN = dict(norm=_plain_norm, linear=_plain_linear, orthogonalize=_plain_orthogonalize, muon=_plain_muon)


def _mx():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from torch_vulkan import mx
    return mx


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_norm(t, c):
    mx, x = _mx(), t["x"]
    y = torch.empty_like(x)
    if not c["train"]:
        mx.layer_norm_forward(x, t["gamma"], t["beta"], EPS, y, None, None, stream=_stream())
        return [y]
    mean, rstd, dx = x.new_empty(c["rows"]), x.new_empty(c["rows"]), torch.empty_like(x)
    dgamma, dbeta = torch.empty_like(t["gamma"]), torch.empty_like(t["beta"])
    mx.layer_norm_forward(x, t["gamma"], t["beta"], EPS, y, mean, rstd, stream=_stream())
    mx.layer_norm_backward(t["dy"], x, mean, rstd, t["gamma"], dx, dgamma, dbeta, stream=_stream())
    return [y, dx, dgamma, dbeta]


def _own_linear(t, c):
    mx, x, w = _mx(), t["x"], t["w"]
    act = mx.ACTIVATIONS[c["act"]]
    y = x.new_empty(c["m"], c["n"])
    if not c["train"]:
        mx.linear_forward(x, w, t["b"], y, activation=act, residual=t["res"], stream=_stream())
        return [y]
    # The layer without an activation keeps no input of one.
    z = None if c["act"] == "none" else torch.empty_like(y)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(t["b"])
    mx.linear_forward(x, w, t["b"], y, activation=act, residual=t["res"], z=z, stream=_stream())
    mx.linear_backward(t["dy"], x, w, z, dx, dw, db, activation=act, stream=_stream())
    return [y, dx, dw, db]


def _own_orthogonalize(t, c):
    out = torch.empty_like(t["grad"])
    _mx().orthogonalize(t["grad"].unbind(0), out.unbind(0), steps=STEPS, coefficients=NS, eps=NS_EPS, stream=_stream())
    return [out]


def _own_muon(t, c):
    _mx().muon_step(t["param"].unbind(0), t["grad"].unbind(0), t["momentum"].unbind(0), lr=LR, weight_decay=DECAY,
                    momentum=MOMENTUM, nesterov=True, steps=STEPS, coefficients=NS, eps=NS_EPS, adjust_lr="original",
                    stream=_stream())
    return [t["param"], t["momentum"]]


_OWN = dict(norm=_own_norm, linear=_own_linear, orthogonalize=_own_orthogonalize, muon=_own_muon)


# ------------------------------------------------------------ in 64 bits
def exact(case, seed):
    t = {k: None if v is None else v.double() for k, v in _inputs(case, seed).items()}
    c = case
    if c["kind"] == "norm":
        leaves = [t["x"].requires_grad_(), t["gamma"].requires_grad_(), t["beta"].requires_grad_()]
        var, mean = torch.var_mean(t["x"], 1, correction=0, keepdim=True)
        y = (t["x"] - mean) / torch.sqrt(var + EPS) * t["gamma"] + t["beta"]
        return [y.detach()] + (list(torch.autograd.grad(y, leaves, t["dy"])) if c["train"] else [])
    if c["kind"] == "linear":
        f = torch.nn.functional
        acts = dict(none=lambda v: v, relu=f.relu, silu=f.silu, gelu=f.gelu,
                    gelu_tanh=lambda v: f.gelu(v, approximate="tanh"))
        leaves = [t["x"].requires_grad_(), t["w"].requires_grad_(), t["b"].requires_grad_()]
        y = acts[c["act"]](torch.addmm(t["b"], t["x"], t["w"].t()))
        if c["residual"]:
            y = y + t["res"]
        return [y.detach()] + (list(torch.autograd.grad(y, leaves, t["dy"])) if c["train"] else [])
    # The iteration acts on singular values alone, p(s) = a s + b s^3 + c s^5:
    # its matrix form in float64, one matrix of the stack at a time.
    def orthogonal(u):
        x = u / max(float(torch.linalg.matrix_norm(u)), NS_EPS)
        small = x @ x.t() if x.shape[0] <= x.shape[1] else x.t() @ x
        eye = torch.eye(small.shape[0], dtype=torch.float64, device=u.device)
        total = eye
        for _ in range(STEPS):
            # X <- q(X X^T) X keeps X = T X0 with T a polynomial of the first Gram matrix.
            q = NS[0] * eye + NS[1] * small + NS[2] * (small @ small)
            total, small = q @ total, q @ small @ q
        return total @ x if x.shape[0] <= x.shape[1] else x @ total

    if c["kind"] == "orthogonalize":
        return [torch.stack([orthogonal(u) for u in t["grad"]])]
    m = MOMENTUM * t["momentum"] + (1 - MOMENTUM) * t["grad"]
    o = torch.stack([orthogonal(u) for u in MOMENTUM * m + (1 - MOMENTUM) * t["grad"]])
    return [(1 - LR * DECAY) * t["param"] - LR * max(1.0, c["rows"] / c["cols"]) ** 0.5 * o, m]


# ------------------------------------------------- bytes and operations
def _ns_flops(rows, cols):
    """Multiply-adds, twice, of the iterations on one matrix: two symmetric
    products, of which one triangle is needed, and a full one."""
    s, l = min(rows, cols), max(rows, cols)
    return STEPS * (1.0 * s * s * l + 1.0 * s * s * s + 2.0 * s * s * l)


def work(case):
    c = case
    if c["kind"] == "norm":
        e = c["rows"] * c["cols"]
        # Forward reads x and writes y; the backward reads x and dy again and writes dx.
        return dict(bytes=4.0 * ((5 if c["train"] else 2) * e + (4 if c["train"] else 2) * c["cols"]),
                    flops=(20.0 if c["train"] else 8.0) * e)
    if c["kind"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        once = m * k + n * k + n + m * n * (2 if c["residual"] else 1)
        return dict(bytes=4.0 * (once + (m * n + m * k + n * k + n if c["train"] else 0)),
                    flops=2.0 * m * n * k * (3 if c["train"] else 1))
    e = c["count"] * c["rows"] * c["cols"]
    return dict(bytes=4.0 * (5 if c["kind"] == "muon" else 2) * e, flops=c["count"] * _ns_flops(c["rows"], c["cols"]))
