"""LayerNorm, torch_vulkan.nn.linear, optim.Muon and the feed-forward example on
the "vulkan" device against CPU torch, with the CPU fallback forbidden.

Parity bar: |err| <= 1e-4 |ref| + 1e-5 max(1, magnitude) against float64, the
bar of the other operators on this device (tests/helpers.py)."""
import copy
import importlib.util
import math
import os

import pytest
import torch
import torch.nn.functional as F

from helpers import assert_close_mag

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module", autouse=True)
def vk():
    import torch_vulkan
    assert torch_vulkan.is_available(), "no gfx950 device visible"
    return torch_vulkan


@pytest.fixture(autouse=True)
def no_fallback(vk, monkeypatch):
    monkeypatch.setenv("TORCH_VULKAN_FORBID_CPU_FALLBACK", "1")
    before = vk.execution_stats()["cpu_fallback_calls"]
    yield
    assert vk.execution_stats()["cpu_fallback_calls"] == before


@pytest.mark.parametrize("shape,norm,affine", [((5, 70), (70,), True), ((2, 3, 129), (129,), True), ((4, 6, 10), (6, 10), True),
                                               ((7, 33), (33,), False), ((3, 1), (1,), True), ((0, 8), (8,), True)])
def test_layer_norm_module(shape, norm, affine):
    g = torch.Generator().manual_seed(len(shape) + norm[0])
    x, dy = torch.randn(shape, generator=g), torch.randn(shape, generator=g)
    m = torch.nn.LayerNorm(norm, elementwise_affine=affine)
    if affine:
        with torch.no_grad():
            m.weight.copy_(torch.randn(norm, generator=g))
            m.bias.copy_(torch.randn(norm, generator=g))
    ref = torch.nn.LayerNorm(norm, elementwise_affine=affine).double()
    ref.load_state_dict({k: v.double() for k, v in m.state_dict().items()})
    xr = x.double().requires_grad_()
    yr = ref(xr)
    yr.backward(dy.double())
    m = m.to("vulkan")
    xv = x.to("vulkan").requires_grad_()
    yv = m(xv)
    yv.backward(dy.to("vulkan"))
    assert_close_mag(yv, yr, what="y")
    assert_close_mag(xv.grad, xr.grad, what="dx")
    if affine:
        mag = dy.double().abs().sum(tuple(range(len(shape) - len(norm)))) * 4 if x.numel() else None
        assert_close_mag(m.weight.grad, ref.weight.grad, mag, what="dgamma")
        assert_close_mag(m.bias.grad, ref.bias.grad, mag, what="dbeta")


def test_layer_norm_strided_input():
    x = torch.randn(40, 9, generator=torch.Generator().manual_seed(0)).to("vulkan").t()
    assert_close_mag(F.layer_norm(x, (40,)), F.layer_norm(x.cpu().double(), (40,)))


@pytest.mark.parametrize("lead", [(), (3,), (4, 5)])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_linear_function(lead, act):
    from torch_vulkan.nn import linear
    g = torch.Generator().manual_seed(len(lead))
    k, n = 37, 50
    acts = dict(none=lambda v: v, relu=F.relu, silu=F.silu, gelu=F.gelu, gelu_tanh=lambda v: F.gelu(v, approximate="tanh"))
    leaves = [torch.randn(*lead, k, generator=g), torch.randn(n, k, generator=g) / 6, torch.randn(n, generator=g),
              torch.randn(*lead, n, generator=g)]
    dy = torch.randn(*lead, n, generator=g)
    r = [t.double().requires_grad_() for t in leaves]
    v = [t.to("vulkan").requires_grad_() for t in leaves]
    yr = acts[act](F.linear(r[0], r[1], r[2])) + r[3]
    yv = linear(v[0], v[1], v[2], act, v[3])
    assert yv.shape == yr.shape
    assert_close_mag(yv, yr, what="y")
    gr = torch.autograd.grad(yr, r, dy.double())
    gv = torch.autograd.grad(yv, v, dy.to("vulkan"))
    for name, a, b in zip(("dx", "dw", "db", "dres"), gv, gr):
        assert_close_mag(a, b, b.abs() + 8, what=name)


def test_linear_broadcast_residual_and_partial_gradients():
    from torch_vulkan.nn import linear
    g = torch.Generator().manual_seed(5)
    x, w, res = torch.randn(6, 9, generator=g), torch.randn(4, 9, generator=g), torch.randn(4, generator=g)
    rv = res.to("vulkan").requires_grad_()
    wv = w.to("vulkan").requires_grad_()
    y = linear(x.to("vulkan"), wv, None, "silu", rv)
    y.backward(torch.ones(6, 4).to("vulkan"))
    wr, rr = w.double().requires_grad_(), res.double().requires_grad_()
    (F.silu(x.double() @ wr.t()) + rr).sum().backward()
    assert_close_mag(rv.grad, rr.grad)
    assert_close_mag(wv.grad, wr.grad, wr.grad.abs() + 8)


def test_refusals():
    from torch_vulkan.nn import Linear, linear
    from torch_vulkan.optim import Muon
    x, w = torch.zeros(2, 3).to("vulkan"), torch.zeros(4, 3).to("vulkan")
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="does not fit"):
        linear(x, torch.zeros(4, 5).to("vulkan"))
    with pytest.raises(RuntimeError, match="bias has shape"):
        linear(x, w, torch.zeros(3).to("vulkan"))
    with pytest.raises(RuntimeError, match="float32"):
        linear(x, torch.zeros(4, 3, dtype=torch.float64).to("vulkan"))
    with pytest.raises(ValueError, match="activation"):
        Linear(3, 4, activation="x")
    with pytest.raises(ValueError, match="only matrices"):
        Muon([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError, match="lr"):
        Muon([torch.nn.Parameter(torch.zeros(3, 3))], lr=-1)
    ops = torch.ops.torch_vulkan
    with pytest.raises(RuntimeError, match="appears twice"):
        ops.muon_step_([w, w], [w, w], [torch.zeros_like(w), torch.zeros_like(w)], 0.1, 0.0, 0.9, True, [1.0, 0.0, 0.0], 1,
                       1e-7, "original")
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.muon_step_([w.t()], [w.t()], [w.t()], 0.1, 0.0, 0.9, True, [1.0, 0.0, 0.0], 1, 1e-7, "original")
    with pytest.raises(RuntimeError, match="three coefficients"):
        ops.orthogonalize([w], [1.0, 2.0], 1, 1e-7)


def reference_muon(p, g, m, lr, wd, mu, nesterov, adjust):
    a, b, c = 3.4445, -4.7750, 2.0315
    m += (1 - mu) * (g - m)
    u = g + mu * (m - g) if nesterov else m
    x = u / max(float(u.norm()), 1e-7)
    x = x.t() if u.shape[0] > u.shape[1] else x
    for _ in range(5):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    x = x.t() if u.shape[0] > u.shape[1] else x
    r = math.sqrt(max(1, u.shape[0] / u.shape[1])) if adjust != "match_rms_adamw" else 0.2 * math.sqrt(max(u.shape))
    p *= 1 - lr * wd
    p -= lr * r * x


@pytest.mark.parametrize("adjust", [None, "match_rms_adamw"])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_trajectory_and_checkpoint(adjust, nesterov):
    from torch_vulkan.optim import Muon
    g = torch.Generator().manual_seed(9)
    shapes = [(20, 33), (33, 20), (20, 33), (64, 64), (1, 7)]
    first = [torch.randn(s, generator=g) for s in shapes]
    dev = [torch.nn.Parameter(p.to("vulkan")) for p in first]
    ref = [p.double() for p in first]
    mom = [torch.zeros_like(p) for p in ref]
    opts = dict(lr=0.05, weight_decay=0.1, momentum=0.9, nesterov=nesterov, adjust_lr_fn=adjust)
    opt = Muon(dev, **opts)
    twin = None
    for step in range(4):
        grads = [torch.randn(s, generator=g) for s in shapes]
        for i, (p, gr) in enumerate(zip(dev, grads)):
            p.grad = None if (step + i) % 4 == 3 else gr.to("vulkan")
            if p.grad is not None:
                reference_muon(ref[i], gr.double(), mom[i], 0.05, 0.1, 0.9, nesterov, adjust)
        if step == 2:  # a restored optimizer goes on bit for bit
            copies = [torch.nn.Parameter(p.detach().clone()) for p in dev]
            twin = Muon(copies, **opts)
            twin.load_state_dict(copy.deepcopy(opt.state_dict()))
        opt.step()
        if twin is not None:
            for c, p in zip(copies, dev):
                c.grad = p.grad
            twin.step()
            for c, p in zip(copies, dev):
                assert torch.equal(c.detach().cpu(), p.detach().cpu())
    for p, r in zip(dev, ref):
        assert_close_mag(p, r, what=f"{tuple(p.shape)}")


def test_feed_forward_example_follows_the_cpu(vk):
    spec = importlib.util.spec_from_file_location("feed_forward", os.path.join(REPO, "pytorch-vulkan_amd", "examples", "feed_forward.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    width, hidden, tokens = 48, 100, 96
    model = ex.build(width, hidden, 2, seed=3)
    params = {k: v.detach().double().requires_grad_() for k, v in model.named_parameters()}
    g = torch.Generator().manual_seed(4)
    x, target = torch.randn(tokens, width, generator=g), torch.randn(tokens, width, generator=g)
    losses = ex.train(model.to("vulkan"), x.to("vulkan"), target.to("vulkan"), 3)
    mom = {k: torch.zeros_like(v) for k, v in params.items()}
    opt = torch.optim.AdamW([v for v in params.values() if v.dim() != 2], lr=0.002, weight_decay=0.0)
    want = []
    for _ in range(3):
        h = x.double()
        for i in range(2):
            q = lambda n: params[f"{i}.{n}"]
            z = F.gelu(F.linear(F.layer_norm(h, (width,), q("norm.weight"), q("norm.bias")), q("up.weight"), q("up.bias")))
            h = F.linear(z, q("down.weight"), q("down.bias")) + h
        loss = F.mse_loss(h, target.double())
        want.append(float(loss.detach()))
        for v in params.values():
            v.grad = None
        loss.backward()
        with torch.no_grad():
            for k, v in params.items():
                if v.dim() == 2:
                    reference_muon(v, v.grad, mom[k], 0.02, 0.0, 0.95, True, None)
        opt.step()
    assert losses == pytest.approx(want, rel=1e-4)
    assert losses[-1] < losses[0]
