"""torch_vulkan.nn and torch_vulkan.optim around the device's operators, which are
replaced by CPU stand-ins: what they are asked for, no GPU calls."""
import pytest
import torch
import torch.nn.functional as F


@pytest.fixture
def calls(monkeypatch):
    """The arguments of every linear_act call, computed on the CPU."""
    import torch_vulkan  # noqa: F401  (registers the operators)
    seen = []

    def linear_act(x, weight, bias, residual, activation, keep_z):
        seen.append(dict(activation=activation, keep_z=keep_z))
        z = F.linear(x, weight, bias)
        y = F.gelu(z) if activation == "gelu" else z
        return y if residual is None else y + residual, z if keep_z else x.new_empty(0)

    monkeypatch.setattr(torch.ops.torch_vulkan, "linear_act", linear_act)
    return seen


def test_linear_keeps_the_activations_input_only_for_a_gradient(calls):
    from torch_vulkan.nn import Linear, linear
    layer, x = Linear(6, 5, activation="gelu"), torch.randn(3, 6)
    kept = lambda: [c["keep_z"] for c in calls]
    with torch.no_grad():
        layer(x)
        layer(x, residual=torch.randn(3, 5))
    with torch.inference_mode():
        layer(x)
    assert kept() == [False] * 3, "serving stores no z"
    calls.clear()
    layer(x)
    layer(x.clone().requires_grad_())
    linear(x.clone().requires_grad_(), layer.weight.detach(), None, "gelu")
    linear(x, layer.weight.detach(), layer.bias, "gelu")
    with torch.no_grad(), torch.enable_grad():
        layer(x)
    assert kept() == [True] * 5, "a gradient asks for z"
    calls.clear()
    linear(x, layer.weight.detach(), None, "gelu", torch.randn(3, 5, requires_grad=True))
    linear(x, layer.weight.detach(), None, "gelu")
    linear(x, layer.weight, layer.bias, "none")
    assert kept() == [False] * 3, "the residual's gradient and a layer without an activation do not"
    assert torch.allclose(layer(x), F.gelu(F.linear(x, layer.weight, layer.bias)))
