"""Refusals and workspace sizes of layer norm, the linear layer and the
orthogonalised momentum step: host validation, no GPU calls."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def mx():
    from torch_vulkan import mx as m
    m.lib()
    return m


FAKE = 4096  # an address that no refused call reads


def refused(mx, call, *args):
    with pytest.raises(mx.MXError) as e:
        mx.check(getattr(mx.lib(), call)(*args))
    return e.value


def test_layer_norm_refusals(mx):
    f = "mx_layer_norm_forward"
    assert refused(mx, f, FAKE, None, None, -1, 4, 1e-5, FAKE, None, None, None).status == mx.MX_ERR_INVALID
    assert "empty rows" in str(refused(mx, f, FAKE, None, None, 2, 0, 1e-5, FAKE, None, None, None))
    assert "null buffer" in str(refused(mx, f, None, None, None, 2, 4, 1e-5, FAKE, None, None, None))
    assert "out of range" in str(refused(mx, f, FAKE, None, None, 2, 1 << 31, 1e-5, FAKE, None, None, None))
    assert "out of range" in str(refused(mx, f, FAKE, None, None, 1 << 59, 16, 1e-5, FAKE, None, None, None))
    b = "mx_layer_norm_backward"
    assert "null buffer" in str(refused(mx, b, None, FAKE, FAKE, FAKE, None, 2, 4, FAKE, None, None, None, 0, None))
    assert refused(mx, b, FAKE, FAKE, FAKE, FAKE, None, -2, 4, FAKE, None, None, None, 0, None).status == mx.MX_ERR_INVALID
    # no rows, nothing to write, nothing asked for: no error, no launch
    mx.check(mx.lib().mx_layer_norm_forward(None, None, None, 0, 4, 1e-5, None, None, None, None))
    mx.check(mx.lib().mx_layer_norm_backward(None, None, None, None, None, 3, 4, None, None, None, None, 0, None))


def test_layer_norm_workspace_too_small_or_misaligned(mx):
    need = mx.layer_norm_backward_workspace(1 << 16, 1024)
    assert need > 0 and mx.layer_norm_backward_workspace(1, 1024) == 0 and mx.layer_norm_backward_workspace(0, 1024) == 0
    args = (FAKE, FAKE, FAKE, FAKE, None, 1 << 16, 1024, FAKE, FAKE, FAKE)
    e = refused(mx, "mx_layer_norm_backward", *args, FAKE, need - 1, None)
    assert e.status == mx.MX_ERR_WORKSPACE and str(need) in str(e)
    assert "aligned" in str(refused(mx, "mx_layer_norm_backward", *args, FAKE + 4, need, None))


def test_linear_refusals(mx):
    f = "mx_linear_forward"
    assert "negative" in str(refused(mx, f, FAKE, FAKE, None, None, 2, -1, 4, 0, FAKE, None, None, 0, None))
    assert "int32" in str(refused(mx, f, FAKE, FAKE, None, None, 1 << 32, 1, 4, 0, FAKE, None, None, 0, None))
    for act in (-1, 5):
        assert "unknown activation" in str(refused(mx, f, FAKE, FAKE, None, None, 2, 3, 4, act, FAKE, None, None, 0, None))
    for x, w, y in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None)):
        assert "null buffer" in str(refused(mx, f, x, w, None, None, 2, 3, 4, 0, y, None, None, 0, None))
    b = "mx_linear_backward"
    assert "null buffer" in str(refused(mx, b, FAKE, FAKE, FAKE, None, 2, 3, 4, mx.ACT_GELU, FAKE, FAKE, FAKE, None, 0, None))
    assert "null buffer" in str(refused(mx, b, FAKE, None, FAKE, None, 2, 3, 4, 0, None, FAKE, None, None, 0, None))
    assert "null buffer" in str(refused(mx, b, FAKE, FAKE, None, None, 2, 3, 4, 0, FAKE, None, None, None, 0, None))
    need = mx.linear_workspace(512, 256, 1024, mx.ACT_GELU, True)
    e = refused(mx, b, FAKE, FAKE, FAKE, FAKE, 512, 256, 1024, mx.ACT_GELU, FAKE, FAKE, FAKE, FAKE, need - 1, None)
    assert e.status == mx.MX_ERR_WORKSPACE
    mx.check(mx.lib().mx_linear_forward(None, None, None, None, 0, 3, 4, 0, None, None, None, 0, None))
    assert mx.linear_workspace(0, 3, 4) == 0 and mx.linear_workspace(0, 3, 4, 0, True) == 0


def ns(mx, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7):
    return mx.NewtonSchulz(steps, a, b, c, eps)


def test_orthogonalize_refusals(mx):
    pair = (mx.MatrixPair * 2)(mx.MatrixPair(FAKE, FAKE, 8, 9), mx.MatrixPair(FAKE, FAKE, 8, 9))
    call = lambda n, p, arr=pair: refused(mx, "mx_orthogonalize", arr, n, C.byref(p), None, 0, None)
    assert "negative count" in str(call(-1, ns(mx)))
    assert "null list" in str(call(1, ns(mx), None))
    assert "steps" in str(call(1, ns(mx, steps=-1))) and "steps" in str(call(1, ns(mx, steps=1001)))
    assert "finite" in str(call(1, ns(mx, a=float("nan")))) and "eps" in str(call(1, ns(mx, eps=0.0)))
    assert "diverge" in str(call(1, ns(mx, a=100.0, steps=20)))
    for bad in (mx.MatrixPair(None, FAKE, 8, 9), mx.MatrixPair(FAKE, None, 8, 9)):
        assert "null buffer at 0" in str(call(1, ns(mx), (mx.MatrixPair * 1)(bad)))
    assert "negative size" in str(call(1, ns(mx), (mx.MatrixPair * 1)(mx.MatrixPair(FAKE, FAKE, -8, 9))))
    assert "longer" in str(call(1, ns(mx), (mx.MatrixPair * 1)(mx.MatrixPair(FAKE, FAKE, 8, (1 << 24) + 1))))
    need = C.c_int64()
    mx.check(mx.lib().mx_orthogonalize_workspace(pair, 2, C.byref(need)))
    assert need.value > 0
    e = refused(mx, "mx_orthogonalize", pair, 2, C.byref(ns(mx)), FAKE, need.value - 1, None)
    assert e.status == mx.MX_ERR_WORKSPACE
    mx.check(mx.lib().mx_orthogonalize(None, 0, C.byref(ns(mx)), None, 0, None))


def test_muon_refusals(mx):
    row = mx.MuonTensor(FAKE, FAKE, FAKE, 8, 9)
    arr = (mx.MuonTensor * 1)(row)

    def hp(lr=0.02, wd=0.1, mom=0.95, adjust=0):
        return mx.MuonHParams(lr, wd, mom, 1, adjust, ns(mx))

    call = lambda h, a=arr: refused(mx, "mx_muon_step", a, 1, C.byref(h), None, 0, None)
    for h in (hp(lr=-1), hp(wd=-1), hp(mom=-0.1), hp(mom=1.5), hp(lr=float("nan")), hp(lr=float("inf"))):
        assert "invalid hyperparameters" in str(call(h))
    assert "adjustment" in str(call(hp(adjust=2)))
    for bad in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None)):
        assert "null buffer at 0" in str(call(hp(), (mx.MuonTensor * 1)(mx.MuonTensor(*bad, 8, 9))))
    mx.check(mx.lib().mx_muon_step(None, 0, C.byref(hp()), None, 0, None))


def test_python_binding_checks_lists_and_shapes(mx):
    a, b = torch.empty(3, 4), torch.empty(4, 3)
    with pytest.raises(ValueError, match="one shape"):
        mx.orthogonalize([a], [b])
    with pytest.raises(ValueError, match="1 inputs, 2 outputs"):
        mx.orthogonalize([a], [a, a])
    with pytest.raises(ValueError, match="one shape"):
        mx.muon_step([a], [b], [a])
    with pytest.raises(ValueError, match="differ in length"):
        mx.muon_step([a], [a, a], [a])
    with pytest.raises(ValueError, match="adjust_lr"):
        mx.muon_step([a], [a], [a], adjust_lr="other")
