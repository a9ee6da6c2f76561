"""GPU parity of layer norm, the linear layer with its epilogue, and the
orthogonalised momentum step (C ABI on torch's GPU tensors) against float64.

Bounds come from the operations' roundings, u = 2^-24 (half a step of FP32
relative to a value):
  * a sum of n terms in a tree or in lanes of at most d sequential terms is off
    by d u of the sum of magnitudes; a row here is summed in at most 40;
  * a product over k of operands without bits left out is off by at most
    (k / 8 + 8) u of the sum of the terms' magnitudes (8 of a term's roundings
    and its dropped pieces, one rounding of the sum every 8 terms or more);
  * the activations and their slopes are Lipschitz with 1.13 and 1.6 and
    evaluated within 16 u (|z| + 1).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NS = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def mx():
    from torch_vulkan import mx as m
    m.lib()
    return m


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, scale=1.0, mean=0.0):
    return torch.randn(*shape, device="cuda", generator=g) * scale + mean


def guarded(*shape):
    """A tensor whose storage goes on behind it (checked by intact())."""
    n = math.prod(shape)
    flat = torch.full((n + 64,), 12345.0, device="cuda")
    return flat[:n].view(*shape), flat[n:]


def intact(*tails):
    for t in tails:
        assert bool((t == 12345.0).all()), "wrote past the end of an output"


def within(got, ref, bound, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())}/{bad.numel()} outside; worst err/bound {float((err / bound).nan_to_num(1e30).max()):.3g}")


# ---------------------------------------------------------------- layer norm
LN_SHAPES = [(1, 1), (3, 2), (2, 3), (1, 4), (5, 5), (7, 64), (33, 63), (65, 65), (17, 127), (9, 128), (40, 131), (21, 255),
             (12, 257), (6, 511), (13, 512), (5, 515), (3, 1023), (1, 1024), (700, 1024), (4, 1025), (3, 1447), (2, 2049),
             (600, 2048), (5, 4095), (3, 4097), (2, 8191), (3, 8200), (2, 16384), (2, 16389), (1, 40001), (3000, 36)]


def ln_ref(x, gamma, beta, eps):
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    xhat = d * rstd
    y = xhat * (gamma if gamma is not None else 1) + (beta if beta is not None else 0)
    return y, mean, rstd, xhat


@pytest.mark.parametrize("rows,cols", LN_SHAPES)
@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm(mx, rows, cols, affine):
    print("layer norm", rows, cols, affine, flush=True)
    g = gen(rows * 7 + cols)
    x = rand(g, rows, cols) * (rand(g, rows, 1).abs() + 0.2) + rand(g, rows, 1)
    gamma, beta = (rand(g, cols, mean=1.0, scale=0.3), rand(g, cols)) if affine else (None, None)
    dy = rand(g, rows, cols)
    (y, t0), (mean, t1), (rstd, t2) = guarded(rows, cols), guarded(rows), guarded(rows)
    mx.layer_norm_forward(x, gamma, beta, 1e-5, y, mean, rstd, stream=stream())
    xd, gd = x.double(), gamma.double() if affine else torch.ones(cols, device="cuda", dtype=torch.double)
    yr, mr, rr, xh = ln_ref(xd, gd, beta.double() if affine else None, 1e-5)
    mag = xd.abs().mean(1, keepdim=True)
    # var is off by 2 x 40 u of itself (and the mean's error squared), rstd by half of that
    hat_err = 40 * U * (rr * mag + xh.abs()) + 8 * U
    within(y, yr, hat_err * gd.abs() + 4 * U * (yr.abs() + (beta.double().abs() if affine else 0)), "y")
    within(mean, mr[:, 0], (41 * U * mag + 1e-30)[:, 0], "mean")
    within(rstd, rr[:, 0], (50 * U * rr * (1 + (rr * mag) ** 2 * 40 * U))[:, 0], "rstd")
    (dx, t3), (dg, t4), (db, t5) = guarded(rows, cols), guarded(cols), guarded(cols)
    mx.layer_norm_backward(dy, x, mean, rstd, gamma, dx, dg, db, stream=stream())
    gr = dy.double() * gd
    a, b = gr.mean(1, keepdim=True), (gr * xh).mean(1, keepdim=True)
    ma, mb = gr.abs().mean(1, keepdim=True), (gr * xh).abs().mean(1, keepdim=True)
    dxr = rr * (gr - a - xh * b)
    dx_bound = rr * (60 * U * (gr.abs() + ma + xh.abs() * mb) + hat_err * mb + xh.abs() * (hat_err * gr.abs()).mean(1, keepdim=True))
    within(dx, dxr, dx_bound + 1e-30, "dx")
    dyd = dy.double()
    deep = 64 + rows / 64
    within(dg, (dyd * xh).sum(0), (deep * U * (dyd * xh).abs() + dyd.abs() * hat_err).sum(0) + 1e-30, "dgamma")
    within(db, dyd.sum(0), deep * U * dyd.abs().sum(0) + 1e-30, "dbeta")
    intact(t0, t1, t2, t3, t4, t5)
    # Statistics left out, single gradients, and the same bits on a second call.
    y2, dx2, dg2, db2 = torch.empty_like(y), torch.empty_like(dx), torch.empty_like(dg), torch.empty_like(db)
    mx.layer_norm_forward(x, gamma, beta, 1e-5, y2, None, None, stream=stream())
    mx.layer_norm_backward(dy, x, mean, rstd, gamma, dx2, None, None, stream=stream())
    mx.layer_norm_backward(dy, x, mean, rstd, gamma, None, dg2, None, stream=stream())
    ws = torch.empty(max(16, mx.layer_norm_backward_workspace(rows, cols)), dtype=torch.uint8, device="cuda")
    mx.layer_norm_backward(dy, x, mean, rstd, gamma, None, None, db2, workspace=ws, stream=stream())
    assert torch.equal(y, y2) and torch.equal(dx, dx2) and torch.equal(dg, dg2) and torch.equal(db, db2)


def test_layer_norm_unaligned_and_in_place(mx):
    g = gen(3)
    flat = rand(g, 1 + 37 * 130)
    x = flat[1:].view(37, 130)
    want = ln_ref(x.double(), None, None, 1e-5)[0]
    mx.layer_norm_forward(x, None, None, 1e-5, x, None, None, stream=stream())
    within(x, want, 100 * U * (want.abs() + 1), "in place, 4-byte aligned")


def test_layer_norm_constant_huge_and_bad_rows(mx):
    x = torch.zeros(6, 300, device="cuda")
    x[0] = 7.0
    x[1] = 1e18 * torch.arange(300, device="cuda")
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] = 1e-30 * torch.arange(300, device="cuda")
    y = torch.empty_like(x)
    mx.layer_norm_forward(x, None, None, 1e-5, y, None, None, stream=stream())
    assert bool((y[0] == 0).all()) and bool((y[5] == 0).all()), "a constant row normalises to zero"
    want = ln_ref(x.double(), None, None, 1e-5)[0]
    within(y[4], want[4], 100 * U * (want[4].abs() + 1e-27), "tiny row")
    assert bool(y[2].isnan().any()) and bool(y[3].isnan().all())
    # (1.5e20)^2 is past FP32: the formula's variance is infinite there, its rstd and the row zero
    assert bool((y[1] == 0).all())


def test_layer_norm_empty(mx):
    x = torch.empty(0, 33, device="cuda")
    dg, db = torch.ones(33, device="cuda"), torch.ones(33, device="cuda")
    mx.layer_norm_forward(x, None, None, 1e-5, x, None, None, stream=stream())
    mx.layer_norm_backward(x, x, x, x, None, x, dg, db, stream=stream())
    assert float(dg.abs().sum()) == 0 and float(db.abs().sum()) == 0


def test_layer_norm_backward_against_differences(mx):
    g = gen(11)
    x, gamma, beta, dy = rand(g, 9, 70), rand(g, 70, mean=1.0), rand(g, 70), rand(g, 9, 70)
    y, mean, rstd = torch.empty_like(x), torch.empty(9, device="cuda"), torch.empty(9, device="cuda")
    dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
    mx.layer_norm_forward(x, gamma, beta, 1e-5, y, mean, rstd, stream=stream())
    mx.layer_norm_backward(dy, x, mean, rstd, gamma, dx, dg, db, stream=stream())
    h = 2.0 ** -7
    for grad, which in ((dx, 0), (dg, 1), (db, 2)):
        d = rand(g, *grad.shape)
        d = d / d.norm()
        loss = []
        for s in (h, -h):
            t = [x, gamma, beta]
            t[which] = t[which] + s * d
            mx.layer_norm_forward(*t, 1e-5, y, None, None, stream=stream())
            loss.append(float((y.double() * dy.double()).sum()))
        diff, exact = (loss[0] - loss[1]) / (2 * h), float((grad.double() * d.double()).sum())
        # a third derivative of order |dy| (unit direction, unit-scale rows) and y's roundings over 2 h
        tol = h * h * float(dy.norm()) + 32 * U * float((y.double() * dy.double()).abs().sum()) / (2 * h)
        assert abs(diff - exact) <= tol, (which, diff, exact, tol)


# -------------------------------------------------------------------- linear
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
F = torch.nn.functional
ACT64 = dict(none=lambda v: v * 1, relu=F.relu, silu=F.silu, gelu=F.gelu, gelu_tanh=lambda v: F.gelu(v, approximate="tanh"))
LINEAR_SHAPES = [(1, 1, 1), (1, 64, 3), (2, 3, 5), (3, 65, 4), (4, 1024, 512), (1, 513, 1000), (8, 100, 70), (13, 40, 64),
                 (17, 33, 129), (64, 64, 64), (65, 63, 66), (130, 257, 131), (200, 128, 300), (257, 512, 260), (31, 2050, 9),
                 (1030, 70, 258), (515, 765, 1026), (600, 1028, 515), (1, 4096, 4096)]


def linear_ref(x, w, b, res, act):
    z = x @ w.t()
    if b is not None:
        z = z + b
    y = ACT64[act](z)
    return z, y if res is None else y + res


@pytest.mark.parametrize("m,k,n", LINEAR_SHAPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear(mx, m, k, n, act):
    print("linear", m, k, n, act, flush=True)
    g = gen(m + 3 * k + 5 * n)
    x, w = rand(g, m, k), rand(g, n, k, scale=k ** -0.5)
    b = rand(g, n, scale=0.3) if (m + n) % 3 else None
    res = rand(g, m, n) if (m + k) % 2 else None
    dy = rand(g, m, n)
    code = mx.ACTIVATIONS[act]
    (y, t0), (z, t1) = guarded(m, n), guarded(m, n)
    mx.linear_forward(x, w, b, y, activation=code, residual=res, z=z, stream=stream())
    d = lambda t: None if t is None else t.double()
    zr, yr = linear_ref(d(x), d(w), d(b), d(res), act)
    mag = d(x).abs() @ d(w).abs().t() + (d(b).abs() if b is not None else 0)
    z_err = (k / 8 + 8) * U * mag
    within(z, zr, z_err, "z")
    within(y, yr, 1.13 * z_err + 16 * U * (zr.abs() + 1) + 4 * U * yr.abs(), "y")
    y2 = torch.empty_like(y)
    mx.linear_forward(x, w, b, y2, activation=code, residual=res, stream=stream())
    assert torch.equal(y, y2)
    if res is not None:  # the output may be the residual's buffer
        into = res.clone()
        mx.linear_forward(x, w, b, into, activation=code, residual=into, stream=stream())
        assert torch.equal(y, into)
    (dx, t2), (dw, t3), (db, t4) = guarded(m, k), guarded(n, k), guarded(n)
    mx.linear_backward(dy, x, w, None if act == "none" else z, dx, dw, db, activation=code, stream=stream())
    zl = d(z).cpu().requires_grad_()
    dz = torch.autograd.grad(ACT64[act](zl), zl, d(dy).cpu())[0].cuda()
    dz_err = 16 * U * d(dy).abs() * (d(z).abs() + 1)
    within(dx, dz @ d(w), ((n / 8 + 8) * U * dz.abs() + dz_err) @ d(w).abs() + 1e-30, "dx")
    within(dw, dz.t() @ d(x), ((m / 8 + 8) * U * dz.abs() + dz_err).t() @ d(x).abs() + 1e-30, "dw")
    within(db, dz.sum(0), ((m / 64 + 64) * U * dz.abs() + dz_err).sum(0) + 1e-30, "db")
    intact(t0, t1, t2, t3, t4)
    # One gradient at a time, with a caller's workspace.
    ws = torch.empty(max(16, mx.linear_workspace(m, k, n, code, True)), dtype=torch.uint8, device="cuda")
    for name, want in (("dx", dx), ("dw", dw), ("db", db)):
        one = {"dx": None, "dw": None, "db": None}
        one[name] = torch.empty_like(want)
        mx.linear_backward(dy, x, w, None if act == "none" else z, one["dx"], one["dw"], one["db"], activation=code,
                           workspace=ws, stream=stream())
        assert torch.equal(one[name], want), name


@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 70), (300, 64, 64), (515, 765, 1026), (2048, 1024, 2048), (3001, 1500, 1501), (20000, 16, 20)])
def test_linear_bias_gradient_alone(mx, m, k, n, act):
    print("linear db alone", m, k, n, act, flush=True)
    g = gen(m + n)
    x, w, z, dy = rand(g, m, k), rand(g, n, k), rand(g, m, n), rand(g, m, n)
    z = None if act == "none" else z
    dx, dw, db, alone = torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    mx.linear_backward(dy, x, w, z, dx, dw, db, activation=mx.ACTIVATIONS[act], stream=stream())
    mx.linear_backward(dy, x, w, z, None, None, alone, activation=mx.ACTIVATIONS[act], stream=stream())
    assert torch.equal(db, alone)


@pytest.mark.parametrize("k,n", [(4, 1), (5, 3), (64, 200), (255, 129), (1023, 61), (1100, 1003), (4096, 40)])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 13, 16, 17, 31, 33, 64])
def test_linear_few_tokens(mx, m, k, n):
    print("few tokens", m, k, n, flush=True)
    g = gen(m * 7 + k + n)
    x, w, b, res = rand(g, m, k), rand(g, n, k, scale=k ** -0.5), rand(g, n, scale=0.3), rand(g, m, n)
    (y, t0), (z, t1) = guarded(m, n), guarded(m, n)
    mx.linear_forward(x, w, b, y, activation=mx.ACT_GELU, residual=res, z=z, stream=stream())
    d = lambda t: t.double()
    zr, yr = linear_ref(d(x), d(w), d(b), d(res), "gelu")
    z_err = (k / 8 + 8) * U * (d(x).abs() @ d(w).abs().t() + d(b).abs())
    within(z, zr, z_err, "z")
    within(y, yr, 1.13 * z_err + 16 * U * (zr.abs() + 1) + 4 * U * yr.abs(), "y")
    intact(t0, t1)


def test_linear_rows_of_any_magnitude(mx):
    """Rows, columns and channels far apart in size keep FP32's accuracy each."""
    g = gen(8)
    m, k, n = 300, 520, 260
    x = rand(g, m, k) * torch.exp2(torch.linspace(-60, 60, m, device="cuda"))[:, None]
    w = rand(g, n, k) * torch.exp2(torch.linspace(40, -40, n, device="cuda"))[:, None]
    y = torch.empty(m, n, device="cuda")
    mx.linear_forward(x, w, None, y, stream=stream())
    mag = x.double().abs() @ w.double().abs().t()
    within(y, x.double() @ w.double().t(), (k / 8 + 8) * U * mag, "y")
    dy = rand(g, m, n) * torch.exp2(torch.linspace(-30, 30, n, device="cuda"))
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda")
    mx.linear_backward(dy, x, w, None, dx, dw, db, stream=stream())
    within(dx, dy.double() @ w.double(), (n / 8 + 8) * U * (dy.double().abs() @ w.double().abs()), "dx")
    within(dw, dy.double().t() @ x.double(), (m / 8 + 8) * U * (dy.double().abs().t() @ x.double().abs()), "dw")


@pytest.mark.parametrize("m,k,n", [(3, 70, 40), (200, 256, 300)])
def test_linear_special_values(mx, m, k, n):
    g = gen(5)
    x, w, b = rand(g, m, k), rand(g, n, k), rand(g, n)
    x[0, 3], x[1, 1], w[2, 0] = float("inf"), float("nan"), 1e38
    x[2, 0] = 100.0
    y = torch.empty(m, n, device="cuda")
    mx.linear_forward(x, w, b, y, activation=mx.ACT_RELU, stream=stream())
    ref = F.relu(x.cpu() @ w.cpu().t() + b.cpu())
    got = y.cpu()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isposinf(), ref.isposinf())


def test_linear_empty(mx):
    e = lambda *s: torch.ones(*s, device="cuda")
    y, z = e(3, 4), e(3, 4)
    mx.linear_forward(e(3, 0), e(4, 0), 2 * e(4), y, activation=mx.ACT_RELU, residual=e(3, 4), z=z, stream=stream())
    assert bool((y == 3).all()) and bool((z == 2).all())
    dw, db, dx = e(4, 5), e(4), e(0, 5)
    mx.linear_backward(e(0, 4), e(0, 5), e(4, 5), None, dx, dw, db, stream=stream())
    assert float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0


def test_linear_backward_against_differences(mx):
    g = gen(21)
    m, k, n = 6, 20, 9
    for act in ACTS[2:]:
        code = mx.ACTIVATIONS[act]
        x, w, b, dy = rand(g, m, k), rand(g, n, k, scale=0.3), rand(g, n), rand(g, m, n)
        y, z = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
        mx.linear_forward(x, w, b, y, activation=code, z=z, stream=stream())
        grads = [torch.empty_like(t) for t in (x, w, b)]
        mx.linear_backward(dy, x, w, z, *grads, activation=code, stream=stream())
        h = 2.0 ** -6
        for i, grad in enumerate(grads):
            d = rand(g, *grad.shape)
            d = d / d.norm()
            loss = []
            for s in (h, -h):
                t = [x, w, b]
                t[i] = t[i] + s * d
                mx.linear_forward(*t, y, activation=code, stream=stream())
                loss.append(float((y.double() * dy.double()).sum()))
            diff, exact = (loss[0] - loss[1]) / (2 * h), float((grad.double() * d.double()).sum())
            # The activations' third derivatives are below 2; a unit direction moves z by |x| or |w| at most.
            reach = max(float(x.norm(dim=1).max()), float(w.norm(dim=1).max()), 1.0)
            tol = h * h / 6 * 2 * reach ** 3 * float(dy.abs().sum()) + 64 * U * float(dy.abs().sum()) * 4 / (2 * h)
            assert abs(diff - exact) <= tol, (act, i, diff, exact, tol)


# ---------------------------------------------------- orthogonalised momentum
def orth(u, steps=5, coef=NS, eps=1e-7):
    a, b, c = coef
    x = u / u.norm().clamp_min(eps)
    if u.shape[0] > u.shape[1]:
        x = x.t()
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


# An iteration multiplies an error in X by at most 3.9 (the polynomial's largest
# divided difference), so one of 2^-21 of |X| in each of five (operands of 23
# bits, 2^-22 of dropped pieces, FP32 sums) ends below 310 x 2^-21.
ORTH_TOL = 310 * 2.0 ** -21
ORTH_SHAPES = [(1, 1), (1, 9), (9, 1), (2, 3), (7, 7), (31, 33), (33, 31), (64, 64), (65, 200), (200, 65), (128, 129),
               (257, 100), (300, 301), (513, 1000), (1000, 513), (260, 2049), (1030, 1025)]


def close(got, ref, what, tol=ORTH_TOL):
    rel = float((got.double() - ref).norm() / ref.norm().clamp_min(1e-30))
    assert rel <= tol, f"{what}: relative error {rel:.3g} > {tol:.3g}"


@pytest.mark.parametrize("rows,cols", ORTH_SHAPES)
def test_orthogonalize(mx, rows, cols):
    print("orthogonalize", rows, cols, flush=True)
    g = gen(rows + 2 * cols)
    ins = [rand(g, rows, cols) * 10.0 ** (3 * i - 4) + rand(g, rows, 1) @ rand(g, 1, cols) * 10.0 ** (3 * i - 4) for i in range(3)]
    pairs = [guarded(rows, cols) for _ in ins]
    mx.orthogonalize(ins, [p[0] for p in pairs], stream=stream())
    intact(*[p[1] for p in pairs])
    for u, (o, _) in zip(ins, pairs):
        want = orth(u.double())
        close(o, want, f"{rows}x{cols}")
        plain = float((orth(u).double() - want).norm() / want.norm())
        close(o, want, f"{rows}x{cols} beside FP32", 4 * plain + 2.0 ** -20)
    same = [u.clone() for u in ins]
    ws = torch.empty(max(16, mx.orthogonalize_workspace(ins)), dtype=torch.uint8, device="cuda")
    mx.orthogonalize(same, same, workspace=ws, stream=stream())
    for o, (p, _) in zip(same, pairs):
        assert torch.equal(o, p), "in place, caller's workspace"


@pytest.mark.parametrize("steps,coef", [(0, NS), (1, NS), (3, (1.5, -0.5, 0.0)), (8, (2.0, -1.5, 0.5)), (2, (15 / 8, -10 / 8, 3 / 8))])
def test_orthogonalize_other_polynomials(mx, steps, coef):
    g = gen(steps)
    u = rand(g, 90, 150)
    o = torch.empty_like(u)
    mx.orthogonalize([u], [o], steps=steps, coefficients=coef, stream=stream())
    # none of these multiplies an error by more than the default polynomial does
    close(o, orth(u.double(), steps, coef), f"{steps} steps of {coef}", ORTH_TOL * max(1, steps / 5))


def test_orthogonalize_mixed_shapes_zero_tiny_huge_and_nan(mx):
    g = gen(77)
    ins = [rand(g, 40, 70), torch.zeros(40, 70, device="cuda"), rand(g, 70, 40), rand(g, 40, 70) * 1e-30,
           rand(g, 70, 40) * 1e30, rand(g, 5, 3), torch.empty(0, 7, device="cuda"), rand(g, 40, 70)]
    ins[7][3, 4] = float("nan")
    outs = [torch.empty_like(u) for u in ins]
    mx.orthogonalize(ins, outs, stream=stream())
    for i in (0, 2, 4, 5):
        close(outs[i], orth(ins[i].double()), f"matrix {i}")
    assert float(outs[1].abs().max()) == 0
    # below eps the matrix is divided by eps, and the iterations are linear there
    close(outs[3], orth(ins[3].double()), "tiny")
    assert bool(outs[7].isnan().all())


@pytest.mark.parametrize("rows,cols,count", [(1, 5, 2), (40, 70, 3), (130, 64, 2), (200, 333, 50), (513, 140, 3)])
@pytest.mark.parametrize("nesterov,adjust", [(True, "original"), (False, "match_rms_adamw")])
def test_muon(mx, rows, cols, count, nesterov, adjust):
    print("muon", rows, cols, count, flush=True)
    g = gen(rows * cols + count)
    p, gr, m = (rand(g, count, rows, cols, scale=s) for s in (1e-2, 1e-3, 1e-3))
    p0, m0 = p.clone(), m.clone()
    lr, wd, mu = 0.5, 0.1, 0.95
    mx.muon_step(p.unbind(0), gr.unbind(0), m.unbind(0), lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov,
                 adjust_lr=adjust, stream=stream())
    r = math.sqrt(max(1, rows / cols)) if adjust == "original" else 0.2 * math.sqrt(max(rows, cols))
    for i in range(count):
        # mu and 1 - mu reach the kernel as FP32
        mr = m0[i].double() + (1 - mu) * (gr[i].double() - m0[i].double())
        within(m[i], mr, 4 * U * (mr.abs() + gr[i].double().abs() + m0[i].double().abs()), "momentum")
        u = gr[i].double() + mu * (mr - gr[i].double()) if nesterov else mr
        o = orth(u)
        moved = (p0[i].double() * (1 - lr * wd) - p[i].double()) / (lr * r)
        err = float((moved - o).norm())
        tol = ORTH_TOL * float(o.norm()) + 4 * U * float(p0[i].double().norm()) / (lr * r) + 310 * 4 * U * float(o.norm())
        assert err <= tol, (i, err, tol)


def test_calls_on_another_stream_and_in_a_graph(mx):
    g = gen(4)
    x, w, b = rand(g, 130, 96), rand(g, 64, 96, scale=0.1), rand(g, 64)
    gamma, dy = rand(g, 96, mean=1.0), rand(g, 130, 64)
    mean, rstd = torch.empty(130, device="cuda"), torch.empty(130, device="cuda")
    h, y, z = torch.empty_like(x), torch.empty(130, 64, device="cuda"), torch.empty(130, 64, device="cuda")
    dh, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    dx, dg, dbt = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
    mom = torch.zeros_like(w)
    need = max(mx.layer_norm_backward_workspace(130, 96), mx.linear_workspace(130, 96, 64, mx.ACT_GELU),
               mx.linear_workspace(130, 96, 64, mx.ACT_GELU, True), mx.muon_workspace([w]), 16)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def step():
        s = stream()
        mx.layer_norm_forward(x, gamma, None, 1e-5, h, mean, rstd, stream=s)
        mx.linear_forward(h, w, b, y, activation=mx.ACT_GELU, z=z, workspace=ws, stream=s)
        mx.linear_backward(dy, h, w, z, dh, dw, db, activation=mx.ACT_GELU, workspace=ws, stream=s)
        mx.layer_norm_backward(dh, x, mean, rstd, gamma, dx, dg, dbt, workspace=ws, stream=s)
        mx.muon_step([w], [dw], [mom], lr=0.01, workspace=ws, stream=s)

    def state():
        return [t.clone() for t in (y, dx, dg, dbt, db, w, mom)]

    w0 = w.clone()
    eager = []
    for _ in range(3):
        step()
        eager.append(state())
    side = torch.cuda.Stream()
    w.copy_(w0)
    mom.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other = state()
    torch.cuda.current_stream().wait_stream(side)
    for a, b_ in zip(eager[0], other):
        assert torch.equal(a, b_)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    w.copy_(w0)
    mom.zero_()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b_ in zip(eager[i], state()):
            assert torch.equal(a, b_), f"replay {i}"


# ------------------------------------------- linear layers on packed operands
# Sizes at which the library packs its operands into two fp16 pieces, forward and
# backward: whole tiles, ragged ones, rows at no 16-byte boundary.
PACKED_SHAPES = [(2048, 2048, 2048), (1537, 765, 2050), (3001, 1003, 2999), (1290, 2052, 1924)]


def packed_case(m, k, n):
    g = gen(m + n)
    return rand(g, m, k), rand(g, n, k, scale=k ** -0.5), rand(g, n, scale=0.3), rand(g, m, n), rand(g, m, n, scale=0.1)


def run_linear(mx, x, w, b, res, dy, code):
    m, k, n = *x.shape, w.shape[0]
    (y, t0), (z, t1), (dx, t2), (dw, t3), (db, t4) = guarded(m, n), guarded(m, n), guarded(m, k), guarded(n, k), guarded(n)
    mx.linear_forward(x, w, b, y, activation=code, residual=res, z=z, stream=stream())
    mx.linear_backward(dy, x, w, z, dx, dw, db, activation=code, stream=stream())
    intact(t0, t1, t2, t3, t4)
    return y, z, dx, dw, db


def check_linear(x, w, b, res, dy, act, out, what):
    """A packed element is off by 2 u of itself or, as rows and columns lie within
    2^8 of the largest, of 2^-16 of that at the least; u / 4 of every term is
    dropped, and a sum of k terms rounds at most 3 k / 16 + 3 times."""
    y, z, dx, dw, db = out
    d = lambda t: t.double()
    k, n, m = x.shape[1], w.shape[0], x.shape[0]
    zr, yr = linear_ref(d(x), d(w), d(b), d(res), act)
    mag = d(x).abs() @ d(w).abs().t() + d(b).abs()
    floor = 2.0 ** -39 * float(x.abs().max()) * d(w).abs().sum(1) + 2.0 ** -39 * float(w.abs().max()) * d(x).abs().sum(1)[:, None]
    z_err = (3 * k / 16 + 12) * U * mag + floor
    within(z, zr, z_err, what + " z")
    within(y, yr, 1.13 * z_err + 16 * U * (zr.abs() + 1) + 4 * U * yr.abs(), what + " y")
    zl = d(z).cpu().requires_grad_()
    dz = torch.autograd.grad(ACT64[act](zl), zl, d(dy).cpu())[0].cuda()
    dz_err = 16 * U * d(dy).abs() * (d(z).abs() + 1)
    top = 2.0 ** -39 * float(dz.abs().max())
    f_x = top * d(w).abs().sum(0) + 2.0 ** -39 * float(w.abs().max()) * dz.abs().sum(1)[:, None]
    f_w = top * d(x).abs().sum(0) + 2.0 ** -39 * float(x.abs().max()) * dz.abs().sum(0)[:, None]
    within(dx, dz @ d(w), ((3 * n / 16 + 12) * U * dz.abs() + dz_err) @ d(w).abs() + f_x + 1e-30, what + " dx")
    within(dw, dz.t() @ d(x), ((3 * m / 16 + 12) * U * dz.abs() + dz_err).t() @ d(x).abs() + f_w + 1e-30, what + " dw")
    within(db, dz.sum(0), ((m / 64 + 64) * U * dz.abs() + dz_err).sum(0) + 1e-30, what + " db")


@pytest.mark.parametrize("m,k,n", PACKED_SHAPES)
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
def test_linear_packed(mx, m, k, n, act):
    print("packed linear", m, k, n, act, flush=True)
    case = packed_case(m, k, n)
    code = mx.ACTIVATIONS[act]
    out = run_linear(mx, *case, code)
    check_linear(*case, act, out, act)
    # Accuracy is FP32's: no further from float64 than twice torch's FP32 product.
    x, w, b = case[:3]
    want = x.double() @ w.double().t() + b.double()
    err = lambda t: float((t.double() - want).norm())
    assert err(out[1]) <= 2 * err(torch.addmm(b, x, w.t()))
    # Masked tokens: rows of zeros cost nothing and stay zero.
    x, w, b, res, dy = case
    dy = dy.clone()
    dy[::3] = 0
    out = run_linear(mx, x, w, b, res, dy, code)
    check_linear(x, w, b, res, dy, act, out, act + " masked")
    assert float(out[2][::3].abs().max()) == 0


def test_linear_packed_scales(mx):
    """Operands far from 1, each as a whole: one scale holds them."""
    m, k, n = 2048, 2048, 2048
    x, w, b, res, dy = packed_case(m, k, n)
    for sx, sw, sg in ((2.0 ** 40, 2.0 ** -30, 2.0 ** 20), (2.0 ** -60, 2.0 ** 50, 2.0 ** -60)):
        y = torch.empty(m, n, device="cuda")
        z = torch.empty_like(y)
        mx.linear_forward(x * sx, w * sw, None, y, z=z, stream=stream())
        base = torch.empty_like(y)
        mx.linear_forward(x, w, None, base, stream=stream())
        assert torch.equal(y, base * (sx * sw)), "powers of two change nothing but the exponent"
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        dx1, dw1 = torch.empty_like(x), torch.empty_like(w)
        mx.linear_backward(dy * sg, x * sx, w * sw, None, dx, dw, None, stream=stream())
        mx.linear_backward(dy, x, w, None, dx1, dw1, None, stream=stream())
        assert torch.equal(dx, dx1 * (sg * sw)) and torch.equal(dw, dw1 * (sg * sx))


def misfits(x, w, dy):
    """Operands that one scale cannot hold, by name."""
    m, k, n = *x.shape, w.shape[0]
    ramp = lambda c, e: torch.exp2(torch.linspace(-e, e, c, device="cuda"))
    yield "rows of x", x * ramp(m, 30)[:, None], w, dy
    yield "a dead column of x", torch.cat([x[:, :1] * 1e-6, x[:, 1:]], 1), w, dy
    yield "channels against each other", x * ramp(k, 20), w * ramp(k, -20), dy
    yield "columns of dy against rows of w", x, w * ramp(n, -40)[:, None], dy * ramp(n, 30)
    yield "a huge element", x, w.index_put((torch.tensor([5], device="cuda"), torch.tensor([7], device="cuda")),
                                           torch.tensor([1e30], device="cuda")), dy
    yield "tiny", x * 1e-36, w, dy * 1e-36


@pytest.mark.parametrize("which", range(6))
def test_linear_packed_misfits(mx, which):
    m, k, n = 2048, 2048, 2048
    x, w, b, res, dy = packed_case(m, k, n)
    name, x, w, dy = list(misfits(x, w, dy))[which]
    print("misfit", name, flush=True)
    y, dx, dw, db = torch.empty(m, n, device="cuda"), torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    mx.linear_forward(x, w, None, y, stream=stream())
    mx.linear_backward(dy, x, w, None, dx, dw, db, stream=stream())
    d = lambda t: t.double()
    within(y, d(x) @ d(w).t(), (k / 8 + 8) * U * (d(x).abs() @ d(w).abs().t()) + 1e-44, name + " y")
    within(dx, d(dy) @ d(w), (n / 8 + 8) * U * (d(dy).abs() @ d(w).abs()) + 1e-44, name + " dx")
    within(dw, d(dy).t() @ d(x), (m / 8 + 8) * U * (d(dy).abs().t() @ d(x).abs()) + 1e-44, name + " dw")


@pytest.mark.parametrize("rows,columns", [(0, 14), (14, 0), (7, 7), (10, 4), (9, 9), (2, 20), (20, 2)])
def test_linear_packed_depths(mx, rows, columns):
    """Half the rows of both operands and half their shared columns far below the
    others: outlier channels and quiet tokens, on both sides of what one scale holds."""
    print("depths", rows, columns, flush=True)
    m, k, n = 2048, 1024, 2048
    x, w, b, res, dy = packed_case(m, k, n)
    step = lambda c, e: torch.where(torch.arange(c, device="cuda") % 2 == 0, 1.0, 2.0 ** -e)
    d = lambda t: t.double()
    # The columns' steps of both operands the same way round, and against each other.
    for turn in (0, 1):
        x1 = x * step(m, rows)[:, None] * step(k, columns)
        w1 = w * step(n, rows)[:, None] * step(k, columns).roll(turn)
        dy1 = dy * step(m, columns)[:, None].roll(turn, 0) * step(n, rows)
        y, dx, dw = torch.empty(m, n, device="cuda"), torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda")
        mx.linear_forward(x1, w1, None, y, stream=stream())
        mx.linear_backward(dy1, x1, w1, None, dx, dw, None, stream=stream())
        within(y, d(x1) @ d(w1).t(), (k / 8 + 8) * U * (d(x1).abs() @ d(w1).abs().t()), f"y {turn}")
        within(dx, d(dy1) @ d(w1), (n / 8 + 8) * U * (d(dy1).abs() @ d(w1).abs()), f"dx {turn}")
        within(dw, d(dy1).t() @ d(x1), (m / 8 + 8) * U * (d(dy1).abs().t() @ d(x1).abs()), f"dw {turn}")


def test_linear_packed_special_values(mx):
    m, k, n = 2048, 2048, 2048
    x, w, b, res, dy = packed_case(m, k, n)
    x[3, 5], x[7, 9] = float("inf"), float("nan")
    y = torch.empty(m, n, device="cuda")
    mx.linear_forward(x, w, b, y, activation=mx.ACT_RELU, stream=stream())
    ref = F.relu(x.cpu() @ w.cpu().t() + b.cpu())
    got = y.cpu()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isposinf(), ref.isposinf())
    zero = torch.zeros_like(x)
    mx.linear_forward(zero, w, b, y, stream=stream())
    assert torch.equal(y, b.expand(m, n))


def test_linear_packed_in_a_graph(mx):
    m, k, n = 2048, 2048, 2048
    x, w, b, res, dy = packed_case(m, k, n)
    y, z = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ws = torch.empty(max(mx.linear_workspace(m, k, n, mx.ACT_GELU), mx.linear_workspace(m, k, n, mx.ACT_GELU, True)),
                     dtype=torch.uint8, device="cuda")

    def step():
        mx.linear_forward(x, w, b, y, activation=mx.ACT_GELU, residual=res, z=z, workspace=ws, stream=stream())
        mx.linear_backward(dy, x, w, z, dx, dw, db, activation=mx.ACT_GELU, workspace=ws, stream=stream())

    step()
    want = [t.clone() for t in (y, z, dx, dw, db)]
    spread = x * torch.exp2(torch.linspace(-30, 30, m, device="cuda"))[:, None]
    keep = x.clone()
    x.copy_(spread)
    step()
    want_spread = [t.clone() for t in (y, z, dx, dw, db)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for inputs, ref in ((keep, want), (spread, want_spread), (keep, want), (spread, want_spread)):
        x.copy_(inputs)
        graph.replay()
        torch.cuda.synchronize()
        for a, b_ in zip((y, z, dx, dw, db), ref):
            assert torch.equal(a, b_)
    with pytest.raises(mx.MXError, match="workspace"):
        side = torch.cuda.CUDAGraph()
        with torch.cuda.graph(side):
            mx.linear_forward(x, w, b, y, stream=stream())
