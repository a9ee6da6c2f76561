"""GPU parity of the feed-forward block's operators (C ABI on torch's GPU
tensors) where their number formats, forms and buffers meet their limits:
polynomials that turn negative, operands whose elements lie far apart, outputs
over inputs, sizes that take each form.

Bounds come from the operations' roundings, u = 2^-24 (half a step of FP32
relative to a value)."""
import math
import random
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


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


def within(got, ref, bound, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())}/{bad.numel()} outside; worst err/bound {float((err / bound).nan_to_num(1e30).max()):.3g}")


# ---------------------------------------------------- orthogonalised momentum
def orth(u, steps, coef, eps=1e-7):
    a, b, c = coef
    x = u / u.norm().clamp_min(eps)
    x = x.t() if u.shape[0] > u.shape[1] else x
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


def few_singular_values(shape, sigma):
    """Rows and columns far apart, one element each: singular values sigma."""
    u = torch.zeros(*shape, device="cuda")
    for i, s in enumerate(sigma):
        u[i * (shape[0] - 1) // max(1, len(sigma) - 1), i * (shape[1] - 1) // max(1, len(sigma) - 1)] = s
    return u


# (coefficients, singular values whose squares add up to 1).  The second pair of
# the last polynomial is where it reaches its largest value, 1.165, at which the
# next iteration's b t + c t^2 is largest.
TURNING = [((3.0, -5.0, 1.0), (1.0,)), ((1.0, -2.0, 0.0), (1.0,)), ((-1.0, 2.0, 0.0), (1.0,)),
           ((3.4445, -4.775, 1.2), (0.5208, 0.85368)), ((3.0, -5.0, 1.0), (0.6, 0.8))]


@pytest.mark.parametrize("shape", [(2, 9), (9, 2), (40, 70), (70, 40), (130, 257), (300, 200)])
@pytest.mark.parametrize("coef,sigma", TURNING)
def test_orthogonalize_polynomials_that_turn_negative(mx, shape, coef, sigma):
    """b t + c t^2 without a reaches further than a + b t + c t^2 does."""
    print("turning", shape, coef, sigma, flush=True)
    a, b, c = coef
    for steps in (1, 2, 3):
        for scale in (1.0, 1e-12):  # below eps the matrix is divided by eps
            u = few_singular_values(shape, sigma) * scale
            o = torch.full_like(u, 7.0)
            mx.orthogonalize([u], [o], steps=steps, coefficients=coef, stream=stream())
            want = orth(u.double(), steps, coef)
            # An iteration is off by 2^-21 of its terms' magnitudes (operands of 23
            # bits, 2^-22 of dropped pieces, FP32 sums) and multiplies an error by
            # the polynomial's slope, 7 at most for these on [0, 1.17].
            terms = abs(a) + 1.4 * abs(b) + 1.9 * abs(c)
            tol = 2.0 ** -21 * terms * sum(7.0 ** i for i in range(steps)) * (1.2 if scale == 1.0 else float(want.norm()))
            assert float((o.double() - want).norm()) <= tol + 1e-30, (steps, scale, float((o.double() - want).norm()), tol)


@pytest.mark.parametrize("count", [1, 3])
def test_muon_polynomial_that_turns_negative(mx, count):
    g = gen(count)
    p, m = rand(g, count, 40, 70, scale=1e-2), torch.zeros(count, 40, 70, device="cuda")
    gr = torch.zeros_like(m)
    gr[:, 17] = rand(g, count, 70)  # one nonzero row
    p0, coef = p.clone(), (3.0, -5.0, 1.0)
    mx.muon_step(p.unbind(0), gr.unbind(0), m.unbind(0), lr=0.5, weight_decay=0.0, momentum=0.5, steps=3, coefficients=coef,
                 stream=stream())
    for i in range(count):
        want = orth(gr[i].double(), 3, coef)  # momentum and Nesterov scale it, the norm divides that out
        moved = (p0[i].double() - p[i].double()) / 0.5
        tol = 2.0 ** -21 * (3 + 7 + 1.9) * 57 * 1.2 + 4 * U * float(p0[i].double().norm()) / 0.5
        assert float((moved - want).norm()) <= tol


# ---------------------------------------------------------------- layer norm
def ln_case(rows, cols):
    g = gen(rows + cols)
    return rand(g, rows, cols) * 3 + 1, rand(g, cols, mean=2.0), rand(g, cols, mean=-1.0), rand(g, rows, cols)


# Every width class, and last rows that leave groups of lanes without one.
IN_PLACE = [(1, 40), (15, 61), (37, 130), (11, 131), (9, 256), (3, 400), (6, 511), (5, 1000), (700, 1023), (3, 2048), (2, 5000), (2, 16001)]


# Widths that are walked from memory.
WALKED = [(5, 1), (70, 3), (3, 16389), (130, 20000)]


@pytest.mark.parametrize("rows,cols", IN_PLACE + WALKED)
def test_layer_norm_forward_over_its_input(mx, rows, cols):
    print("layer norm in place", rows, cols, flush=True)
    x, gamma, beta, _ = ln_case(rows, cols)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    mx.layer_norm_forward(x, gamma, beta, 1e-5, y, mean, rstd, stream=stream())
    for _ in range(5):
        over, m, r = x.clone(), torch.empty_like(mean), torch.empty_like(rstd)
        mx.layer_norm_forward(over, gamma, beta, 1e-5, over, m, r, stream=stream())
        assert torch.equal(over, y) and torch.equal(m, mean) and torch.equal(r, rstd)


@pytest.mark.parametrize("rows,cols", IN_PLACE + WALKED)
@pytest.mark.parametrize("which", ["dy", "x"])
def test_layer_norm_backward_over_an_input(mx, rows, cols, which):
    print("layer norm backward in place", rows, cols, which, flush=True)
    x, gamma, beta, dy = ln_case(rows, cols)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    mx.layer_norm_forward(x, gamma, beta, 1e-5, y, mean, rstd, stream=stream())
    dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
    mx.layer_norm_backward(dy, x, mean, rstd, gamma, dx, dg, db, stream=stream())
    for _ in range(5):
        t = {"dy": dy.clone(), "x": x.clone()}
        g, b = torch.empty_like(dg), torch.empty_like(db)
        mx.layer_norm_backward(t["dy"], t["x"], mean, rstd, gamma, t[which], g, b, stream=stream())
        assert torch.equal(t[which], dx) and torch.equal(g, dg) and torch.equal(b, db)


# -------------------------------------------------------------------- linear
F = torch.nn.functional


def check_products(mx, x, w, dy, what):
    """Every product within what FP32 products of whole operands are off by: 8 u of
    a term's roundings and dropped pieces, u of the sum every 8 terms."""
    m, k, n = *x.shape, w.shape[0]
    y, dx, dw = torch.empty(m, n, device="cuda"), torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda")
    mx.linear_forward(x, w, None, y, stream=stream())
    mx.linear_backward(dy, x, w, None, dx, dw, None, stream=stream())
    d = lambda t: t.double()
    within(y, d(x) @ d(w).t(), (k / 8 + 8) * U * (d(x).abs() @ d(w).abs().t()) + 1e-44, what + " y")
    within(dx, d(dy) @ d(w), (n / 8 + 8) * U * (d(dy).abs() @ d(w).abs()) + 1e-44, what + " dx")
    within(dw, d(dy).t() @ d(x), (m / 8 + 8) * U * (d(dy).abs().t() @ d(x).abs()) + 1e-44, what + " dw")


def activations(g, kind, *shape):
    return {"silu": lambda: F.silu(rand(g, *shape, scale=6.0)), "gelu": lambda: F.gelu(rand(g, *shape, scale=2.0)),
            "squared relu": lambda: F.relu(rand(g, *shape)) ** 2, "cubes": lambda: rand(g, *shape) ** 9,
            "subnormal": lambda: rand(g, *shape).index_put_((torch.tensor([3], device="cuda"),), torch.tensor(1e-41, device="cuda"))}[kind]()


def weights(g, kind, n, k):
    if kind == "identity":
        return torch.eye(n, k, device="cuda")
    if kind == "dense":
        return rand(g, n, k, scale=k ** -0.5)
    w = torch.zeros(n, k, device="cuda")  # one or four nonzero elements a row
    for _ in range(1 if kind == "one a row" else 4):
        w[torch.arange(n, device="cuda"), torch.randint(k, (n,), device="cuda", generator=g)] = rand(g, n)
    return w


@pytest.mark.parametrize("m,k,n", [(2048, 2048, 2048), (1537, 1025, 2050)])
@pytest.mark.parametrize("kind", ["silu", "gelu", "squared relu", "cubes", "subnormal"])
@pytest.mark.parametrize("weight", ["identity", "one a row", "four a row", "dense"])
def test_linear_elements_far_below_the_largest(mx, m, k, n, kind, weight):
    """Elements far below their operand's largest, alone or nearly alone in a sum."""
    print("far below", m, k, n, kind, weight, flush=True)
    g = gen(m + len(kind))
    x, w = activations(g, kind, m, k), weights(g, weight, n, k)
    check_products(mx, x, w, activations(g, kind, m, n), f"{kind} {weight}")
    # Either operand's, and those of a sparse gradient.
    check_products(mx, rand(g, m, k), activations(g, kind, n, k), weights(g, weight, m, n), f"{kind} {weight} turned")


@pytest.mark.parametrize("depth", [20, 24, 28, 30, 34, 40, 60])
def test_linear_sums_of_small_elements_alone(mx, depth):
    """Quarters of x far below the others, met by those columns of w that are not zero."""
    print("checkerboard", depth, flush=True)
    m, k, n = 2048, 1024, 2048
    g = gen(depth)
    upper = lambda c: torch.arange(c, device="cuda") < c // 2
    even = lambda c: torch.arange(c, device="cuda") % 2 == 0
    board = lambda r, c, low: torch.where(even(r)[:, None] == upper(c)[None], 1.0, low)
    x = rand(g, m, k) * board(m, k, 2.0 ** -depth)
    w = rand(g, n, k) * board(n, k, 0.0)
    dy = rand(g, m, n) * board(m, n, 2.0 ** -depth)
    check_products(mx, x, w, dy, f"checkerboard {depth}")
    check_products(mx, x * 2.0 ** 40, w, dy * board(m, n, 0.0), f"checkerboard {depth}, half of dy")


def test_linear_silu_tails(mx):
    """Relative to the value itself: exp2 and the reciprocal are good to 2 u each,
    and four roundings make it 8 u; results of less than 2^-126 may go to zero.  An
    identity weight, so that z is the input's own value."""
    z = torch.cat([-torch.linspace(2.0 ** -10, 100, 6000, device="cuda"), torch.linspace(0, 100, 2000, device="cuda"),
                   torch.tensor([-1e4, -3e38, 3e38, 200.0], device="cuda")]).view(-1, 4)
    eye, y, kept = torch.eye(4, device="cuda"), torch.empty_like(z), torch.empty_like(z)
    mx.linear_forward(z, eye, None, y, activation=mx.ACT_SILU, z=kept, stream=stream())
    assert torch.equal(kept, z)
    v = z.double()
    s = torch.sigmoid(v)
    small = 2.0 ** -126 * (v.abs() + 1)
    within(y, v * s, 8 * U * (v * s).abs() + small, "y")
    # s (1 + z (1 - s)): s to 7 u, 1 - s to u + 7 u s, the product and the sum to u each.
    dx = torch.empty_like(z)
    mx.linear_backward(torch.ones_like(z), z, eye, z, dx, None, None, activation=mx.ACT_SILU, stream=stream())
    inner = v * (1 - s)
    want = s * (1 + inner)
    bound = U * s * (9 * (1 + inner).abs() + v.abs() * (1 + 7 * s) + inner.abs() + 1) + 2.0 ** -126 * (v.abs() + 1) ** 2
    within(dx, want, bound, "slope")


@pytest.mark.parametrize("m,k,n", [(9000, 300, 1030), (70000, 514, 520), (200, 4096, 70000)])
def test_linear_far_below_in_long_lists(mx, m, k, n):
    """Rows and columns whose counts are in several words, and in lists of more than
    65536; weights that cover the small elements, and weights that do not."""
    print("long lists", m, k, n, flush=True)
    g = gen(m)
    x, dy = F.gelu(rand(g, m, k, scale=2.0)), F.gelu(rand(g, m, n, scale=2.0))
    check_products(mx, x, rand(g, n, k, scale=k ** -0.5), dy, "dense")
    # One column of w alone meets x's, one row of it dy's.
    w = torch.zeros(n, k, device="cuda")
    w[:, 7], w[11] = rand(g, n), rand(g, k)
    check_products(mx, x, w, dy, "one column and row")


def test_linear_without_room_for_pieces(mx):
    """A card so full that packed operands (0.56 GiB for the backward, 0.06 forward) find
    no room, while dz (0.25 GiB) does: the products without scratch take the call."""
    m, k, n = 8192, 1024, 8192
    g = gen(2)
    x, w, dy, b = rand(g, m, k), rand(g, n, k, scale=k ** -0.5), rand(g, m, n), rand(g, n)
    y, z, dx, dw, db = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)

    def forward():
        mx.linear_forward(x, w, b, y, activation=mx.ACT_GELU, residual=dy, z=z, stream=stream())

    def backward():
        mx.linear_backward(dy, x, w, z, dx, dw, db, activation=mx.ACT_GELU, stream=stream())

    def release():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        mx.check(mx.lib().mx_empty_cache())

    assert mx.linear_workspace(m, k, n, mx.ACT_GELU) > 64 << 20 and mx.linear_workspace(m, k, n, mx.ACT_GELU, True) > 560 << 20
    forward()
    backward()
    want = [t.clone() for t in (y, z, dx, dw, db)]
    for t in (y, dx, dw, db):  # z is an argument of the backward, which runs first
        t.fill_(float("nan"))
    fillers = []

    def fill(left):  # the driver finds a little more once most is taken
        release()
        for _ in range(8):
            over = torch.cuda.mem_get_info()[0] - left
            if over < 4 << 20:
                break
            fillers.append(torch.empty(over, dtype=torch.uint8, device="cuda"))
        assert torch.cuda.mem_get_info()[0] <= left + (8 << 20)

    try:
        fill(400 << 20)
        backward()
        torch.cuda.synchronize()
        fill(40 << 20)
        forward()
        torch.cuda.synchronize()
    finally:
        fillers.clear()
        release()
    # Both are within FP32's bound of the terms, so of each other within twice that.
    mag = x.abs() @ w.abs().t() + b.abs()
    z_err = 2 * (k / 8 + 8) * U * mag.double()
    within(z, want[1].double(), z_err, "z")
    within(y, want[0].double(), 1.13 * z_err + 32 * U * (want[1].double().abs() + 1) + 8 * U * want[0].double().abs(), "y")
    dz_err = 32 * U * dy.double().abs() * (want[1].double().abs() + 1)
    dz = (dy * 1.13).abs().double()
    within(dx, want[2].double(), (2 * (n / 8 + 8) * U * dz + dz_err) @ w.double().abs(), "dx")
    within(dw, want[3].double(), (2 * (m / 8 + 8) * U * dz + dz_err).t() @ x.double().abs(), "dw")
    within(db, want[4].double(), (2 * (m / 64 + 64) * U * dz + dz_err).sum(0), "db")


# ------------------------------------------------------------ launches counted
def test_launches_are_counted(mx):
    """Of calls whose launches are known from their sizes, and on the device surface."""
    g = gen(1)
    e = lambda *s: torch.empty(*s, device="cuda")
    x, w, b = rand(g, 9, 64), rand(g, 32, 64), rand(g, 32)
    mean, rstd = e(9), e(9)
    mx.layer_norm_forward(x, None, None, 1e-5, e(9, 64), mean, rstd, stream=stream())
    assert mx.last_launches() == 1
    mx.layer_norm_backward(x, x, mean, rstd, None, e(9, 64), None, None, stream=stream())
    assert mx.last_launches() == 1
    big = rand(g, 5000, 64)
    mean, rstd = e(5000), e(5000)
    mx.layer_norm_forward(big, None, None, 1e-5, e(5000, 64), mean, rstd, stream=stream())
    mx.layer_norm_backward(big, big, mean, rstd, None, e(5000, 64), e(64), e(64), stream=stream())
    assert mx.last_launches() == 2, "the rows, and the column sums' second part"
    mx.linear_forward(x, w, b, e(9, 32), stream=stream())
    assert mx.last_launches() == 1
    m = rand(g, 30, 50)
    for steps in (0, 1, 5):
        mx.orthogonalize([m], [torch.empty_like(m)], steps=steps, stream=stream())
        assert mx.last_launches() == (2 + steps), "norm, first, one a step; or norm and scaling"
    x, w = rand(g, 2048, 2048), rand(g, 2048, 2048)
    mx.linear_forward(x, w, None, e(2048, 2048), stream=stream())
    assert mx.last_launches() in (4, 5), "two passes, product, (join,) the products behind"
    mx.linear_backward(x, x, w, None, e(2048, 2048), e(2048, 2048), None, stream=stream())
    assert mx.last_launches() in (5, 6)
    before = mx.last_launches()
    mx.gemm(w, w, e(2048, 2048), stream=stream())
    mx.linear_workspace(64, 64, 64)
    assert mx.last_launches() == before, "other calls do not count"
    mx.linear_backward(x[:0], x[:0], w, None, None, None, None, stream=stream())
    assert mx.last_launches() == 0

    import torch_vulkan as vk
    from torch_vulkan.nn import linear
    xv, wv = x.cpu().to("vulkan"), w.cpu().to("vulkan")
    before = vk.execution_stats()["kernel_launches"]
    with torch.no_grad():
        linear(xv, wv)
    assert vk.execution_stats()["kernel_launches"] - before in (4, 5)


def test_refusal_behind_an_allocation_keeps_its_message():
    """Overlapping views, found once the call has taken its scratch from the allocator."""
    import torch_vulkan  # noqa: F401  (the device's operators)
    ops = torch.ops.torch_vulkan
    flat = torch.ones(100).to("vulkan")
    a, b = flat[:60].view(6, 10), flat[50:].view(5, 10)
    z = lambda t: torch.zeros(t.shape).to("vulkan")
    with pytest.raises(RuntimeError, match="overlaps another"):
        ops.muon_step_([a, b], [z(a), z(b)], [z(a), z(b)], 0.1, 0.0, 0.9, True, [1.0, 0.0, 0.0], 1, 1e-7, "original")
    ops.muon_step_([a], [z(a)], [z(a)], 0.1, 0.5, 0.9, True, [1.0, 0.0, 0.0], 1, 1e-7, "original")
    assert torch.equal(flat.cpu(), torch.cat([torch.full((60,), 1 - 0.1 * 0.5), torch.ones(40)]))


# ---------------------------------------- every tile, split and direction of a product
# Sizes whose plan takes them, and what the plan has to name so that a changed choice
# of tiles does not empty the list: whole tiles, tiles shared by several workgroups
# (0+n x parts), or both.
ORTH_PLANS = [
    ((4096, 4096, 1), r"gram<128>512\+\d+x\d+ poly<128>512\+\d+x\d+ update<256>\d+$"),
    ((1024, 1024, 16), r"gram<128>\d+ poly<128>\d+ update<256>\d+$"),
    ((2300, 700, 8), r"gram<128>\d+ poly<128>\d+ update<256>\d+$"),
    ((1500, 2048, 1), r"gram<128>0\+\d+x\d+ poly<128>0\+\d+x\d+ update<128>\d+$"),
    ((2048, 1536, 1), r"gram<128>0\+\d+x\d+ poly<128>0\+\d+x\d+ update<128>\d+$"),
    ((1280, 1600, 4), r"gram<128>\d+ poly<128>\d+ update<128>\d+\+\d+x\d+"),
    ((1600, 1280, 4), r"gram<128>\d+ poly<128>\d+ update<128>\d+\+\d+x\d+"),
    ((1500, 1536, 2), r"update<64>\d+\+\d+x\d+"),
    ((2300, 2048, 1), r"update<64>\d+\+\d+x\d+"),
    ((2048, 2300, 2), r"gram<64>\d+\+\d+x\d+ poly<64>\d+\+\d+x\d+ update<128>\d+\+\d+x\d+"),
    ((1600, 1000, 8), r"gram<64>\d+\+\d+x\d+ poly<64>\d+\+\d+x\d+ update<256>\d+$"),
    ((1000, 513, 6), r"gram<64>\d+ poly<64>\d+ update<128>\d+$"),
    ((200, 4100, 2), r"gram<64,deep>0\+\d+x\d+ poly<64,deep>\d+ update<128>\d+$"),
    ((915, 915, 22), r"gram<256>\d+ poly<256>\d+"),
    ((3011, 8394, 1), r"gram<256>0\+\d+x\d+ poly<256>0\+\d+x\d+"),
    ((4257, 4257, 1), r"update<256>\d+\+\d+x\d+"),
    ((7525, 2707, 1), r"update<256>\d+\+\d+x\d+"),
]
# Of |X| after five iterations: 2^-21 in each, multiplied by 3.9 at most in every later one.
ORTH_TOL = 310 * 2.0 ** -21
NS = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("shape,plan", ORTH_PLANS)
def test_orthogonalize_on_every_tile(mx, shape, plan):
    rows, cols, count = shape
    name = mx.orthogonalize_variant(rows, cols, count)
    print("orthogonalize", shape, name, flush=True)
    assert re.search(plan, name), name
    g = gen(rows + cols)
    ins = rand(g, count, rows, cols) + 3 * rand(g, count, rows, 4) @ rand(g, count, 4, cols)
    flat = torch.full((count * rows * cols + 64,), 12345.0, device="cuda")
    outs = flat[:-64].view(count, rows, cols)
    mx.orthogonalize(ins.unbind(0), outs.unbind(0), stream=stream())
    assert bool((flat[-64:] == 12345.0).all()), "wrote past the end"
    for i in {0, count // 2, count - 1}:
        want = orth(ins[i].double(), 5, NS)
        rel = float((outs[i].double() - want).norm() / want.norm())
        assert rel <= ORTH_TOL, (i, rel)
        # The same bound holds of the error's largest singular value, of 1.2 at most: of every row.
        worst = float((outs[i].double() - want).norm(dim=1).max())
        assert worst <= 1.2 * ORTH_TOL, (i, worst)


@pytest.mark.parametrize("shape,plan", [p for p in ORTH_PLANS if p[0] in (
    (1280, 1600, 4), (1600, 1280, 4), (1024, 1024, 16), (2300, 700, 8), (1500, 1536, 2), (2300, 2048, 1), (7525, 2707, 1))])
def test_muon_on_every_tile(mx, shape, plan):
    """The last product's stores, and the joins of its shared tiles, on a parameter."""
    rows, cols, count = shape
    assert re.search(plan, mx.orthogonalize_variant(rows, cols, count))
    print("muon", shape, flush=True)
    g = gen(rows)
    p, gr, m = (rand(g, count, rows, cols, scale=s) for s in (1e-2, 1e-3, 1e-3))
    p0, m0 = p.clone(), m.clone()
    lr, wd, mu = 0.5, 0.1, 0.95
    mx.muon_step(p.unbind(0), gr.unbind(0), m.unbind(0), lr=lr, weight_decay=wd, momentum=mu, stream=stream())
    for i in {0, count - 1}:
        mr = m0[i].double() + (1 - mu) * (gr[i].double() - m0[i].double())
        within(m[i], mr, 4 * U * (mr.abs() + gr[i].double().abs() + m0[i].double().abs()), "momentum")
        o = orth(gr[i].double() + mu * (mr - gr[i].double()), 5, NS)
        r = math.sqrt(max(1, rows / cols))
        moved = (p0[i].double() * (1 - lr * wd) - p[i].double()) / (lr * r)
        tol = ORTH_TOL * float(o.norm()) + 4 * U * float(p0[i].double().norm()) / (lr * r) + 310 * 4 * U * float(o.norm())
        assert float((moved - o).norm()) <= tol


# --------------------------------------- linear forwards and gradients on every form
# (m, k, n), the start of the products' names, forward or backward.
LINEAR_PLANS = [
    ((256, 4096, 4096), r"gemm_kernel<128x128x16,KVEC,KVEC>\+split"),
    ((128, 4096, 4094), r"gemm_kernel<64x64x16,KVEC,KVEC>\+split"),
    ((100, 2048, 1000), r"gemm_kernel<64x64x16,KVEC,KVEC>\+split"),
    ((100, 6001, 1000), r"gemm_kernel<64x64x16,KSCALAR,KSCALAR>\+split"),
    ((8192, 256, 1024), r"gemm_kernel<128x128x16,KVEC,KVEC>\+bias"),
    ((600, 300, 5000), r"gemm_kernel<64x64x16,KVEC,KVEC>\+bias"),
    ((20001, 65, 300), r"gemm_kernel<128x128x16,KSCALAR,KSCALAR>\+bias"),
    ((700, 700, 700), r"small<8>"),
    ((700, 40, 700), r"small<1>"),
    ((300, 100, 700), r"small<4>"),
    ((33, 4096, 64), r"few"),
    ((2048, 2048, 2048), r"packed"),
]


def slope(act, z):
    """The activations' derivatives, in the type of z."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))
    return s + 2 * c * z * s * (1 - s) * (1 + 3 * 0.044715 * z * z)


def check_layer(mx, x, w, b, res, dy, act, workspace=False, what=""):
    """One layer, forward with everything in its epilogue and backward, against 64 bits."""
    m, k, n = *x.shape, w.shape[0]
    code = mx.ACTIVATIONS[act]
    fn = dict(relu=F.relu, silu=F.silu, gelu=F.gelu, gelu_tanh=lambda v: F.gelu(v, approximate="tanh"))[act]
    room = lambda back: torch.empty(max(16, mx.linear_workspace(m, k, n, code, back)), dtype=torch.uint8, device="cuda") if workspace else None
    nan = lambda *s: torch.full(s, float("nan"), device="cuda")
    y, z, dx, dw, db = nan(m, n), nan(m, n), nan(m, k), nan(n, k), nan(n)
    mx.linear_forward(x, w, b, y, activation=code, residual=res, z=z, workspace=room(False), stream=stream())
    into = res.clone()
    mx.linear_forward(x, w, b, into, activation=code, residual=into, workspace=room(False), stream=stream())
    assert torch.equal(into, y), what + ": into the residual's buffer"
    mx.linear_backward(dy, x, w, z, dx, dw, db, activation=code, workspace=room(True), stream=stream())
    d = lambda t: t.double()
    zr = d(x) @ d(w).t() + d(b)
    z_err = (k / 8 + 8) * U * (d(x).abs() @ d(w).abs().t() + d(b).abs())
    yr = fn(zr) + d(res)
    within(z, zr, z_err, what + " z")
    within(y, yr, 1.13 * z_err + 16 * U * (zr.abs() + 1) + 4 * U * yr.abs(), what + " y")
    dz = d(dy) * slope(act, d(z))
    dz_err = 16 * U * d(dy).abs() * (d(z).abs() + 1)
    within(dx, dz @ d(w), ((n / 8 + 8) * U * dz.abs() + dz_err) @ d(w).abs() + 1e-30, what + " dx")
    within(dw, dz.t() @ d(x), ((m / 8 + 8) * U * dz.abs() + dz_err).t() @ d(x).abs() + 1e-30, what + " dw")
    within(db, dz.sum(0), ((m / 64 + 64) * U * dz.abs() + dz_err).sum(0) + 1e-30, what + " db")


@pytest.mark.parametrize("shape,plan", LINEAR_PLANS)
@pytest.mark.parametrize("workspace", [False, True])
def test_linear_on_every_form(mx, shape, plan, workspace):
    m, k, n = shape
    print("linear form", shape, mx.linear_variant(*shape), "|", mx.linear_variant(*shape, True), flush=True)
    assert re.match(plan, mx.linear_variant(*shape)), mx.linear_variant(*shape)
    g = gen(m + k)
    act = ["gelu", "silu", "gelu_tanh", "relu"][(m + k + n) % 4]
    check_layer(mx, rand(g, m, k), rand(g, n, k, scale=k ** -0.5), rand(g, n, scale=0.3), rand(g, m, n), rand(g, m, n), act,
                workspace, str(shape))


LINEAR_BACKWARD_PLANS = [
    ((128, 4096, 4096), r"gemm_kernel<64x64x16,KVEC,RVEC>\+split gemm_kernel<256x128x16,RVEC,RVEC>"),
    ((20000, 64, 300), r"gemm_kernel<64x64x16,KVEC,RVEC> gemm_kernel<64x64x16,RVEC,RVEC>\+split"),
    ((200000, 129, 129), r"gemm_kernel<\w+,KSCALAR,RSCALAR> gemm_kernel<64x64x16,RSCALAR,RSCALAR>\+split"),
    ((8192, 256, 1024), r"packed"),
    ((100, 2048, 1000), r"small<4>"),
    ((8, 40, 30), r"small<1>"),
]


@pytest.mark.parametrize("shape,plan", LINEAR_BACKWARD_PLANS)
@pytest.mark.parametrize("workspace", [False, True])
def test_linear_backward_on_every_form(mx, shape, plan, workspace):
    m, k, n = shape
    print("linear backward form", shape, mx.linear_variant(*shape, True), flush=True)
    assert re.match(plan, mx.linear_variant(*shape, True)), mx.linear_variant(*shape, True)
    g = gen(m + n)
    check_layer(mx, rand(g, m, k), rand(g, n, k, scale=k ** -0.5), rand(g, n, scale=0.3), rand(g, m, n), rand(g, m, n), "gelu",
                workspace, str(shape))


@pytest.mark.parametrize("tile", ["0", "1", "2", "3"])
@pytest.mark.parametrize("shape", [(2048, 2048, 2048), (2049, 2052, 2060), (2050, 1025, 2047)])
def test_linear_left_to_the_other_products(mx, monkeypatch, tile, shape):
    """Operands that packed products leave, with everything in the epilogue of the
    kernels that take them, on each of their tiles (256-wide ones where k % 4 == 0)."""
    m, k, n = shape
    assert mx.linear_variant(m, k, n) == "packed" and mx.linear_variant(m, k, n, True) == "packed"
    monkeypatch.setenv("MX_GEMM_TILE", tile)
    print("left out", shape, tile, flush=True)
    g = gen(k)
    spread = torch.exp2(torch.linspace(-30, 10, m, device="cuda"))[:, None]
    sparse = torch.zeros(n, k, device="cuda")
    sparse[torch.arange(n, device="cuda"), torch.randint(k, (n,), device="cuda", generator=g)] = rand(g, n)
    check_layer(mx, rand(g, m, k) * spread, sparse, rand(g, n, scale=0.3), rand(g, m, n), rand(g, m, n) * spread, "gelu", False,
                f"{shape} tile {tile}")


@pytest.mark.parametrize("at", [0, 31, 32, 777, 2047, 2048])
@pytest.mark.parametrize("low", [2.0 ** -45, 0.0])
def test_linear_one_row_or_column_far_below(mx, at, low):
    """One row or column of an operand alone is small (or zero: masked), everything else
    dense with a few deep elements, so that the counts decide."""
    print("one row", at, low, flush=True)
    m = k = n = 2049
    assert mx.linear_variant(m, k, n) == "packed" and mx.linear_variant(m, k, n, True) == "packed"
    g = gen(at)

    def operand():
        t = rand(g, m, k)
        t.view(-1)[torch.randint(m * k, (5,), device="cuda", generator=g)] = 2.0 ** -48
        return t

    for which in range(6):
        x, w, dy = operand(), operand(), operand()
        t = (x, w, dy)[which % 3]
        if which < 3:
            t[at] *= low
        else:
            t[:, at] *= low
        check_products(mx, x, w, dy, f"{'x w dy'.split()[which % 3]} {'row' if which < 3 else 'column'} {at} {low}")


def test_calls_stay_within_their_workspaces(mx):
    """Guards behind the bytes that the queries name, over random sizes and addresses."""
    rng = random.Random(5)
    g = gen(5)

    def room(need):
        t = torch.full((max(need, 16) + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        return t[:max(need, 16)], t[max(need, 16):]

    def unaligned(*s):
        return rand(g, math.prod(s) + 1)[1:].view(*s) if rng.random() < 0.3 else rand(g, *s)

    log = lambda hi: max(1, round(math.exp(rng.uniform(0, math.log(hi)))))
    for i in range(60):
        m, k, n = log(5000), log(3000), log(3000)
        act = rng.randrange(5)
        print("workspace", i, m, k, n, act, mx.linear_variant(m, k, n), "|", mx.linear_variant(m, k, n, True), flush=True)
        x, w, dy, z = unaligned(m, k), unaligned(n, k), unaligned(m, n), unaligned(m, n)
        y, dx, dw, db = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda")
        ws, guard = room(mx.linear_workspace(m, k, n, act))
        mx.linear_forward(x, w, db, y, activation=act, workspace=ws, stream=stream())
        ws, guard2 = room(mx.linear_workspace(m, k, n, act, True))
        mx.linear_backward(dy, x, w, z, dx, dw, db, activation=act, workspace=ws, stream=stream())
        rows, cols = log(3000), log(20000)
        x, y = unaligned(rows, cols), torch.empty(rows, cols, device="cuda")
        mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
        ws, guard3 = room(mx.layer_norm_backward_workspace(rows, cols))
        mx.layer_norm_backward(x, x, mean, rstd, None, y, torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda"),
                               workspace=ws, stream=stream())
        mats = [unaligned(r, c) for r, c in [(log(1500), log(1500))] * rng.randint(1, 5) + [(log(200), log(3000))]]
        ws, guard4 = room(mx.orthogonalize_workspace(mats))
        mx.orthogonalize(mats, [torch.empty_like(t) for t in mats], workspace=ws, stream=stream())
        ws, guard5 = room(mx.muon_workspace(mats))
        mx.muon_step([t.clone() for t in mats], mats, [torch.zeros_like(t) for t in mats], workspace=ws, stream=stream())
        for at, t in enumerate((guard, guard2, guard3, guard4, guard5)):
            assert bool((t == 0x5A).all()), (i, at)


# ------------------------------------------------- more than 2^31 elements to a tensor
def sampled(count):
    """The first and last rows, and some between."""
    return torch.cat([torch.arange(16), torch.arange(count // 2, count // 2 + 16), torch.arange(count - 32, count)]).to("cuda")


@pytest.mark.parametrize("k,plan", [(64, "gemm_kernel"), (512, "packed")])
def test_linear_outputs_past_32_bit_offsets(mx, k, plan):
    m, n = 66001, 33001  # 2.18e9 elements
    assert mx.linear_variant(m, k, n).startswith(plan)
    print("large linear", m, k, n, mx.linear_variant(m, k, n), "|", mx.linear_variant(m, k, n, True), flush=True)
    g = gen(k)
    x, w, b, dy = rand(g, m, k), rand(g, n, k, scale=k ** -0.5), rand(g, n), rand(g, m, n)
    y, z = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    mx.linear_forward(x, w, b, y, activation=mx.ACT_SILU, residual=dy, z=z, stream=stream())
    mx.linear_backward(dy, x, w, z, dx, dw, db, activation=mx.ACT_SILU, stream=stream())
    d = lambda t: t.double()
    r = sampled(m)
    zr = d(x[r]) @ d(w).t() + d(b)
    z_err = (k / 8 + 8) * U * (d(x[r]).abs() @ d(w).abs().t() + d(b).abs())
    yr = F.silu(zr) + d(dy[r])
    within(z[r], zr, z_err, "z")
    within(y[r], yr, 1.13 * z_err + 16 * U * (zr.abs() + 1) + 4 * U * yr.abs(), "y")
    dz, err = d(dy[r]) * slope("silu", d(z[r])), 16 * U * d(dy[r]).abs() * (d(z[r]).abs() + 1)
    within(dx[r], dz @ d(w), ((n / 8 + 8) * U * dz.abs() + err) @ d(w).abs(), "dx")
    c = sampled(n)
    dz, err = d(dy[:, c]) * slope("silu", d(z[:, c])), 16 * U * d(dy[:, c]).abs() * (d(z[:, c]).abs() + 1)
    within(dw[c], dz.t() @ d(x), ((m / 8 + 8) * U * dz.abs() + err).t() @ d(x).abs(), "dw")
    within(db[c], dz.sum(0), ((m / 64 + 64) * U * dz.abs() + err).sum(0), "db")


@pytest.mark.parametrize("rows,cols", [(140001, 16001), (70001, 32001)])
def test_layer_norm_past_32_bit_offsets(mx, rows, cols):
    print("large layer norm", rows, cols, flush=True)
    g = gen(rows)
    x, gamma, beta, dy = rand(g, rows, cols), rand(g, cols, mean=1.0), rand(g, cols), rand(g, rows, cols)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    mx.layer_norm_forward(x, gamma, beta, 1e-5, y, mean, rstd, stream=stream())
    r = sampled(rows)
    dg, db = torch.empty_like(gamma), torch.empty_like(beta)
    xd, dyd, gd = x[r].double(), dy[r].double(), gamma.double()
    rr = 1 / torch.sqrt(xd.var(1, correction=0, keepdim=True) + 1e-5)
    xh = (xd - xd.mean(1, keepdim=True)) * rr
    # unit rows: the statistics are off by 40 u, and everything behind them by a few u more
    within(y[r], xh * gd + beta.double(), 60 * U * ((xh.abs() + 1) * gd.abs() + beta.double().abs()), "y")
    c = sampled(cols)
    xc = (x[:, c].double() - mean.double()[:, None]) * rstd.double()[:, None]
    dyc = dy[:, c].double()
    mx.layer_norm_backward(dy, x, mean, rstd, gamma, y, dg, db, stream=stream())
    gr = dyd * gd
    want = rr * (gr - gr.mean(1, keepdim=True) - xh * (gr * xh).mean(1, keepdim=True))
    within(y[r], want, 100 * U * (gr.abs() + gr.abs().mean(1, keepdim=True) + xh.abs()) * rr, "dx")
    deep = 64 + rows / 64
    within(dg[c], (dyc * xc).sum(0), (deep * U * (dyc * xc).abs()).sum(0), "dgamma")
    within(db[c], dyc.sum(0), (deep * U * dyc.abs()).sum(0), "dbeta")


@pytest.mark.parametrize("rows,cols", [(900, 2400001), (2400001, 900), (130, 16777216)])
def test_orthogonalize_past_32_bit_offsets(mx, rows, cols):
    print("large orthogonalize", rows, cols, mx.orthogonalize_variant(rows, cols), flush=True)
    g = gen(rows)
    u = rand(g, rows, cols)
    o = torch.empty_like(u)
    mx.orthogonalize([u], [o], stream=stream())
    mx.check(mx.lib().mx_empty_cache())
    turned = rows > cols
    x = u.t() if turned else u
    s = min(rows, cols)
    gram = torch.zeros(s, s, dtype=torch.double, device="cuda")
    for part in x.split(1 << 18, dim=1):
        p = part.double()
        gram += p @ p.t()
    norm2 = gram.diagonal().sum()
    a, b, c = NS
    eye = torch.eye(s, dtype=torch.double, device="cuda")
    total, gram = eye / norm2.sqrt(), gram / norm2
    for _ in range(5):  # X stays a polynomial of its first Gram matrix times itself
        q = a * eye + b * gram + c * gram @ gram
        total, gram = q @ total, q @ gram @ q
    at = sampled(max(rows, cols))
    want = total @ x[:, at].double()
    got = (o[at].t() if turned else o[:, at]).double()
    # FP32 sums of l terms, 16 to a rounding, are off by a walk of l / 16 of them in each
    # iteration, which the later ones multiply as they do the pieces' errors.
    worst = float(((got - want).norm(dim=0) / want.norm(dim=0)).max())
    assert worst <= ORTH_TOL + 310 * U * math.sqrt(max(rows, cols) / 16), worst
    print("worst column", worst)
