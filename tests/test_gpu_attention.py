"""GPU parity of the attention layer's operators (rotation, attention, paged cache,
attention over it; C ABI on torch's GPU tensors) against float64.

Bounds come from the operations' roundings, u = 2^-24 (half a step of FP32
relative to a value):
  * a product over k of operands without bits left out is off by at most
    (k / 8 + 8) u of the sum of the terms' magnitudes (8 of a term's roundings
    and its dropped pieces, one rounding of the sum every 8 terms or more);
  * a score is such a product, and times the scale 3 u of itself more; the
    exponent and lse are rounded at the size of the largest score, and exp2 is off
    by 2 u of its value: a probability is off by twice the score's error (its own and
    the sum's) and 8 u (1 + largest score) of itself;
  * what is summed over n tokens is such a product of the probabilities, added up
    tile by tile of 32: (n / 32 + 32) u of the sum of the terms' magnitudes.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TAIL = 12345.0


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
    flat = torch.full((n + 64,), TAIL, device="cuda")
    return flat[:n].view(*shape), flat[n:]


def intact(*tails):
    for t in tails:
        assert bool((t == TAIL).all()), "wrote past the end of an output"


def within(got, ref, bound, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())}/{bad.numel()} outside; worst err/bound {float((err / bound).nan_to_num(1e30).max()):.3g}")


def strided(g, tokens, heads, dim, gap=0, heads_first=False):
    """A packed tensor whose rows lie `gap` elements further apart, or whose heads lie outside its tokens."""
    if heads_first:
        return rand(g, heads, tokens, dim).transpose(0, 1)
    return rand(g, tokens, heads * dim + gap)[:, :heads * dim].unflatten(1, (heads, dim))


# ------------------------------------------------------------------- rotation
def frequencies(rot, base=10000.0, factor=1.0):
    return [base ** (-2.0 * i / max(rot, 1)) / factor for i in range(rot // 2)]


def rotary_ref(x, w, positions, freqs, interleaved, magnitude, eps):
    """(outputs, sum of the terms' magnitudes) in float64."""
    rot = 2 * len(freqs)
    xh, r = x, torch.ones_like(x[..., :1])
    if eps is not None:
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        xh = x * r * (1 if w is None else w)
    a = positions.double()[:, None, None] * torch.tensor(freqs, dtype=torch.double, device=x.device)
    c, s = torch.cos(a) * magnitude, torch.sin(a) * magnitude
    first = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    second = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    y, mag = xh.clone(), xh.detach().abs().clone()
    if rot:
        p, q = xh[..., first], xh[..., second]
        y[..., first], y[..., second] = p * c - q * s, q * c + p * s
        both = p.detach().abs() + q.detach().abs()
        mag[..., first] = mag[..., second] = both * abs(magnitude)
    return y, mag, r


ROTARY = [(1, 1, 0, 1, 0), (1, 2, 1, 2, 2), (3, 1, 1, 7, 4), (5, 3, 1, 16, 16), (2, 0, 3, 20, 12), (67, 4, 2, 22, 22),
          (33, 16, 4, 64, 64), (9, 5, 5, 65, 34), (130, 3, 1, 80, 80), (40, 2, 2, 96, 32), (257, 8, 2, 128, 128),
          (3, 33, 7, 128, 64), (31, 2, 1, 130, 130), (12, 2, 2, 255, 200), (65, 1, 1, 256, 256), (1500, 4, 1, 64, 64)]


@pytest.mark.parametrize("tokens,hq,hk,dim,rot", ROTARY)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", ["none", "plain", "weights"])
def test_rotary(mx, tokens, hq, hk, dim, rot, interleaved, norm):
    print("rotary", tokens, hq, hk, dim, rot, interleaved, norm, flush=True)
    g = gen(tokens * 31 + dim)
    eps, magnitude, freqs = (None if norm == "none" else 1e-6), 1.25, frequencies(rot, factor=2.0)
    x = [strided(g, tokens, h, dim, gap=3 * i + 1) * 2 if h else None for i, h in enumerate((hq, hk))]
    w = [rand(g, dim, mean=1.0, scale=0.3) if norm == "weights" and h else None for h in (hq, hk)]
    dy = [rand(g, tokens, h, dim) if h else None for h in (hq, hk)]
    pos = torch.randint(-5, 200000, (tokens,), device="cuda", generator=g)
    plan = mx.Rotary(freqs, interleaved=interleaved, magnitude=magnitude)
    outs = [guarded(tokens, h, dim) if h else (None, None) for h in (hq, hk)]
    mx.qk_norm_rotary_forward(x[0], x[1], pos, plan, outs[0][0], outs[1][0], w[0], w[1], eps, stream=stream())
    grads = [guarded(tokens, h, dim) if h else (None, None) for h in (hq, hk)]
    dws = [guarded(dim) if v is not None else (None, None) for v in w]
    back = lambda a, b, c, d, **kw: mx.qk_norm_rotary_backward(
        dy[0], dy[1], x[0] if eps is not None else None, x[1] if eps is not None else None, pos, plan, a, b, c, d, w[0], w[1],
        eps, stream=stream(), **kw)
    back(grads[0][0], grads[1][0], dws[0][0], dws[1][0])
    for i, h in enumerate((hq, hk)):
        if not h:
            continue
        # (autograd of the reference runs on the CPU: the engine knows one accelerator, the "vulkan" device)
        xd = x[i].double().cpu().requires_grad_()
        wd = w[i].double().cpu().requires_grad_() if w[i] is not None else None
        y, mag, r = rotary_ref(xd, wd, pos.cpu(), freqs, interleaved, magnitude, eps)
        # Angles are within 2^-27 of a turn and sine and cosine within 4 u, the norm's square sum within
        # 10 u (a lane's 4, 6 of lanes), its root half of that: 24 u a term in all.
        within(outs[i][0].cpu(), y.detach(), 24 * U * mag + 1e-30, "y")
        leaves = [xd] + ([wd] if wd is not None else [])
        ref = torch.autograd.grad(y, leaves, dy[i].double().cpu())
        gm = rotary_ref(dy[i].double().cpu().abs(), None, pos.cpu(), freqs, interleaved, magnitude, None)[1]  # of the turned back gradient
        if eps is None:
            within(grads[i][0].cpu(), ref[0], 24 * U * gm + 1e-30, "dx")
        else:
            gw = gm * (1 if wd is None else wd.detach().abs())
            xr = (xd * r).detach().abs()
            within(grads[i][0].cpu(), ref[0], 80 * U * r.detach() * (gw + xr * (gw * xr).mean(-1, keepdim=True)) + 1e-30, "dx")
        if wd is not None:
            within(dws[i][0].cpu(), ref[1], (80 + tokens * h / 64) * U * (gm * xr).sum((0, 1)) + 1e-30, "dw")
    intact(*(t for _, t in outs + grads + dws if t is not None))
    # Single gradients and a caller's workspace give the same bits.
    ws = torch.empty(max(16, mx.qk_norm_rotary_workspace(tokens, hq, hk, dim, plan, eps)), dtype=torch.uint8, device="cuda")
    for i in range(2):
        for j, (t, _) in enumerate((grads[i], dws[i])):
            if t is None:
                continue
            args = [None] * 4
            args[i + 2 * j] = again = torch.empty_like(t)
            back(*args, workspace=ws)
            assert torch.equal(again, t)


def test_rotary_in_place_and_extremes(mx):
    g = gen(3)
    plan, pos = mx.Rotary(frequencies(64)), torch.tensor([0, 2 ** 40, -2 ** 40, 10 ** 6], device="cuda")
    q, k = rand(g, 4, 3, 64), rand(g, 4, 1, 64)
    a, b = torch.empty_like(q), torch.empty_like(k)
    mx.qk_norm_rotary_forward(q, k, pos, plan, a, b, eps=1e-6, stream=stream())
    y, mag, _ = rotary_ref(q.double(), None, pos, frequencies(64), False, 1.0, 1e-6)
    # An angle of 2^40 is off by 2^40 2^-53 2 of a radian in 64 bits.
    within(a, y, (24 * U + 2 ** -11) * mag, "far positions")
    within(a[[0, 3]], y[[0, 3]], 24 * U * mag[[0, 3]], "near positions")
    qi, ki = q.clone(), k.clone()
    mx.qk_norm_rotary_forward(qi, ki, pos, plan, qi, ki, eps=1e-6, stream=stream())
    assert torch.equal(qi, a) and torch.equal(ki, b)
    gi = a.clone()
    want = torch.empty_like(gi)
    mx.qk_norm_rotary_backward(a, None, q, None, pos, plan, want, None, eps=1e-6, stream=stream())
    mx.qk_norm_rotary_backward(gi, None, q, None, pos, plan, gi, None, eps=1e-6, stream=stream())
    assert torch.equal(gi, want)
    # A row of zeros, a NaN in one head, an infinity in another: the other rows keep their bits.
    q2 = q.clone()
    q2[1, 0] = 0
    q2[2, 1, 5] = float("nan")
    q2[3, 2, 7] = float("inf")
    c = torch.empty_like(q)
    mx.qk_norm_rotary_forward(q2, None, pos, plan, c, None, eps=1e-6, stream=stream())
    assert bool((c[1, 0] == 0).all()) and bool(c[2, 1].isnan().all())
    keep = torch.ones(4, 3, dtype=torch.bool, device="cuda")
    keep[1, 0] = keep[2, 1] = keep[3, 2] = False
    assert torch.equal(c[keep], a[keep])
    dw = torch.full((64,), 7.0, device="cuda")
    mx.qk_norm_rotary_backward(a[:0], None, q[:0], None, pos[:0], plan, None, None, dq_weight=dw, eps=1e-6, stream=stream())
    assert bool((dw == 0).all()), "no tokens: zero gradients"


# ------------------------------------------------------------------ attention
def visible(n, window, sinks):
    i = torch.arange(n, device="cuda")
    back = i[:, None] - i[None, :]
    return (back >= 0) & ((back < window) | (i < sinks)[None, :]) if window else back >= 0


def attention_ref(q, k, v, do, window, sinks, scale):
    """One sequence in float64: name -> (value, bound), heads first inside."""
    h, kv, n, d = q.shape[1], k.shape[1], q.shape[0], q.shape[2]
    q, do = (t.double().transpose(0, 1) for t in (q, do))
    k, v = (t.double().transpose(0, 1).repeat_interleave(h // kv, 0) for t in (k, v))
    seen = visible(n, window, sinks)
    s = scale * (q @ k.transpose(1, 2))
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    lse = torch.logsumexp(s, -1)
    top = s.masked_fill(~seen, 0).abs().amax(-1, keepdim=True)
    es = (d / 8 + 11) * U * abs(scale) * (q.abs() @ k.abs().transpose(1, 2)) * seen  # of a score
    worst = es.amax(-1, keepdim=True)
    rel = es + worst + 8 * U * (1 + top)
    deep = (n / 32 + 32) * U
    out = p @ v
    eo = (p * (rel + deep)) @ v.abs()
    dp, delta = do @ v.transpose(1, 2), (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    edelta = (d / 8 + 8) * U * (do * out).abs().sum(-1, keepdim=True) + (do.abs() * eo).sum(-1, keepdim=True)
    eds = p * ((d / 8 + 8) * U * (do.abs() @ v.abs().transpose(1, 2)) + edelta) + (rel + 4 * U) * ds.abs()
    eds = eds + p * 2 * U * (dp.abs() + delta.abs())
    t = lambda x: x.transpose(1, 2)
    shared = lambda x: x.view(kv, h // kv, n, d).sum(1).transpose(0, 1)
    rows = lambda x: x.transpose(0, 1)
    return dict(out=(rows(out), rows(eo)),
                lse=(lse, worst[..., 0] + 8 * U * (1 + top[..., 0] + lse.abs())),
                dq=(rows(scale * (ds @ k)), rows(abs(scale) * ((eds + deep * ds.abs()) @ k.abs()))),
                dk=(shared(scale * (t(ds) @ q)), shared(abs(scale) * (t(eds + 2 * deep * ds.abs()) @ q.abs()))),
                dv=(shared(t(p) @ do), shared(t(p * (rel + 2 * deep)) @ do.abs())))


def run_attention(mx, q, k, v, do, starts, **form):
    (out, t0), (lse, t1) = guarded(*q.shape), guarded(q.shape[1], q.shape[0])
    (dq, t2), (dk, t3), (dv, t4) = guarded(*q.shape), guarded(*k.shape), guarded(*v.shape)
    mx.attention_forward(q, k, v, out, starts=starts, lse=lse, stream=stream(), **form)
    mx.attention_backward(do, q, k, v, out, lse, dq, dk, dv, starts=starts, stream=stream(), **form)
    intact(t0, t1, t2, t3, t4)
    return dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)


def starts_of(lengths, first=0):
    return torch.tensor([first] + list(lengths), dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)


ATTENTION = [
    ([1], 1, 1, 1, 0, 0), ([2], 2, 1, 3, 0, 0), ([31], 1, 1, 16, 0, 0), ([32], 3, 3, 32, 0, 0), ([33], 2, 2, 33, 0, 0),
    ([63, 0, 65], 2, 1, 20, 0, 0), ([64], 4, 2, 64, 7, 0), ([127], 2, 1, 80, 1, 0), ([128], 2, 2, 96, 32, 3),
    ([129, 1, 1, 200], 6, 2, 128, 64, 1), ([300], 3, 1, 65, 33, 40), ([257], 8, 1, 64, 100, 4), ([5, 700], 2, 2, 128, 0, 0),
    ([513], 4, 4, 48, 512, 600), ([0, 0, 40, 0], 2, 1, 128, 16, 2), ([1000], 2, 1, 128, 130, 70),
    ([1] * 70, 1, 1, 8, 0, 0), ([3, 30, 300] * 30, 2, 1, 32, 20, 5), ([2049], 1, 1, 64, 0, 0), ([640], 12, 3, 80, 128, 4),
    # first tokens seen from past the window: several chunks of queries, several blocks of keys
    ([2500, 31, 1100], 4, 2, 64, 40, 4), ([3100], 2, 1, 96, 200, 150), ([70, 1025, 400], 6, 2, 128, 1, 33), ([900, 900], 8, 1, 40, 600, 129),
    ([2300, 700], 2, 1, 32, 50, 700),  # more first tokens than are dealt out
    # enough workgroups of 128 rows not to be halved
    ([200, 33] * 250, 1, 1, 20, 40, 3), ([200, 33] * 250, 1, 1, 64, 0, 0), ([33, 200] * 250, 1, 1, 80, 100, 70),
    ([200, 33] * 250, 1, 1, 128, 0, 0), ([33, 200] * 250, 1, 1, 100, 50, 4), ([900, 40, 311], 6, 2, 112, 0, 0), ([777, 64], 2, 1, 128, 300, 5),
   
    # enough rows for workgroups of eight waves
    ([2600, 1500], 64, 32, 32, 0, 0), ([4200], 64, 2, 128, 300, 2)]


@pytest.mark.parametrize("lengths,h,kv,d,window,sinks", ATTENTION)
def test_attention(mx, lengths, h, kv, d, window, sinks):
    print("attention", lengths[:4], h, kv, d, window, sinks, flush=True)
    total, g = sum(lengths), gen(sum(lengths) * 7 + d)
    before, behind = 3, 5  # rows of no sequence
    t = before + total + behind
    q, k, v = strided(g, t, h, d, gap=1), strided(g, t, kv, d, heads_first=True), strided(g, t, kv, d, gap=4)
    do = rand(g, t, h, d)
    scale = 1.3 / math.sqrt(d)
    starts = starts_of(lengths, before)
    form = dict(window=window, sinks=sinks, scale=scale)
    got = run_attention(mx, q, k, v, do, starts, **form)
    at = before
    for n in lengths:
        r = slice(at, at + n)
        at += n
        if n == 0:
            continue
        for name, (ref, bound) in attention_ref(q[r], k[r], v[r], do[r], window, sinks, scale).items():
            within(got[name][:, r] if name == "lse" else got[name][r], ref, bound + 1e-30, f"{name} of {n}")
    for name, x in got.items():
        x = x.transpose(0, 1) if name == "lse" else x
        assert bool((x[:before] == TAIL).all()) and bool((x[t - behind:] == TAIL).all()), f"{name}: rows of no sequence"
    again = run_attention(mx, q, k, v, do, starts, **form)
    assert all(torch.equal(got[n], again[n]) for n in got), "the same call, other bits"
    # Single gradients, and a forward without lse.
    out = torch.full_like(got["out"], TAIL)
    mx.attention_forward(q, k, v, out, starts=starts, stream=stream(), **form)
    assert torch.equal(out, got["out"])
    for i, name in enumerate(("dq", "dk", "dv")):
        only = [None] * 3
        only[i] = torch.full_like(got[name], TAIL)
        mx.attention_backward(do, q, k, v, got["out"], got["lse"], *only, starts=starts, stream=stream(), **form)
        assert torch.equal(only[i], got[name]), name


@pytest.mark.parametrize("sequences,n", [(1, 96), (3, 50), (7, 1)])
def test_attention_equal_lengths(mx, sequences, n):
    g, t = gen(n), sequences * n
    q, k, v, do = rand(g, t, 4, 32), rand(g, t, 2, 32), rand(g, t, 2, 32), rand(g, t, 4, 32)
    a = run_attention(mx, q, k, v, do, starts_of([n] * sequences))
    b = run_attention(mx, q, k, v, do, None, sequences=sequences)
    assert all(torch.equal(a[x], b[x]) for x in a)


def test_attention_gradients_against_differences(mx):
    """<gradient, step> against (f(x + step) - f(x - step)) / 2 of f = sum(out w) in float64 around the kernel's
    gradients: the central difference of steps of 1e-4 is off by their square, 1e-8 of third derivatives of order 1."""
    g = gen(11)
    lengths, h, kv, d, window, sinks = [70, 41], 4, 2, 40, 24, 3
    t = sum(lengths)
    x = dict(q=rand(g, t, h, d), k=rand(g, t, kv, d), v=rand(g, t, kv, d))
    w = rand(g, t, h, d)
    got = run_attention(mx, x["q"], x["k"], x["v"], w, starts_of(lengths), window=window, sinks=sinks)

    def f(x):
        total, at = 0.0, 0
        for n in lengths:
            r = slice(at, at + n)
            q = x["q"][r].transpose(0, 1)
            k, v = (x[y][r].transpose(0, 1).repeat_interleave(h // kv, 0) for y in "kv")
            s = (q @ k.transpose(1, 2) / math.sqrt(d)).masked_fill(~visible(n, window, sinks), -math.inf)
            total += float((torch.softmax(s, -1) @ v * w[r].double().transpose(0, 1)).sum())
            at += n
        return total

    xd = {n: y.double() for n, y in x.items()}
    for name in "qkv":
        step = rand(g, *x[name].shape).double() * 1e-4
        diff = (f({**xd, name: xd[name] + step}) - f({**xd, name: xd[name] - step})) / 2
        dot = float((got["d" + name].double() * step).sum())
        size = float((got["d" + name].double() * step).abs().sum())
        assert abs(diff - dot) <= 1e-5 * size, (name, diff, dot, size)


def test_attention_keeps_what_is_not_seen_apart(mx):
    """NaN, infinities and huge values in rows that others do not see change no bit of those."""
    g = gen(5)
    lengths, h, kv, d, window, sinks = [90, 100, 75], 4, 2, 64, 20, 2
    t = sum(lengths)
    q, k, v, do = rand(g, t, h, d), rand(g, t, kv, d), rand(g, t, kv, d), rand(g, t, h, d)
    form = dict(window=window, sinks=sinks)
    clean = run_attention(mx, q, k, v, do, starts_of(lengths), **form)
    bad = 90 + 47  # position 47 of the second sequence: seen by its rows 47 .. 66
    rows = torch.arange(t, device="cuda")
    reached = (rows >= bad) & (rows < bad + window)
    # keys that a reached row sees
    touched = ((rows > bad - window) & (rows < bad + window)) | ((rows >= 90) & (rows < 90 + sinks))
    for value in (math.nan, math.inf, -math.inf):
        for where in ("k", "v"):
            x = dict(k=k.clone(), v=v.clone())
            x[where][bad, 1, 3] = value
            got = run_attention(mx, q, x["k"], x["v"], do, starts_of(lengths), **form)
            for name in ("out", "dq"):
                assert torch.equal(got[name][~reached], clean[name][~reached]), (name, where, value)
                assert torch.equal(got[name][:, :2], clean[name][:, :2]), "the other key head's rows"
                assert bool(got[name][reached][:, 2:].isnan().all()), (name, where, value)
            assert torch.equal(got["lse"][:, ~reached], clean["lse"][:, ~reached])
            for name in ("dk", "dv"):
                assert torch.equal(got[name][~touched], clean[name][~touched]), (name, where, value)
                assert torch.equal(got[name][:, 0], clean[name][:, 0])
                assert bool(got[name][bad, 1].isnan().all()), (name, where, value)
        for where in ("q", "do"):
            x = dict(q=q.clone(), do=do.clone())
            x[where][bad, 3, 0] = value
            got = run_attention(mx, x["q"], k, v, x["do"], starts_of(lengths), **form)
            other = rows != bad
            for name in ("out", "dq"):
                assert torch.equal(got[name][other], clean[name][other]), (name, where, value)
            assert bool(got["dq"][bad, 3].isnan().all())
            keys = ((rows > bad - window) & (rows <= bad)) | ((rows >= 90) & (rows < 90 + sinks))
            for name in ("dk", "dv"):
                assert torch.equal(got[name][~keys], clean[name][~keys]), (name, where, value)
                assert bool(got[name][keys][:, 1].isnan().all()), (name, where, value)


def test_attention_far_magnitudes(mx):
    """Rows far apart in size, tiny gradients, scores of hundreds: the bounds hold row by row."""
    g = gen(9)
    n, h, kv, d = 150, 2, 1, 64
    level = torch.exp2(torch.randint(-30, 10, (n, 1, 1), device="cuda", generator=g).float())
    q, k, v = rand(g, n, h, d) * 4, rand(g, n, kv, d) * 6, rand(g, n, kv, d) * level
    do = rand(g, n, h, d) * level * 2.0 ** -40
    got = run_attention(mx, q, k, v, do, None)
    for name, (ref, bound) in attention_ref(q, k, v, do, 0, 0, d ** -0.5).items():
        within(got[name] if name != "lse" else got[name], ref, bound + 1e-40, name)


def test_attention_starts_out_of_order_stay_in_range(mx):
    """Entries that the call's contract excludes: nothing outside the outputs is written."""
    g = gen(2)
    t = 130
    q, k, v, do = rand(g, t, 2, 32), rand(g, t, 1, 32), rand(g, t, 1, 32), rand(g, t, 2, 32)
    for bad in ([0, 100, 40, 130], [-7, 500, 2 ** 31 - 1, -2 ** 31], [130, 0, 130, 0], [90, 80, 70, 60]):
        run_attention(mx, q, k, v, do, torch.tensor(bad, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


# ------------------------------------------------- captured and on streams
def replay(call, outputs, inputs):
    """Captures call(), then replays it on changed inputs with eager work between; every replay equals the eager call."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
    torch.cuda.current_stream().wait_stream(s)
    for i in range(3):
        for t in inputs:
            t.mul_(-0.75)
        call()
        want = [t.clone() for t in outputs]
        for t in outputs:
            t.fill_(TAIL)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs, want)), f"replay {i}"


def test_attention_captured(mx):
    g, n, h, kv, d = gen(4), [100, 60], 4, 2, 64
    t = sum(n)
    q, k, v, do = rand(g, t, h, d), rand(g, t, kv, d), rand(g, t, kv, d), rand(g, t, h, d)
    out, lse, dq, dk, dv = torch.empty_like(q), q.new_empty(h, t), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws = torch.empty(max(mx.attention_workspace(t, 2, h, kv, d), mx.attention_workspace(t, 2, h, kv, d, True, window=30, sinks=2)),
                     dtype=torch.uint8, device="cuda")
    starts = starts_of(n)

    def call():
        mx.attention_forward(q, k, v, out, starts=starts, window=30, sinks=2, lse=lse, workspace=ws, stream=stream())
        mx.attention_backward(do, q, k, v, out, lse, dq, dk, dv, starts=starts, window=30, sinks=2, workspace=ws, stream=stream())

    replay(call, [out, lse, dq, dk, dv], [q, do])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), pytest.raises(mx.MXError, match="workspace"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            mx.attention_forward(q, k, v, out, starts=starts, stream=stream())


def test_rotary_captured(mx):
    g = gen(6)
    q, k, dq, dk = rand(g, 50, 4, 64), rand(g, 50, 2, 64), rand(g, 50, 4, 64), rand(g, 50, 2, 64)
    qw, pos, plan = rand(g, 64, mean=1.0), torch.arange(50, device="cuda"), mx.Rotary(frequencies(64))
    outs = [torch.empty_like(t) for t in (q, k, dq, dk)] + [torch.empty_like(qw)]
    ws = torch.empty(mx.qk_norm_rotary_workspace(50, 4, 2, 64, plan, 1e-6), dtype=torch.uint8, device="cuda")

    def call():
        mx.qk_norm_rotary_forward(q, k, pos, plan, outs[0], outs[1], qw, None, 1e-6, stream=stream())
        mx.qk_norm_rotary_backward(dq, dk, q, k, pos, plan, outs[2], outs[3], outs[4], None, qw, None, 1e-6, workspace=ws,
                                   stream=stream())

    replay(call, outs, [q, dq, dk])


# ---------------------------------------------------------------- the cache
def new_cache(mx, g, pages, kv, page, d, kind):
    """A cache full of what must not be read: NaN (and bytes with NaN scales)."""
    if kind == "i8":
        k = torch.randint(-127, 128, (pages, kv, page, d), device="cuda", dtype=torch.int8, generator=g)
        v = torch.randint(-127, 128, (pages, kv, d, page), device="cuda", dtype=torch.int8, generator=g)
        return mx.KVCache(k, v, *(torch.full((pages, kv, page), math.nan, device="cuda") for _ in range(2)))
    return mx.KVCache(*(torch.full(s, math.nan, device="cuda") for s in ((pages, kv, page, d), (pages, kv, d, page))))


def tables(g, lengths, page, spare=2):
    width = max(1, max((n + page - 1) // page for n in lengths))
    order = torch.randperm(len(lengths) * width + spare, device="cuda", generator=g)
    return order[:len(lengths) * width].view(len(lengths), width).to(torch.int32), len(lengths) * width + spare


def quantised(x):
    """What 8 bits hold of rows x, in float64 (the rounding of the exact quotient)."""
    scale = (x.double().abs().amax(-1, keepdim=True) / 127).float().double()
    q = torch.where(scale > 0, torch.round(x.double() / scale), torch.zeros_like(x.double())).clamp(-127, 127)
    return q * scale


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


CACHE = [([1], [1], 16, 1, 16), ([1], [17], 16, 2, 32), ([3, 0, 5], [3, 9, 30], 16, 1, 48), ([40], [40], 16, 2, 80),
         ([33, 1, 70], [90, 1, 70], 32, 3, 96), ([128, 64], [200, 64], 64, 2, 128), ([1] * 20, list(range(1, 21)), 48, 2, 64),
         ([300], [1000], 128, 1, 112)]


@pytest.mark.parametrize("new,lengths,page,kv,d", CACHE)
@pytest.mark.parametrize("kind", ["i8", "f32"])
def test_cache_write_and_read(mx, new, lengths, page, kv, d, kind):
    print("cache", new[:4], lengths[:4], page, kv, d, kind, flush=True)
    g = gen(sum(lengths) + d)
    table, pages = tables(g, lengths, page)
    cache = new_cache(mx, g, pages, kv, page, d, kind)
    held = [t.clone() for t in cache.tensors if t is not None]
    t = sum(new)
    k = strided(g, t, kv, d, gap=5) * (rand(g, t, 1, 1).abs() + 0.1)
    v = strided(g, t, kv, d, heads_first=True)
    k[0, 0] = 0  # a row without a scale
    batch = mx.KVBatch(table, i32(lengths), t, starts_of(new))
    mx.kv_cache_write(cache, batch, k, v, stream=stream())
    (ko, t0), (vo, t1) = guarded(t, kv, d), guarded(t, kv, d)
    mx.kv_cache_read(cache, batch, ko, vo, stream=stream())
    intact(t0, t1)
    for got, x in ((ko, k), (vo, v)):
        if kind == "f32":
            assert torch.equal(got, x)
        else:
            ref = quantised(x)
            within(got, ref, U * ref.abs(), "read back")  # one rounding of the product with the scale
            assert bool(((got.double() - x.double()).abs() <= x.double().abs().amax(-1, keepdim=True) / 127 * (0.5 + 300 * U)).all())
    # Nothing but the new tokens' places has changed.
    at, mask = 0, torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b, (n, length) in enumerate(zip(new, lengths)):
        for p in range(length - n, length):
            mask[int(table[b, p // page]), p % page] = True
    for now, then in zip([x for x in cache.tensors if x is not None], held):
        keep = ~mask[:, None, :, None] if now.dim() == 4 and now.shape[2] == page and now.shape[3] == d else None
        if now.dim() == 3:
            keep = ~mask[:, None, :]
        elif now is cache.tensors[1]:
            keep = ~mask[:, None, None, :]
        keep = keep.expand(now.shape)
        same = (now == then) | (now != now) & (then != then)
        assert bool(same[keep].all()), "a place of other tokens was written"


def test_cache_ties_and_special_rows(mx):
    """Halves round to even, and rows of zeros, of the least and largest numbers, of NaN and infinities."""
    d, page = 32, 16
    x = torch.zeros(9, 1, d, device="cuda")
    x[0, 0] = (torch.arange(d, device="cuda") - 15.5) * 2.0  # scale 2^k
    x[0, 0, 0] = 127.0 * 2
    x[1, 0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5], device="cuda")
    x[2, 0, 0] = 2.0 ** -149
    x[2, 0, 1] = 2.0 ** -142
    x[3, 0] = 3.4e38
    x[3, 0, ::2] *= -0.5
    x[4, 0, 7] = math.nan
    x[5, 0, 8] = math.inf
    x[6, 0, 9] = -math.inf
    x[7, 0, :3] = torch.tensor([1e-44, 5e-45, 3e-45], device="cuda")
    cache = new_cache(mx, gen(1), 3, 1, page, d, "i8")
    batch = mx.KVBatch(i32([[2, 0]]), i32([12]), 9)
    mx.kv_cache_write(cache, batch, x, x, stream=stream())
    k, v = torch.empty_like(x), torch.empty_like(x)
    mx.kv_cache_read(cache, batch, k, v, stream=stream())
    assert torch.equal(k.nan_to_num(77.0), v.nan_to_num(77.0))
    fine = [0, 1, 2, 3, 7, 8]
    ref = quantised(x)
    # one rounding, of half the least number at least
    within(k[fine], ref[fine], (U * ref.abs() + 2.0 ** -150)[fine], "rows")
    assert k[1, 0, :4].tolist() == [127.0, 0.0, 2.0, -2.0]
    assert bool(k[4:7].isnan().all()), "NaN and infinities"
    steps = cache.tensors[0][2, 0, 3:12].double()
    assert bool((steps.abs() <= 127).all()) and bool((cache.tensors[0][2, 0, 10] == 0).all()), "no steps of a scale of 0"
    # random rows and scales: every step is the rounding of the exact quotient
    g = gen(12)
    x = rand(g, 4000, 1, 128) * torch.exp2(torch.randint(-60, 60, (4000, 1, 1), device="cuda", generator=g).float())
    cache = new_cache(mx, g, 250, 1, page, 128, "i8")
    batch = mx.KVBatch(torch.arange(250, device="cuda", dtype=torch.int32)[None], i32([4000]), 4000)
    mx.kv_cache_write(cache, batch, x, x, stream=stream())
    scale = (x.double().abs().amax(-1) / 127).float()
    assert torch.equal(cache.tensors[2].flatten(), scale.flatten())
    want = torch.round(x.double() / scale.double()[..., None])
    assert torch.equal(cache.tensors[0].double().view(4000, 1, 128), want)
    assert torch.equal(cache.tensors[1].double().view(250, 128, page).transpose(1, 2).reshape(4000, 1, 128), want)


@pytest.mark.parametrize("kind", ["i8", "f32"])
def test_cache_absent_places(mx, kind):
    """Positions before the first, past the table and on no page are not written, and read as zero."""
    g, page, d, kv = gen(7), 16, 32, 2
    cache = new_cache(mx, g, 4, kv, page, d, kind)
    held = [t.clone() for t in cache.tensors if t is not None]
    table = i32([[1, -1, 2], [4, 2 ** 31 - 1, -2 ** 31], [0, 3, -5], [-1, -1, -1]])
    new, lengths = [40, 30, 10, 4], [45, 30, 4, 2 ** 31 - 1]
    t = sum(new)
    x = rand(g, t + 3, kv, d)  # three rows of no sequence
    batch = mx.KVBatch(table, i32(lengths), t + 3, starts_of(new))
    mx.kv_cache_write(cache, batch, x, -x, stream=stream())
    k, v = torch.full_like(x, TAIL), torch.full_like(x, TAIL)
    mx.kv_cache_read(cache, batch, k, v, stream=stream())
    there = torch.zeros(t + 3, dtype=torch.bool, device="cuda")
    # sequence 0: positions 5 .. 44 on pages 1, none, 2; sequence 2: positions -6 .. 3 on page 0
    there[0:11] = True    # 5 .. 15
    there[27:40] = True   # 32 .. 44
    there[70 + 6:80] = True
    exact = quantised(x) if kind == "i8" else x.double()
    within(k[there], exact[there], U * exact[there].abs(), "k")
    within(v[there], -exact[there], U * exact[there].abs(), "v")
    absent = ~there
    absent[t:] = False
    assert bool((k[absent] == 0).all()) and bool((v[absent] == 0).all())
    assert bool((k[t:] == TAIL).all()) and bool((v[t:] == TAIL).all()), "rows of no sequence"
    for now, then in zip([x for x in cache.tensors if x is not None], held):
        assert bool(((now[3] == then[3]) | (then[3] != then[3]) & (now[3] != now[3])).all()), "a page of no position"


# ---------------------------------------------------- attention over a cache
def paged_ref(q, k, v, pos, seen, scale):
    """One sequence: q [n, h, d], k and v [len, kv, d] in float64, seen [n, len]; (out, bound)."""
    h, kv, d = q.shape[1], k.shape[1], q.shape[2]
    q = q.double().transpose(0, 1)
    k, v = (t.transpose(0, 1).repeat_interleave(h // kv, 0) for t in (k, v))
    s = (scale * (q @ k.transpose(1, 2))).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0) * seen
    top = s.masked_fill(~seen, 0).abs().amax(-1, keepdim=True) if k.shape[1] else s.new_zeros(h, q.shape[1], 1)
    es = (d / 8 + 12) * U * abs(scale) * (q.abs() @ k.abs().transpose(1, 2)) * seen
    worst = es.amax(-1, keepdim=True) if k.shape[1] else s.new_zeros(h, q.shape[1], 1)
    rel = es + worst + 8 * U * (1 + top)
    deep = (k.shape[1] / 32 + 40) * U
    return (p @ v).transpose(0, 1), ((p * (rel + deep)) @ v.abs()).transpose(0, 1)


PAGED = [([1], [1], 16, 1, 1, 16, 0, 0), ([1], [33], 16, 4, 1, 32, 0, 0), ([1, 1], [500, 7], 64, 8, 2, 128, 0, 0),
         ([5], [5], 16, 2, 2, 80, 0, 0), ([40, 3], [100, 3], 32, 6, 2, 64, 0, 0), ([1] * 9, [60 * i + 1 for i in range(9)], 48, 3, 3, 96, 0, 0),
         ([1], [3000], 64, 16, 1, 128, 0, 0), ([2, 0, 1], [900, 4, 333], 16, 12, 4, 48, 100, 5), ([130], [700], 64, 4, 2, 112, 64, 40),
         ([70], [70], 16, 33, 1, 16, 1, 0), ([1, 30], [5000, 4000], 128, 2, 1, 64, 1000, 16), ([257], [2000], 32, 5, 5, 32, 0, 0),
         # chunks of many rows: packed tiles, keys of a row shared by workgroups, eight waves where there are rows enough
         ([400], [1100], 64, 8, 2, 128, 0, 0), ([330, 0, 350], [400, 90, 350], 16, 6, 2, 96, 100, 5), ([200, 210], [900, 210], 32, 16, 2, 48, 64, 40),
         ([900], [950], 128, 4, 4, 32, 0, 0), ([900] * 5, [901 + 13 * i for i in range(5)], 48, 60, 10, 64, 70, 2),
         ([1] * 3 + [2500], [5, 600, 1, 2600], 16, 3, 1, 80, 33, 1)]


def fill(mx, g, cache, table, lengths, page, kv, d, kind):
    """Every token of every sequence written; what the cache holds of them, in float64."""
    t = sum(lengths)
    k, v = rand(g, t, kv, d) * (rand(g, t, kv, 1).abs() + 0.3), rand(g, t, kv, d)
    mx.kv_cache_write(cache, mx.KVBatch(table, i32(lengths), t, starts_of(lengths)), k, v, stream=stream())
    return (quantised(k), quantised(v)) if kind == "i8" else (k.double(), v.double())


@pytest.mark.parametrize("new,lengths,page,h,kv,d,window,sinks", PAGED)
@pytest.mark.parametrize("kind", ["i8", "f32"])
def test_paged_attention(mx, new, lengths, page, h, kv, d, window, sinks, kind):
    print("paged", new[:4], lengths[:4], page, h, kv, d, window, sinks, kind, flush=True)
    g = gen(sum(lengths) + d)
    table, pages = tables(g, lengths, page)
    cache = new_cache(mx, g, pages, kv, page, d, kind)
    k, v = fill(mx, g, cache, table, lengths, page, kv, d, kind)
    if window:
        # Pages that the window has left are released: the table names none.
        for b, (n, length) in enumerate(zip(new, lengths)):
            for e in range(table.shape[1]):
                if e * page >= sinks and (e + 1) * page <= length - n - window + 1:
                    table[b, e] = -1
    t = sum(new)
    q = strided(g, t + 2, h, d, gap=1)  # two rows of no sequence
    batch = mx.KVBatch(table, i32(lengths), t + 2, starts_of(new))
    out, tail = guarded(t + 2, h, d)
    scale = 1.2 / math.sqrt(d)
    form = dict(window=window, sinks=sinks, scale=scale)
    mx.attention_paged(cache, batch, q, out, stream=stream(), **form)
    intact(tail)
    at = row = 0
    for n, length in zip(new, lengths):
        pos, keys = torch.arange(length - n, length, device="cuda"), torch.arange(length, device="cuda")
        back = pos[:, None] - keys[None, :]
        seen = (back >= 0) & ((back < window) | (keys < sinks)[None, :]) if window else back >= 0
        if n:
            ref, bound = paged_ref(q[row:row + n], k[at:at + length], v[at:at + length], pos, seen, scale)
            within(out[row:row + n], ref, bound + 1e-30, f"{n} of {length}")
        at, row = at + length, row + n
    assert bool((out[t:] == TAIL).all()), "rows of no sequence"
    ws = torch.empty(max(16, mx.attention_paged_workspace(cache, batch, h, window=window, sinks=sinks)), dtype=torch.uint8,
                     device="cuda")
    again = torch.full_like(out, TAIL)
    mx.attention_paged(cache, batch, q, again, workspace=ws, stream=stream(), **form)
    assert torch.equal(again, out), "the same call, other bits"


@pytest.mark.parametrize("kind", ["i8", "f32"])
def test_paged_rows_that_see_nothing_and_poison(mx, kind):
    """Empty sequences, positions before the first, absent pages: 0. NaN reaches only the rows that see it."""
    g, page, h, kv, d = gen(8), 16, 4, 2, 64
    lengths = [100, 60, 33]
    table, pages = tables(g, lengths, page)
    cache = new_cache(mx, g, pages, kv, page, d, kind)
    fill(mx, g, cache, table, lengths, page, kv, d, kind)
    q = rand(g, 24, h, d)
    run = lambda tab, lens, n, **form: (out := torch.full((sum(n), h, d), TAIL, device="cuda"), mx.attention_paged(
        cache, mx.KVBatch(tab, i32(lens), sum(n), starts_of(n)), q[:sum(n)], out, stream=stream(), **form))[0]
    seen = lambda out: bool((out != 0).any(-1).all())  # (single elements of 8 bits are 0 now and then)
    none = torch.full_like(table, -1)
    assert bool((run(none, lengths, [4, 4, 4]) == 0).all()), "no pages"
    out = run(table, [0, -3, 2], [4, 4, 4])
    assert bool((out[:10] == 0).all()) and seen(out[10:]), "positions before the first"
    assert seen(run(table, lengths, [4, 4, 4], window=2)[:4])
    gone = table.clone()
    gone[0, 4:] = pages + 9  # positions 64 .. are on no page of the cache
    out = run(gone, lengths, [4, 4, 4], window=8)
    assert bool((out[:4] == 0).all()) and seen(out[4:])
    # NaN in place 52 of the second sequence (of 60): its rows 52 .. see it, one key head.
    clean = run(table, lengths, [1, 12, 11])
    narrow = run(table, lengths, [1, 12, 11], window=5)
    k, v, ks, vs = cache.tensors
    at, slot = int(table[1, 52 // page]), 52 % page
    for which in ("k", "v"):
        x = (k if which == "k" else v) if kind == "f32" else (ks if which == "k" else vs)
        kept = x.clone()
        if kind == "i8":
            x[at, 1, slot] = math.nan
        elif which == "k":
            x[at, 1, slot, 9] = math.nan
        else:
            x[at, 1, 9, slot] = math.inf
        got, close = run(table, lengths, [1, 12, 11]), run(table, lengths, [1, 12, 11], window=5)
        x.copy_(kept)
        pos = torch.arange(48, 60, device="cuda")
        for out, want, reached in ((got, clean, pos >= 52), (close, narrow, (pos >= 52) & (pos < 57))):
            rows = torch.zeros(24, dtype=torch.bool, device="cuda")
            rows[1:13] = reached
            assert torch.equal(out[~rows], want[~rows]) and torch.equal(out[:, :2], want[:, :2]), which
            assert bool(out[rows][:, 2:].isnan().any(-1).all()), which


def test_paged_captured_and_on_another_stream(mx):
    g, page, h, kv, d = gen(10), 32, 8, 2, 128
    lengths = [2000, 700]
    table, pages = tables(g, lengths, page)
    cache = new_cache(mx, g, pages, kv, page, d, "i8")
    fill(mx, g, cache, table, lengths, page, kv, d, "i8")
    k, v, q = rand(g, 2, kv, d), rand(g, 2, kv, d), rand(g, 2, h, d)
    batch = mx.KVBatch(table, i32(lengths), 2)
    out = torch.empty_like(q)
    ws = torch.empty(max(16, mx.attention_paged_workspace(cache, batch, h)), dtype=torch.uint8, device="cuda")

    def call():
        mx.kv_cache_write(cache, batch, k, v, stream=stream())
        mx.attention_paged(cache, batch, q, out, workspace=ws, stream=stream())

    replay(call, [out], [q, k, v])
    # The batch's lengths are device data: a replayed graph sees them change.
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        batch.tensors[1].sub_(1)
        call()
        moved = out.clone()
        batch.tensors[1].add_(1)
        call()
    s.synchronize()
    assert not torch.equal(moved, out)


# ------------------------------------------------------- a layer, end to end
def test_prompt_then_tokens_equal_training(mx):
    """A sequence attended to at once, and as a prompt in two chunks and single tokens over an FP32 cache: the same
    rows within the bounds of both, and the rotation of a token alone has the bits of the whole."""
    g = gen(21)
    n, h, kv, d, page = 90, 4, 2, 64, 16
    x, y, v = rand(g, n, h, d), rand(g, n, kv, d), rand(g, n, kv, d)
    w, plan, pos = rand(g, d, mean=1.0, scale=0.1), mx.Rotary(frequencies(d)), torch.arange(n, device="cuda")
    turn = lambda r: (a := torch.empty_like(x[r]), b := torch.empty_like(y[r]), mx.qk_norm_rotary_forward(
        x[r], y[r], pos[r], plan, a, b, w, w, 1e-6, stream=stream()))[:2]
    q, k = turn(slice(0, n))
    whole = torch.empty_like(q)
    mx.attention_forward(q, k, v, whole, window=40, sinks=3, stream=stream())
    bound = attention_ref(q, k, v, torch.zeros_like(q), 40, 3, d ** -0.5)["out"][1] * 2
    cache = new_cache(mx, g, 8, kv, page, d, "f32")
    table = torch.randperm(8, device="cuda", generator=g)[None, :6].to(torch.int32).contiguous()
    at = 0
    for new in [33, 40] + [1] * 17:
        r = slice(at, at + new)
        at += new
        qs, ks = turn(r)
        assert torch.equal(qs, q[r]) and torch.equal(ks, k[r])
        batch = mx.KVBatch(table, i32([at]), new)
        mx.kv_cache_write(cache, batch, ks, v[r], stream=stream())
        out = torch.empty_like(qs)
        mx.attention_paged(cache, batch, qs, out, window=40, sinks=3, stream=stream())
        within(out, whole[r].double(), bound[r], f"rows {r}")


# ------------------------------------------------------------ sizes and streams
def test_paged_lengths_out_of_range(mx):
    """Lengths and starts that the contract excludes: absent places, rows of zeros, nothing out of range."""
    g, page, h, kv, d = gen(14), 16, 4, 2, 32
    for kind in ("i8", "f32"):
        for rows in (1, 200):  # both forms
            cache = new_cache(mx, g, 6, kv, page, d, kind)
            table = torch.arange(6, device="cuda", dtype=torch.int32).view(3, 2).contiguous()
            q, x = rand(g, 3 * rows, h, d), rand(g, 3 * rows, kv, d)
            for lengths in ([2 ** 31 - 1, -2 ** 31, 32], [40, 0, -1], [1 << 30, 33, -(1 << 30)]):
                for window in (0, 20):
                    batch = mx.KVBatch(table, i32(lengths), 3 * rows)
                    mx.kv_cache_write(cache, batch, x, x, stream=stream())
                    out, tail = guarded(3 * rows, h, d)
                    mx.attention_paged(cache, batch, q, out, window=window, sinks=3, stream=stream())
                    k, v = torch.empty_like(x), torch.empty_like(x)
                    mx.kv_cache_read(cache, batch, k, v, stream=stream())
                    intact(tail)
                    for b, n in enumerate(lengths):
                        if n <= 0:
                            assert bool((out[b * rows:(b + 1) * rows] == 0).all()) and bool((k[b * rows:(b + 1) * rows] == 0).all())


def test_calls_on_two_streams(mx):
    """The same calls on two streams at once, scratch from the allocator: each has its own results."""
    g, n, h, kv, d = gen(15), 700, 4, 2, 64
    inputs = [[rand(g, n, x, d) for x in (h, kv, kv, h)] for _ in range(2)]
    alone = [run_attention(mx, *x, None, window=100, sinks=3) for x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    for _ in range(3):
        both = []
        for s, x in zip(streams, inputs):
            with torch.cuda.stream(s):
                out, lse = torch.empty_like(x[0]), x[0].new_empty(h, n)
                dq, dk, dv = torch.empty_like(x[0]), torch.empty_like(x[1]), torch.empty_like(x[2])
                mx.attention_forward(*x[:3], out, lse=lse, window=100, sinks=3, stream=stream())
                mx.attention_backward(x[3], *x[:3], out, lse, dq, dk, dv, window=100, sinks=3, stream=stream())
                both.append(dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv))
        torch.cuda.synchronize()
        for got, want in zip(both, alone):
            assert all(torch.equal(got[x], want[x]) for x in want)


@pytest.fixture
def returned(mx):
    """What a large test took goes back to the card."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    mx.check(mx.lib().mx_empty_cache())


def test_attention_and_rotation_past_2_to_31_elements(mx, returned):
    """The last sequence of a batch of more than 2^31 elements."""
    g, h, d, n = gen(16), 130, 128, 300
    t = (1 << 31) // (h * d) + 2 * n
    tail = [rand(g, n, h, d) for _ in range(4)]
    q, k, v, do = (torch.zeros(t, h, d, device="cuda") for _ in tail)
    for x, y in zip((q, k, v, do), tail):
        x[-n:] = y
    starts, form = i32([0, n, t - n, t]), dict(window=33, sinks=2)
    scratch = torch.empty(mx.attention_workspace(t, 3, h, h, d, True, 33, 2), dtype=torch.uint8, device="cuda")
    plan, pos = mx.Rotary(frequencies(d)), torch.arange(t, device="cuda")
    out, small = torch.empty_like(q), torch.empty_like(tail[0])
    mx.qk_norm_rotary_forward(q, None, pos, plan, out, None, eps=1e-6, stream=stream())
    mx.qk_norm_rotary_forward(tail[0], None, pos[-n:].contiguous(), plan, small, None, eps=1e-6, stream=stream())
    assert torch.equal(out[-n:], small)
    lse = q.new_empty(h, t)
    mx.attention_forward(q, k, v, out, starts=starts, lse=lse, workspace=scratch, stream=stream(), **form)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    mx.attention_backward(do, q, k, v, out, lse, dq, dk, dv, starts=starts, workspace=scratch, stream=stream(), **form)
    got = dict(out=out[-n:], lse=lse[:, -n:], dq=dq[-n:], dk=dk[-n:], dv=dv[-n:])
    for name, (ref, bound) in attention_ref(*tail, 33, 2, d ** -0.5).items():
        within(got[name], ref, bound + 1e-30, name)


@pytest.mark.parametrize("kind", ["i8", "f32"])
def test_cache_past_2_to_31_elements(mx, returned, kind):
    g, page, h, kv, d = gen(17), 64, 8, 4, 128
    pages = (1 << 31) // (page * kv * d) + 40
    make = lambda *s, dtype: torch.empty(*s, dtype=dtype, device="cuda")
    e = torch.int8 if kind == "i8" else torch.float32
    k, v = make(pages, kv, page, d, dtype=e), make(pages, kv, d, page, dtype=e)
    scales = [make(pages, kv, page, dtype=torch.float32) for _ in range(2)] if kind == "i8" else []
    cache = mx.KVCache(k, v, *scales)
    table = torch.arange(pages - 10, pages, device="cuda", dtype=torch.int32)[None].contiguous()
    keys, values = rand(g, 640, kv, d), rand(g, 640, kv, d)
    batch = mx.KVBatch(table, i32([640]), 640)
    mx.kv_cache_write(cache, batch, keys, values, stream=stream())
    ko, vo = torch.empty_like(keys), torch.empty_like(values)
    mx.kv_cache_read(cache, batch, ko, vo, stream=stream())
    kr, vr = (quantised(keys), quantised(values)) if kind == "i8" else (keys.double(), values.double())
    within(ko, kr, U * kr.abs(), "k")
    within(vo, vr, U * vr.abs(), "v")
    for n in (1, 640):  # a token, and a chunk
        q = rand(g, n, h, d)
        out = torch.empty_like(q)
        mx.attention_paged(cache, mx.KVBatch(table, i32([640]), n), q, out, stream=stream())
        pos, at = torch.arange(640 - n, 640, device="cuda"), torch.arange(640, device="cuda")
        ref, bound = paged_ref(q, kr, vr, pos, pos[:, None] >= at[None, :], d ** -0.5)
        within(out, ref, bound + 1e-30, f"{n} rows")


# ------------------------------------------------------- sizes and values at the borders
@pytest.mark.parametrize("kind", ["i8", "f32"])
@pytest.mark.parametrize("new,length", [(1, 1500), (3, 3000), (500, 1500)])
def test_paged_largest_windows_see_everything(mx, new, length, kind):
    """A window that no sequence fills is none at all, however large the number."""
    g, page, h, kv, d = gen(length + new), 64, 8, 2, 64
    table, pages = tables(g, [length], page)
    cache = new_cache(mx, g, pages, kv, page, d, kind)
    fill(mx, g, cache, table, [length], page, kv, d, kind)
    q, batch = rand(g, new, h, d), mx.KVBatch(table, i32([length]), new)
    run = lambda window: (out := torch.full_like(q, TAIL), mx.attention_paged(
        cache, batch, q, out, window=window, stream=stream()))[0]
    whole = run(0)
    for window in (2 ** 31, 2 ** 40, 2 ** 63 - 200, 2 ** 63 - 1):
        assert torch.equal(run(window), whole), window


def test_attention_largest_windows_see_everything(mx):
    g, n = gen(31), 700
    x = [rand(g, n, h, 64) for h in (4, 2, 2, 4)]
    whole = run_attention(mx, *x, None)
    for window in (2 ** 31, 2 ** 63 - 1):
        got = run_attention(mx, *x, None, window=window, sinks=2 ** 63 - 1)
        assert all(torch.equal(got[name], whole[name]) for name in whole), window


@pytest.mark.parametrize("kind", ["i8", "f32"])
@pytest.mark.parametrize("new,length,window", [(1, 130, 70), (5, 140, 70), (7, 200, 100), (100, 229, 150), (100, 300, 190)])
def test_paged_positions_past_the_table(mx, new, length, window, kind):
    """New tokens behind the table's 128 places, with a window that ends inside it: each sees its own window's keys."""
    g, page, h, kv, d, places = gen(length + new), 64, 16, 2, 64, 128
    table, pages = tables(g, [places], page)
    cache = new_cache(mx, g, pages, kv, page, d, kind)
    k, v = fill(mx, g, cache, table, [places], page, kv, d, kind)
    q, out = rand(g, new, h, d), torch.empty(new, h, d, device="cuda")
    mx.attention_paged(cache, mx.KVBatch(table, i32([length]), new), q, out, window=window, stream=stream())
    pos, keys = torch.arange(length - new, length, device="cuda"), torch.arange(places, device="cuda")
    back = pos[:, None] - keys[None, :]
    ref, bound = paged_ref(q, k, v, pos, (back >= 0) & (back < window), d ** -0.5)
    within(out, ref, bound + 1e-30, "rows past the table")
    if kind == "f32":
        # The keys before the last row's window hold anything.
        first = int(pos[-1]) - window + 1
        page_of, slot = int(table[0, (first - 1) // page]), (first - 1) % page
        cache.tensors[0][page_of, 0, slot] = math.nan
        again = torch.empty_like(out)
        mx.attention_paged(cache, mx.KVBatch(table, i32([length]), new), q, again, window=window, stream=stream())
        assert torch.equal(again[-1], out[-1])


@pytest.mark.parametrize("kind", ["i8", "f32"])
@pytest.mark.parametrize("new", [1, 100])
def test_paged_far_positions_and_large_windows(mx, new, kind):
    """Positions past 2^30, whose window of 2^30 or more reaches a short table's keys: in part or whole."""
    g, page, h, kv, d, places = gen(new), 32, 16, 2, 64, 64
    table, pages = tables(g, [places], page)
    cache = new_cache(mx, g, pages, kv, page, d, kind)
    k, v = fill(mx, g, cache, table, [places], page, kv, d, kind)
    q = rand(g, new, h, d)
    keys = torch.arange(places, device="cuda")
    for length in (2 ** 30 + 40, 2 ** 31 - 1):
        pos = torch.arange(length - new, length, device="cuda")
        back = pos[:, None] - keys[None, :]
        for window in (2 ** 30, 2 ** 30 + 77, 2 ** 31 - 30, 2 ** 31 - 1, 2 ** 40, 2 ** 63 - 1):
            out = torch.empty_like(q)
            mx.attention_paged(cache, mx.KVBatch(table, i32([length]), new), q, out, window=window, stream=stream())
            ref, bound = paged_ref(q, k, v, pos, back < window, d ** -0.5)
            within(out, ref, bound + 1e-30, f"length {length}, window {window}")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 64), (20, 12), (22, 10), (65, 34), (255, 198), (7, 2)])
def test_rotary_elements_behind_the_turned_part_stay_alone(mx, dim, rot, interleaved):
    """Elements past rotary_dim pass through, whatever they and their neighbours hold."""
    g, tokens, h = gen(dim), 9, 3
    plan, pos = mx.Rotary(frequencies(rot), interleaved=interleaved, magnitude=1.25), torch.arange(tokens, device="cuda")
    x = rand(g, tokens, h, dim)
    forward = lambda t, **kw: (out := torch.empty_like(t), mx.qk_norm_rotary_forward(
        t, None, pos, plan, out, None, stream=stream(), **kw))[0]
    backward = lambda t, **kw: (out := torch.empty_like(t), mx.qk_norm_rotary_backward(
        t, None, None, None, pos, plan, out, None, stream=stream(), **kw))[0]
    for turn in (forward, backward):
        clean = turn(x)
        assert torch.equal(clean[..., rot:], x[..., rot:])
        for value in (math.inf, -math.inf, math.nan, 3.4e38):
            for e in {rot, rot + (dim - rot) // 2, dim - 1}:
                y = x.clone()
                y[4, 1, e] = value
                got = turn(y)
                assert torch.equal(got[4, 1, e].nan_to_num(7.0, 8.0, 9.0), y[4, 1, e].nan_to_num(7.0, 8.0, 9.0)), (e, value)
                got[4, 1, e] = x[4, 1, e]
                assert torch.equal(got, clean), (e, value)
    # An infinite weight of one such element, under a norm.
    w = rand(g, dim, mean=1.0, scale=0.1)
    clean = forward(x, q_weight=w, eps=1e-6)
    for e in {rot, dim - 1}:
        v = w.clone()
        v[e] = math.inf
        got = forward(x, q_weight=v, eps=1e-6)
        assert torch.equal(got[..., e], x[..., e].sign() * math.inf), e
        got[..., e] = clean[..., e]
        assert torch.equal(got, clean), e


def test_attention_keeps_huge_values_that_are_not_seen_apart(mx):
    """The largest finite numbers, and queries that the scale takes past them, change no bit of rows that do not see them."""
    g = gen(6)
    lengths, h, kv, d, window, sinks = [90, 100, 75], 4, 2, 64, 20, 2
    t = sum(lengths)
    q, k, v, do = rand(g, t, h, d), rand(g, t, kv, d), rand(g, t, kv, d), rand(g, t, h, d)
    bad = 90 + 47
    rows = torch.arange(t, device="cuda")
    reached = (rows >= bad) & (rows < bad + window)
    touched = ((rows > bad - window) & (rows < bad + window)) | ((rows >= 90) & (rows < 90 + sinks))
    keys = ((rows > bad - window) & (rows <= bad)) | ((rows >= 90) & (rows < 90 + sinks))
    most = torch.finfo(torch.float32).max
    for scale in (0.125, 4.0):
        form = dict(window=window, sinks=sinks, scale=scale)
        clean = run_attention(mx, q, k, v, do, starts_of(lengths), **form)
        for value in (most, -most, 0.9975 * most, 1e38):
            for where in ("k", "v"):
                x = dict(k=k.clone(), v=v.clone())
                x[where][bad, 1, 3] = value
                got = run_attention(mx, q, x["k"], x["v"], do, starts_of(lengths), **form)
                for name in ("out", "dq"):
                    assert torch.equal(got[name][~reached], clean[name][~reached]), (name, where, value)
                    assert torch.equal(got[name][:, :2], clean[name][:, :2]), "the other key head's rows"
                for name in ("dk", "dv"):
                    assert torch.equal(got[name][~touched], clean[name][~touched]), (name, where, value)
                    assert torch.equal(got[name][:, 0], clean[name][:, 0])
            for where in ("q", "do"):
                x = dict(q=q.clone(), do=do.clone())
                x[where][bad, 3, 0] = value
                got = run_attention(mx, x["q"], k, v, x["do"], starts_of(lengths), **form)
                for name in ("out", "dq"):
                    assert torch.equal(got[name][rows != bad], clean[name][rows != bad]), (name, where, value)
                for name in ("dk", "dv"):
                    assert torch.equal(got[name][~keys], clean[name][~keys]), (name, where, value)


@pytest.mark.parametrize("new", [4, 140])
def test_paged_keeps_huge_values_that_are_not_seen_apart(mx, new):
    g, page, h, kv, d, length, window = gen(11), 16, 4, 2, 64, 300, 150
    table, pages = tables(g, [length], page)
    cache = new_cache(mx, g, pages, kv, page, d, "f32")
    fill(mx, g, cache, table, [length], page, kv, d, "f32")
    q = rand(g, new, h, d)
    run = lambda: (out := torch.empty_like(q), mx.attention_paged(
        cache, mx.KVBatch(table, i32([length]), new), q, out, window=window, stream=stream()))[0]
    clean = run()
    j = length - new - window + 2  # seen by the first two rows or so, and by no later one
    reached = torch.arange(length - new, length, device="cuda") - j < window
    at, slot = int(table[0, j // page]), j % page
    most = torch.finfo(torch.float32).max
    for which in (0, 1):
        x = cache.tensors[which][at, 1, slot] if which == 0 else cache.tensors[which][at, 1, :, slot]
        kept = x.clone()
        for value in (most, -most, math.inf):
            x[9] = value
            got = run()
            assert torch.equal(got[~reached], clean[~reached]) and torch.equal(got[:, :2], clean[:, :2]), (which, value)
        x.copy_(kept)


@pytest.mark.parametrize("kind", ["i8", "f32"])
@pytest.mark.parametrize("new", [1, 110])
def test_paged_rows_that_see_a_bad_value_with_no_probability(mx, new, kind):
    """A value that is not finite makes the rows that see it NaN also where its probability is 0."""
    g, page, h, kv, d, length = gen(12), 16, 16, 2, 64, 250
    table, pages = tables(g, [length], page)
    cache = new_cache(mx, g, pages, kv, page, d, kind)
    k = torch.full((length, kv, d), -8.0, device="cuda")
    k[10] = 8.0
    v = rand(g, length, kv, d)
    v[20, 1, 5] = math.nan
    mx.kv_cache_write(cache, mx.KVBatch(table, i32([length]), length), k, v, stream=stream())
    q, out = torch.full((new, h, d), 8.0, device="cuda"), torch.empty(new, h, d, device="cuda")
    mx.attention_paged(cache, mx.KVBatch(table, i32([length]), new), q, out, stream=stream())
    within(out[:, :8], v[10, 0].double() if kind == "f32" else quantised(v[10])[0], 64 * U * v[10, 0].double().abs(), "the other key head")
    assert bool(out[:, 8:, 5].isnan().all()), kind


def test_attention_backward_without_query_heads(mx):
    """Key heads that no query head shares have gradients of 0, in the sequences' rows alone."""
    g = gen(13)
    k = rand(g, 50, 2, 40)
    none = torch.empty(50, 0, 40, device="cuda")
    starts = starts_of([20, 0, 23], 3)
    for want in ((True, True), (True, False), (False, True)):
        outs = [guarded(50, 2, 40) if w else (None, None) for w in want]
        mx.attention_backward(none, none, k, k, none, torch.empty(0, 50, device="cuda"), torch.empty_like(none), outs[0][0],
                              outs[1][0], starts=starts, stream=stream())
        for x, tail in outs:
            if x is not None:
                intact(tail)
                assert bool((x[3:46] == 0).all())
    x = torch.full((50, 2, 40), TAIL, device="cuda")
    mx.attention_backward(none, none, k, k, none, torch.empty(0, 50, device="cuda"), None, x, None, starts=starts, stream=stream())
    assert bool((x[:3] == TAIL).all()) and bool((x[46:] == TAIL).all()), "rows of no sequence"


def test_rotary_angles(mx):
    """Cosines and sines themselves: pairs (1, 0) are turned into them.  The functions are off by a step at most
    (u for values above 1/2), the correction by what the angle's rounding left is rounded once (u / 2)."""
    g = gen(14)
    freqs = frequencies(128)
    plan, pos = mx.Rotary(freqs), torch.randint(0, 1 << 20, (4000,), device="cuda", generator=g)
    x = torch.cat([torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")]).expand(4000, 1, 128)
    out = torch.empty(4000, 1, 128, device="cuda")
    mx.qk_norm_rotary_forward(x, None, pos, plan, out, None, stream=stream())
    a = (pos.double()[:, None, None] * torch.tensor(freqs, dtype=torch.double, device="cuda"))
    ref = torch.cat([torch.cos(a), torch.sin(a)], -1)
    within(out, ref, 1.5 * U * torch.ones_like(ref), "cosines and sines")
