"""torch_vulkan.nn's rotation, attention, cache, attention layer and the decoder example
on the "vulkan" device against CPU torch, with the CPU fallback forbidden.

Parity bar: |err| <= 1e-4 |ref| + 1e-5 max(1, magnitude) against float64, the
bar of the other operators on this device (tests/helpers.py)."""
import importlib.util
import math
import os

import pytest
import torch

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


def seen(n, window, sinks):
    i = torch.arange(n)
    back = i[:, None] - i[None, :]
    return (back >= 0) & ((back < window) | (i < sinks)[None, :]) if window else back >= 0


def attention_ref(q, k, v, lengths, window=0, sinks=0, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    group, outs, at = q.shape[1] // k.shape[1], [], 0
    for n in lengths:
        a, b, c = q[at:at + n].transpose(0, 1), k[at:at + n].transpose(0, 1), v[at:at + n].transpose(0, 1)
        s = scale * a @ b.repeat_interleave(group, 0).transpose(1, 2)
        p = torch.softmax(s.masked_fill(~seen(n, window, sinks), -math.inf), -1)
        outs.append((p @ c.repeat_interleave(group, 0)).transpose(0, 1))
        at += n
    return torch.cat(outs + [q.new_zeros(len(q) - at, *q.shape[1:])])


def rotary_ref(x, w, positions, freqs, interleaved, magnitude, eps):
    if eps is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 if w is None else w)
    r = 2 * len(freqs)
    a = positions.double()[:, None, None] * torch.tensor(freqs, dtype=torch.double)
    c, s = torch.cos(a) * magnitude, torch.sin(a) * magnitude
    p, q = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    one, two = p * c - q * s, q * c + p * s
    turned = torch.stack([one, two], -1).flatten(-2) if interleaved else torch.cat([one, two], -1)
    return torch.cat([turned, x[..., r:]], -1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [None, "plain", "weights"])
def test_qk_norm_rotary(interleaved, norm):
    from torch_vulkan.nn import qk_norm_rotary, rotary_frequencies
    g = torch.Generator().manual_seed(1)
    t, hq, hk, d = 37, 6, 2, 48
    freqs, pos = rotary_frequencies(32, factor=4.0, trained=512), torch.randint(0, 5000, (t,), generator=g)
    eps = None if norm is None else 1e-6
    leaves = [torch.randn(t, hq, d, generator=g), torch.randn(t, hk, d, generator=g)]
    if norm == "weights":
        leaves += [1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g)]
    dy = [torch.randn(t, hq, d, generator=g), torch.randn(t, hk, d, generator=g)]
    r, v = [x.double().requires_grad_() for x in leaves], [x.to("vulkan").requires_grad_() for x in leaves]
    form = dict(interleaved=interleaved, magnitude=1.1, eps=eps)
    wr, wv = (r[2:], v[2:]) if norm == "weights" else ([None, None], [None, None])
    yr = [rotary_ref(r[i], wr[i], pos, freqs, interleaved, 1.1, eps) for i in range(2)]
    yv = qk_norm_rotary(v[0], v[1], pos.to("vulkan"), freqs, q_weight=wv[0], k_weight=wv[1], **form)
    gr = torch.autograd.grad(yr, r, [x.double() for x in dy])
    gv = torch.autograd.grad(yv, v, [x.to("vulkan") for x in dy])
    for name, a, b in zip(("q", "k"), yv, yr):
        assert_close_mag(a, b, what=name)
    for name, a, b in zip(("dq", "dk", "dqw", "dkw"), gv, gr):
        assert_close_mag(a, b, b.abs() + 8, what=name)


def test_rotary_frequencies():
    from torch_vulkan.nn import rotary_frequencies
    plain = rotary_frequencies(64)
    assert plain[0] == 1.0 and len(plain) == 32 and abs(plain[31] - 10000 ** (-62 / 64)) < 1e-12
    assert rotary_frequencies(64, factor=4.0) == [f / 4 for f in plain]
    parts = rotary_frequencies(64, factor=4.0, trained=2048)
    assert parts[0] == plain[0] and parts[-1] == plain[-1] / 4
    assert all(f / 4 <= p <= f for p, f in zip(parts, plain)) and any(f / 4 < p < f for p, f in zip(parts, plain))
    for bad in (dict(rotary_dim=3), dict(rotary_dim=4, base=0.0), dict(rotary_dim=4, factor=-1.0),
                dict(rotary_dim=4, trained=8, turns=(2.0, 1.0))):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 2)])
def test_attention(window, sinks):
    from torch_vulkan.nn import attention
    g = torch.Generator().manual_seed(3)
    lengths, h, kv, d = [33, 1, 50], 6, 2, 40
    t = sum(lengths) + 3  # rows of no sequence: zeros
    leaves = [torch.randn(t, h, d, generator=g), torch.randn(t, kv, d, generator=g), torch.randn(t, kv, d, generator=g)]
    dy = torch.randn(t, h, d, generator=g)
    starts = torch.tensor([0, 33, 34, 84], dtype=torch.int32)
    r, v = [x.double().requires_grad_() for x in leaves], [x.to("vulkan").requires_grad_() for x in leaves]
    yr = attention_ref(*r, lengths, window, sinks)
    yv = attention(*v, starts=starts.to("vulkan"), window=window, sinks=sinks)
    assert_close_mag(yv, yr, what="out")
    for name, a, b in zip(("dq", "dk", "dv"), torch.autograd.grad(yv, v, dy.to("vulkan")), torch.autograd.grad(yr, r, dy.double())):
        assert_close_mag(a, b, b.abs() + 8, what=name)
        assert bool((a.cpu()[84:] == 0).all())


def test_attention_views_of_one_projection():
    from torch_vulkan.nn import attention
    g = torch.Generator().manual_seed(4)
    t, kv, d = 40, 2, 32
    q, both = torch.randn(4, t, d, generator=g), torch.randn(t, 2 * kv * d, generator=g)
    qv = q.to("vulkan").requires_grad_()
    bv = both.to("vulkan").requires_grad_()
    k, v = (x.view(t, kv, d) for x in bv.split(kv * d, 1))
    y = attention(qv.transpose(0, 1), k, v, sequences=2)
    qr, br = q.double().requires_grad_(), both.double().requires_grad_()
    k, v = (x.reshape(t, kv, d) for x in br.split(kv * d, 1))
    yr = attention_ref(qr.transpose(0, 1), k, v, [20, 20])
    assert_close_mag(y, yr)
    y.sum().backward()
    yr.sum().backward()
    assert_close_mag(qv.grad, qr.grad, qr.grad.abs() + 8)
    assert_close_mag(bv.grad, br.grad, br.grad.abs() + 8)
    # only one of the gradients, of a leaf without the others
    k = both[:, :kv * d].reshape(t, kv, d)
    kv_only = k.to("vulkan").requires_grad_()
    attention(q.transpose(0, 1).to("vulkan"), kv_only, k.to("vulkan")).sum().backward()
    kr = k.double().requires_grad_()
    attention_ref(q.transpose(0, 1).double(), kr, k.double(), [t]).sum().backward()
    assert_close_mag(kv_only.grad, kr.grad, kr.grad.abs() + 8)


def quantised(x):
    scale = (x.double().abs().amax(-1, keepdim=True) / 127).float().double()
    return torch.where(scale > 0, torch.round(x.double() / scale), 0.0) * scale


@pytest.mark.parametrize("dtype", [torch.int8, torch.float32])
def test_cache(dtype):
    from torch_vulkan.nn import KVCache
    g = torch.Generator().manual_seed(5)
    lengths, h, kv, d, page = [50, 3, 20], 4, 2, 48, 16
    t = sum(lengths)
    k, v, q = (torch.randn(t, n, d, generator=g) for n in (kv, kv, h))
    cache = KVCache(16, kv, page, d, dtype)
    table = torch.randperm(16, generator=g)[:12].view(3, 4).to(torch.int32)
    starts = torch.tensor([0, 50, 53, 73], dtype=torch.int32)
    batch = dict(table=table.to("vulkan"), lengths=torch.tensor(lengths, dtype=torch.int32).to("vulkan"), starts=starts.to("vulkan"))
    cache.write(k.transpose(0, 1).contiguous().to("vulkan").transpose(0, 1), v.to("vulkan"), **batch)
    kr, vr = (quantised(k), quantised(v)) if dtype == torch.int8 else (k.double(), v.double())
    ko, vo = cache.read(t, **batch)
    assert_close_mag(ko, kr, what="k")
    assert_close_mag(vo, vr, what="v")
    out = cache.attention(q.to("vulkan"), window=17, sinks=1, **batch)
    assert_close_mag(out, attention_ref(q.double(), kr, vr, lengths, 17, 1), what="a prompt")
    # a token of each, without starts
    last = [49, 52, 72]
    one = cache.attention(q[last].to("vulkan"), batch["table"], batch["lengths"], window=17, sinks=1)
    assert_close_mag(one, out.cpu().double()[last], what="a token")


def test_refusals():
    from torch_vulkan.nn import Attention, KVCache, attention, qk_norm_rotary
    x = lambda *s: torch.zeros(*s).to("vulkan")
    with pytest.raises(RuntimeError, match="float32|Float"):
        attention(torch.zeros(2, 2, 8, dtype=torch.float64).to("vulkan"), x(2, 2, 8), x(2, 2, 8))
    with pytest.raises(RuntimeError, match="do not fit"):
        attention(x(2, 2, 8), x(3, 2, 8), x(3, 2, 8))
    with pytest.raises(RuntimeError, match="evenly"):
        attention(x(2, 3, 8), x(2, 2, 8), x(2, 2, 8))
    with pytest.raises(RuntimeError, match="head_dim"):
        attention(x(2, 2, 136), x(2, 2, 136), x(2, 2, 136))
    with pytest.raises(RuntimeError, match="do not divide"):
        attention(x(5, 2, 8), x(5, 2, 8), x(5, 2, 8), sequences=2)
    with pytest.raises(RuntimeError, match="starts"):
        attention(x(2, 2, 8), x(2, 2, 8), x(2, 2, 8), starts=torch.tensor([0, 2]).to("vulkan"))
    with pytest.raises(RuntimeError, match="vulkan"):
        attention(x(2, 2, 8), x(2, 2, 8), torch.zeros(2, 2, 8))
    with pytest.raises(RuntimeError, match="positions"):
        qk_norm_rotary(x(2, 2, 8), x(2, 1, 8), None, [1.0])
    with pytest.raises(RuntimeError, match="without a norm"):
        qk_norm_rotary(x(2, 2, 8), x(2, 1, 8), None, [], q_weight=x(8))
    with pytest.raises(RuntimeError, match="rotary_dim"):
        qk_norm_rotary(x(2, 2, 8), x(2, 1, 8), torch.zeros(2, dtype=torch.int64).to("vulkan"), [1.0] * 5)
    with pytest.raises(ValueError, match="multiples of 16"):
        KVCache(4, 2, 20, 32)
    with pytest.raises(ValueError, match="dtype"):
        KVCache(4, 2, 16, 32, torch.float16)
    cache = KVCache(4, 2, 16, 32)
    batch = dict(table=torch.zeros(1, 2, dtype=torch.int32).to("vulkan"), lengths=torch.ones(1, dtype=torch.int32).to("vulkan"))
    with pytest.raises(RuntimeError, match="do not fit"):
        cache.write(x(1, 1, 32), x(1, 1, 32), **batch)
    with pytest.raises(RuntimeError, match="does not fit"):
        cache.attention(x(1, 2, 16), **batch)
    with pytest.raises(RuntimeError, match="lengths"):
        cache.attention(x(1, 2, 32), batch["table"], torch.ones(2, dtype=torch.int32).to("vulkan"))
    with pytest.raises(ValueError, match="evenly"):
        Attention(32, 4, 3)


def decoder():
    spec = importlib.util.spec_from_file_location("decoder", os.path.join(REPO, "pytorch-vulkan_amd", "examples", "decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def cpu_decoder(model, x, positions, lengths):
    """The example's model on the CPU in float64, from its parameters."""
    F = torch.nn.functional
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in model.named_parameters()}
    h = x.double()
    for i, block in enumerate(model.blocks):
        at, n = f"blocks.{i}.", block.attention
        y = F.layer_norm(h, h.shape[-1:], p[at + "norm1.weight"], p[at + "norm1.bias"])
        q, k, v = (F.linear(y, p[at + f"attention.{s}.weight"]).view(len(x), -1, n.head_dim) for s in "qkv")
        q = rotary_ref(q, p[at + "attention.q_weight"], positions, n.frequencies, False, 1.0, n.eps)
        k = rotary_ref(k, p[at + "attention.k_weight"], positions, n.frequencies, False, 1.0, n.eps)
        o = attention_ref(q, k, v, lengths, n.window, n.sinks).reshape(len(x), -1)
        h = h + F.linear(o, p[at + "attention.out.weight"])
        y = F.layer_norm(h, h.shape[-1:], p[at + "norm2.weight"], p[at + "norm2.bias"])
        u = F.gelu(F.linear(y, p[at + "up.weight"], p[at + "up.bias"]))
        h = h + F.linear(u, p[at + "down.weight"], p[at + "down.bias"])
    return h, p


def test_decoder_gradients():
    m = decoder()
    model, lengths = m.build(64, heads=4, kv_heads=2, window=12, sinks=2).to("vulkan"), [30, 1, 41]
    x, positions, starts, target = m.data(lengths, 64)
    y = model(x.to("vulkan"), positions.to("vulkan"), starts.to("vulkan"))
    ref, p = cpu_decoder(model, x, positions, lengths)
    assert_close_mag(y, ref, ref.abs() + 8, what="out")
    torch.nn.functional.mse_loss(y, target.to("vulkan")).backward()
    torch.nn.functional.mse_loss(ref, target.double()).backward()
    for name, t in model.named_parameters():
        assert_close_mag(t.grad, p[name].grad, what=name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8])
def test_decoder_serves_what_it_computes_at_once(dtype):
    """Tokens from the cache are the rows that the whole sequence has; 8 bits keep them near."""
    m = decoder()
    model = m.build(64, heads=4, kv_heads=2, window=12, sinks=2).to("vulkan")
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randn(n, 64, generator=g) for n in (20, 3, 33)]
    out = m.serve(model, prompts, 6, dtype)
    for prompt, rows in zip(prompts, out):
        whole = torch.cat([prompt, rows[:-1]])
        ref, _ = cpu_decoder(model, whole, torch.arange(len(whole)), [len(whole)])
        ref = ref.detach()[len(prompt) - 1:]
        if dtype == torch.float32:
            assert_close_mag(rows, ref, ref.abs() + 8)
        else:
            assert float((rows.double() - ref).norm() / ref.norm()) < 0.05


def test_decoder_trains_on_a_stream(vk):
    m = decoder()
    model = m.build(32, heads=2, kv_heads=1).to("vulkan")
    batch = [t.to("vulkan") for t in m.data([20, 30], 32)]
    s = vk.Stream()
    s.wait_stream(vk.current_stream())
    with s:
        losses = m.train(model, *batch, 3)
    vk.current_stream().wait_stream(s)
    assert all(math.isfinite(x) for x in losses)


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8])
def test_layer_with_the_largest_window(dtype):
    """window=2 ** 63 - 1 is no window, in training and in serving: a prompt and a token over more keys than a workgroup takes."""
    from torch_vulkan.nn import Attention, KVCache
    torch.manual_seed(9)
    n, page = 1300, 64
    layers = [Attention(64, 4, 2, window=w) for w in (0, 2 ** 63 - 1)]
    layers[1].load_state_dict(layers[0].state_dict())
    x, positions = torch.randn(n, 64).to("vulkan"), torch.arange(n).to("vulkan")
    table, count = torch.arange(22, dtype=torch.int32)[None].to("vulkan"), lambda v: torch.tensor([v], dtype=torch.int32).to("vulkan")
    outs = []
    for layer in layers:
        layer.to("vulkan")
        cache = KVCache(22, 2, page, 16, dtype)
        with torch.no_grad():
            outs.append([layer(x, positions).cpu(),
                         layer(x[:-1], positions[:-1], cache=cache, table=table, lengths=count(n - 1)).cpu(),
                         layer(x[-1:], positions[-1:], cache=cache, table=table, lengths=count(n)).cpu()])
    for none, largest in zip(*outs):
        assert torch.equal(none, largest)


def test_key_heads_without_query_heads():
    """Their gradients are zeros, not memory as it was."""
    from torch_vulkan.nn import attention
    k, v = (torch.randn(40, 2, 32).to("vulkan").requires_grad_() for _ in range(2))
    attention(torch.empty(40, 0, 32).to("vulkan"), k, v, scale=1.0).sum().backward()
    for x in (k, v):
        assert bool((x.grad.cpu() == 0).all())
