"""The attention layer of a language model, in training and in serving, as cases that can be timed.

Four operators that belong together, FP32 outside and in the sums: the norm and
rotation of queries and keys, causal attention over packed sequences (sliding
window, first tokens that stay visible, shared key heads) with its gradients,
the paged cache of keys and values as it is written and read back, and
attention of new tokens over that cache.  ``listed()`` names twelve pieces of
such work, ``draw()`` gives others of the same ranges, ``run()`` passes one of
them through elementary torch operations or, where ``own`` is true, through
this backend's kernels (``torch_vulkan.mx`` on the tensors' own device
pointers), and ``exact()`` restates it in float64.

Case fields: ``kind`` selects the operator, the others are its sizes.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-vulkan_amd")

EPS = 1e-6           # norm of queries and keys
BASE = 10000.0       # rotation: frequencies BASE^(-2 i / rotary_dim)


def listed():
    return [
        # One decoded token through the rotation alone, neighbouring elements
        # paired, half of the head turned: latency.
        dict(name="rotary_token", kind="rotary", tokens=1, heads=16, kv_heads=4, dim=128, rotary=64, interleaved=True,
             norm=False, factor=1.0, train=False),
        # A training micro-batch, norm and rotation forward and all gradients.
        dict(name="rotary_train", kind="rotary", tokens=8192, heads=16, kv_heads=4, dim=128, rotary=128, interleaved=False,
             norm=True, factor=4.0, train=True),
        # A small training step of four short sequences.
        dict(name="attention_short_train", kind="attention", lengths="256 256 256 256", heads=12, kv_heads=12, dim=64,
             window=0, sinks=0, train=True),
        # Training, two sequences, four query heads to a key head.
        dict(name="attention_train", kind="attention", lengths="2048 2048", heads=16, kv_heads=4, dim=128, window=0,
             sinks=0, train=True),
        # Documents of odd lengths packed behind each other, an odd head, a
        # window and visible first tokens, forward and gradients.
        dict(name="attention_packed_train", kind="attention", lengths="1 733 1291 64 65 2048 17 787", heads=12, kv_heads=3,
             dim=80, window=512, sinks=4, train=True),
        # A long prompt through a layer with a window: forward alone.
        dict(name="attention_long_prompt", kind="attention", lengths="16384", heads=16, kv_heads=16, dim=64, window=4096,
             sinks=4, train=False),
        # A decoding step of 64 sequences: a token each into an unquantised cache, and back.
        dict(name="cache_step_f32", kind="cache", sequences=64, new=1, context=2048, heads=16, kv_heads=4, dim=128, page=16,
             type="f32", spread=0.5),
        # Three prompts quantised into the cache, and read back.
        dict(name="cache_prompt_i8", kind="cache", sequences=3, new=1365, context=2000, heads=16, kv_heads=8, dim=128,
             page=64, type="i8", spread=0.3),
        # One sequence decodes one token: latency, the keys shared out over the chip.
        dict(name="paged_token_i8", kind="paged", sequences=1, new=1, context=4096, heads=16, kv_heads=4, dim=128, page=64,
             type="i8", spread=0.0, window=0, sinks=0),
        # A decoding step of 64 sequences of uneven lengths.
        dict(name="paged_batch_i8", kind="paged", sequences=64, new=1, context=8192, heads=32, kv_heads=8, dim=128, page=64,
             type="i8", spread=0.9, window=0, sinks=0),
        # The same over an unquantised cache, odd sizes, every query head with keys of its own.
        dict(name="paged_batch_f32", kind="paged", sequences=17, new=2, context=3001, heads=9, kv_heads=9, dim=80, page=16,
             type="f32", spread=0.7, window=0, sinks=0),
        # Chunks of 512 new tokens of four long prompts, under a window with visible first tokens.
        dict(name="paged_chunk_i8", kind="paged", sequences=4, new=512, context=12288, heads=16, kv_heads=4, dim=128,
             page=64, type="i8", spread=0.2, window=4096, sinks=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def _heads(rng, most):
    kv = _log(rng, 1, 16)
    return kv * rng.choice([g for g in (1, 1, 2, 3, 4, 6, 8, 16) if kv * g <= most]), kv


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "attention", "attention", "attention", "cache", "paged", "paged", "paged"])
    if kind == "rotary":
        heads, kv = _heads(rng, 32)
        dim = 2 * _log(rng, 8, 64) if rng.random() < 0.5 else rng.choice([32, 64, 96, 128])
        tokens = max(1, min(_log(rng, 1, 32768), 8192 * 20 * 128 // ((heads + kv) * dim)))
        return dict(kind=kind, tokens=tokens, heads=heads, kv_heads=kv, dim=dim,
                    rotary=dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2), interleaved=rng.random() < 0.5,
                    norm=rng.random() < 0.6, factor=rng.choice([1.0, 1.0, 2.0, 8.0]), train=rng.random() < 0.6)
    if kind == "attention":
        heads, kv = _heads(rng, 32)
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128]) if rng.random() < 0.7 else _log(rng, 16, 128)
        window = 0 if rng.random() < 0.4 else _log(rng, 16, 4096)
        sinks = 0 if rng.random() < 0.5 else _log(rng, 1, 64)
        train = rng.random() < 0.7
        lengths = [_log(rng, 1, 8192) for _ in range(_log(rng, 1, 12))]
        while len(lengths) > 1 and heads * dim * sum(n * n for n in lengths) > 8 * 128 * 4096 * 4096:
            lengths.remove(max(lengths))
        lengths[0] = min(lengths[0], int(math.sqrt(8 * 128 * 4096.0 * 4096.0 / (heads * dim))))
        return dict(kind=kind, lengths=" ".join(map(str, lengths)), heads=heads, kv_heads=kv, dim=dim, window=window,
                    sinks=sinks, train=train)
    heads, kv = _heads(rng, 32)
    c = dict(kind=kind, sequences=_log(rng, 1, 64), new=1 if rng.random() < 0.4 else _log(rng, 1, 1024),
             context=_log(rng, 1, 16384), heads=heads, kv_heads=kv, dim=16 * rng.choice([1, 2, 4, 4, 5, 6, 8, 8]),
             page=rng.choice([16, 32, 64, 64, 128]), type=rng.choice(["i8", "i8", "f32"]), spread=rng.choice([0.0, 0.5, 0.9]))
    c["context"] = max(c["context"], c["new"])
    # No more keys and values than the largest listed case has, and no more scores.
    most = 64 * 8192 * 8 * 64 // (4 if c["type"] == "f32" else 1)
    while c["sequences"] > 1 and c["sequences"] * c["context"] * kv * c["dim"] > most:
        c["sequences"] //= 2
    if kind == "paged":
        c["window"] = 0 if rng.random() < 0.6 else _log(rng, 16, 4096)
        c["sinks"] = 0 if rng.random() < 0.6 else _log(rng, 1, 64)
        while c["new"] > 1 and c["sequences"] * c["new"] * c["context"] * heads * c["dim"] > 4 * 512 * 12288 * 16 * 64:
            c["new"] = max(1, c["new"] // 2)
    else:
        while c["new"] > 1 and c["sequences"] * c["new"] * kv * c["dim"] > 4096 * 8 * 128:
            c["new"] = max(1, c["new"] // 2)
    return c


# ------------------------------------------------------------------ inputs
def _frequencies(c):
    """Angles a position: BASE^(-2 i / rotary), a longer context's positions squeezed by ``factor``."""
    return [BASE ** (-2.0 * i / c["rotary"]) / c["factor"] for i in range(c["rotary"] // 2)]


def _contexts(case, seed):
    """Length of every sequence of a cached batch, its new tokens included."""
    rng = random.Random(seed * 1000003 + 17)
    low = max(case["new"], int(case["context"] * (1 - case["spread"])))
    return [case["context"]] + [rng.randint(low, case["context"]) for _ in range(case["sequences"] - 1)]


def _quantise(x):
    """Signed bytes and their scale, one to a token and head: the largest magnitude is 127 steps.
    The quotient is rounded from float64: next to a half step float32 could go the other way."""
    scale = (x.abs().amax(-1, keepdim=True).double() / 127).float()
    q = torch.where(scale > 0, torch.round(x.double() / scale.double()), 0.0).clamp(-127, 127)
    return q, scale


def _slots(table, page, position):
    """Page and place in it of positions [B, n] of the sequences of a block table."""
    return torch.gather(table.long(), 1, position // page), position % page


def _inputs(case, seed):
    """Tensors of one case by name, made on the GPU from the seed alone."""
    g, c = torch.Generator(device="cuda").manual_seed(seed), case

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=g) * scale + mean

    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "rotary":
        t = c["tokens"]
        # A position anywhere in a long context for a decoded token, sequences from their start for others.
        start = torch.randint(0, 100000, (1,), device="cuda", generator=g)
        pos = start + torch.arange(t, device="cuda") if t < 64 else torch.arange(t, device="cuda") % 2048
        out = dict(q=normal(t, h * d).view(t, h, d), k=normal(t, kv * d).view(t, kv, d), positions=pos)
        if c["norm"]:
            out.update(qw=normal(d, scale=0.2, mean=1.0), kw=normal(d, scale=0.2, mean=1.0))
        if c["train"]:
            out.update(dq=normal(t, h, d, scale=0.05), dk=normal(t, kv, d, scale=0.05))
        return out
    if c["kind"] == "attention":
        lengths = list(map(int, c["lengths"].split()))
        t = sum(lengths)
        both = normal(t, 2 * kv * d)  # one projection gives keys and values
        starts = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        out = dict(q=normal(t, h, d), k=both[:, :kv * d].view(t, kv, d), v=both[:, kv * d:].view(t, kv, d), starts=starts)
        if c["train"]:
            out["do"] = normal(t, h, d, scale=0.05)
        return out
    b, n, page = c["sequences"], c["new"], c["page"]
    contexts = _contexts(c, seed)
    width = (c["context"] + page - 1) // page
    pages = b * width + 3
    table = torch.randperm(pages, device="cuda", generator=g)[:b * width].view(b, width).to(torch.int32)
    lengths = torch.tensor(contexts, device="cuda", dtype=torch.int32)
    kd, vd = (pages, kv, page, d), (pages, kv, d, page)
    out = dict(table=table, lengths=lengths)
    if c["kind"] == "cache":
        # What the cache held before: other sequences' tokens.
        if c["type"] == "i8":
            out.update(kc=torch.randint(-127, 128, kd, device="cuda", dtype=torch.int8, generator=g),
                       vc=torch.randint(-127, 128, vd, device="cuda", dtype=torch.int8, generator=g),
                       ks=normal(pages, kv, page, scale=0.01).abs(), vs=normal(pages, kv, page, scale=0.01).abs())
        else:
            out.update(kc=normal(*kd), vc=normal(*vd))
        level = normal(b * n, kv, 1).abs() + 0.2
        out.update(k=normal(b * n, kv, d) * level, v=normal(b * n, kv, d) * level)
        return out
    level = normal(pages, kv, page, 1).abs() * 0.3 + 0.8
    k, v = normal(*kd) * level, normal(pages, kv, page, d) * level
    if c["type"] == "i8":
        (kq, ks), (vq, vs) = _quantise(k), _quantise(v)
        out.update(kc=kq.to(torch.int8), vc=vq.transpose(2, 3).contiguous().to(torch.int8), ks=ks[..., 0].contiguous(),
                   vs=vs[..., 0].contiguous())
    else:
        out.update(kc=k, vc=v.transpose(2, 3).contiguous())
    out["q"] = normal(b * n, h, d)
    return out


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# --------------------------------------------------------------- operators
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state, state["case"])
    with torch.no_grad():
        return _PLAIN[kind](state, state["case"])


def _angles(t, c, like):
    """cos and sin [tokens, 1, rotary / 2]; the angle itself in float64, which far positions need."""
    f = torch.tensor(_frequencies(c), dtype=torch.float64, device=like.device)
    a = t["positions"].double()[:, None, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def _halves(x, c):
    r = c["rotary"]
    return (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])


def _turn(x, cos, sin, c):
    a, b = _halves(x, c)
    y = x.clone()
    ya, yb = _halves(y, c)
    ya.copy_(a * cos - b * sin)
    yb.copy_(b * cos + a * sin)
    return y


def _plain_rotary(t, c):
    cos, sin = _angles(t, c, t["q"])
    outs, grads = [], []
    for x, w, dy in ((t["q"], t.get("qw"), t.get("dq")), (t["k"], t.get("kw"), t.get("dk"))):
        xh = x
        if c["norm"]:
            rstd = (x * x).mean(-1, keepdim=True).add(EPS).rsqrt()
            xh = x * rstd
        outs.append(_turn(xh * w if c["norm"] else xh, cos, sin, c))
        if c["train"]:
            g = _turn(dy, cos, -sin, c)
            if c["norm"]:
                gw = g * w
                grads += [rstd * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (g * xh).sum((0, 1))]
            else:
                grads.append(g)
    return outs + grads


def _visible(rows, keys, window, sinks):
    """Which keys (positions) the rows (positions) see."""
    back = rows[..., :, None] - keys[..., None, :]
    near = back >= 0
    return near & ((back < window) | (keys < sinks)[..., None, :]) if window else near


def _plain_attention(t, c):
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    group, scale = h // kv, 1 / math.sqrt(d)
    out = torch.empty_like(t["q"])
    grads = [torch.empty_like(t["q"]), torch.empty_like(t["k"]), torch.empty_like(t["v"])] if c["train"] else []
    at = 0
    for n in map(int, c["lengths"].split()):
        rows = slice(at, at + n)
        at += n
        pos = torch.arange(n, device=out.device)
        hidden = ~_visible(pos, pos, c["window"], c["sinks"])
        # As many key heads at once as keep a score matrix within 4 GiB.
        step = max(1, min(kv, (1 << 30) // (group * n * n)))
        for k0 in range(0, kv, step):
            k1 = min(kv, k0 + step)
            heads = slice(k0 * group, k1 * group)
            q = t["q"][rows, heads].transpose(0, 1)
            k, v = (t[x][rows, k0:k1].transpose(0, 1).repeat_interleave(group, 0) for x in "kv")
            s = torch.matmul(q, k.transpose(1, 2)).mul_(scale).masked_fill_(hidden, -math.inf)
            p = s.sub_(s.amax(-1, keepdim=True)).exp_()
            p = p.div_(p.sum(-1, keepdim=True))
            o = torch.matmul(p, v)
            out[rows, heads] = o.transpose(0, 1)
            if c["train"]:
                do = t["do"][rows, heads].transpose(0, 1)
                dp = torch.matmul(do, v.transpose(1, 2))
                ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                shared = lambda x: x.view(k1 - k0, group, n, d).sum(1).transpose(0, 1)
                grads[0][rows, heads] = torch.matmul(ds, k).transpose(0, 1)
                grads[1][rows, k0:k1] = shared(torch.matmul(ds.transpose(1, 2), q))
                grads[2][rows, k0:k1] = shared(torch.matmul(p.transpose(1, 2), do))
    return [out] + grads


def _new_positions(t, c):
    return t["lengths"].long()[:, None] - c["new"] + torch.arange(c["new"], device=t["lengths"].device)


def _plain_cache(t, c):
    b, n, kv, d = c["sequences"], c["new"], c["kv_heads"], c["dim"]
    page, place = _slots(t["table"], c["page"], _new_positions(t, c))
    k, v = t["k"].view(b, n, kv, d), t["v"].view(b, n, kv, d)
    if c["type"] == "i8":
        (k, ks), (v, vs) = _quantise(k), _quantise(v)
        t["ks"][page, :, place], t["vs"][page, :, place] = ks[..., 0], vs[..., 0]
    t["kc"][page, :, place] = k.to(t["kc"].dtype)
    t["vc"][page, :, :, place] = v.to(t["vc"].dtype)
    # Read back: the values that the cache stands for.
    k, v = t["kc"][page, :, place].float(), t["vc"][page, :, :, place].float()
    if c["type"] == "i8":
        k, v = k * t["ks"][page, :, place][..., None], v * t["vs"][page, :, place][..., None]
    return [k.view(b * n, kv, d), v.view(b * n, kv, d)]


def _plain_paged(t, c):
    b, n, h, kv, d = c["sequences"], c["new"], c["heads"], c["kv_heads"], c["dim"]
    group, length = h // kv, t["table"].shape[1] * c["page"]
    pages = t["table"].long()
    k = t["kc"][pages].float()                      # [b, pages, kv, page, d]
    v = t["vc"][pages].float()                      # [b, pages, kv, d, page]
    if c["type"] == "i8":
        k.mul_(t["ks"][pages][..., None])
        v.mul_(t["vs"][pages][..., None, :])
    k = k.transpose(1, 2).reshape(b, kv, length, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, kv, length, d)
    q = t["q"].view(b, n, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, kv, group * n, d)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(d)).view(b, kv, group, n, length)
    seen = _visible(_new_positions(t, c), torch.arange(length, device=q.device).expand(b, length), c["window"], c["sinks"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(b, kv, group * n, length)
    o = torch.matmul(p, v).view(b, kv, group, n, d)
    return [o.permute(0, 3, 1, 2, 4).reshape(b * n, h, d)]


_PLAIN = dict(rotary=_plain_rotary, attention=_plain_attention, cache=_plain_cache, paged=_plain_paged)


def _mx():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from torch_vulkan import mx
    return mx


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _kept(t, name, make):
    """What a program keeps from call to call beside its tensors: made on a state's first pass."""
    if name not in t:
        t[name] = make()
    return t[name]


def _cache(t, c):
    mx = _mx()
    return (_kept(t, "cache", lambda: mx.KVCache(t["kc"], t["vc"], t.get("ks"), t.get("vs"))),
            _kept(t, "batch", lambda: mx.KVBatch(t["table"], t["lengths"], c["sequences"] * c["new"])))


def _own_rotary(t, c):
    mx, q, k = _mx(), t["q"], t["k"]
    plan = _kept(t, "plan", lambda: mx.Rotary(_frequencies(c), interleaved=c["interleaved"]))
    norm = dict(q_weight=t["qw"], k_weight=t["kw"], eps=EPS) if c["norm"] else {}
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    mx.qk_norm_rotary_forward(q, k, t["positions"], plan, q_out, k_out, stream=_stream(), **norm)
    if not c["train"]:
        return [q_out, k_out]
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    if not c["norm"]:
        mx.qk_norm_rotary_backward(t["dq"], t["dk"], None, None, t["positions"], plan, dq, dk, stream=_stream())
        return [q_out, k_out, dq, dk]
    dqw, dkw = torch.empty_like(t["qw"]), torch.empty_like(t["kw"])
    mx.qk_norm_rotary_backward(t["dq"], t["dk"], q, k, t["positions"], plan, dq, dk, dqw, dkw, stream=_stream(), **norm)
    return [q_out, k_out, dq, dqw, dk, dkw]


def _own_attention(t, c):
    mx, q, k, v = _mx(), t["q"], t["k"], t["v"]
    form = dict(starts=t["starts"], window=c["window"], sinks=c["sinks"], stream=_stream())
    out = torch.empty_like(q)
    if not c["train"]:
        mx.attention_forward(q, k, v, out, **form)
        return [out]
    lse = q.new_empty(c["heads"], q.shape[0])
    dq, dk, dv = torch.empty_like(q), k.new_empty(k.shape), v.new_empty(v.shape)
    mx.attention_forward(q, k, v, out, lse=lse, **form)
    mx.attention_backward(t["do"], q, k, v, out, lse, dq, dk, dv, **form)
    return [out, dq, dk, dv]


def _own_cache(t, c):
    mx, s = _mx(), _stream()
    k, v = torch.empty_like(t["k"]), torch.empty_like(t["v"])
    cache, batch = _cache(t, c)
    mx.kv_cache_write(cache, batch, t["k"], t["v"], stream=s)
    mx.kv_cache_read(cache, batch, k, v, stream=s)
    return [k, v]


def _own_paged(t, c):
    out = torch.empty_like(t["q"])
    cache, batch = _cache(t, c)
    _mx().attention_paged(cache, batch, t["q"], out, window=c["window"], sinks=c["sinks"], stream=_stream())
    return [out]


_OWN = dict(rotary=_own_rotary, attention=_own_attention, cache=_own_cache, paged=_own_paged)


# ------------------------------------------------------------ in 64 bits
def exact(case, seed):
    t, c = _inputs(case, seed), case
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    double = lambda x: x.double()

    def softmax_rows(q, k, v, rows, keys):
        """Attention of one query head over one key head."""
        s = (q @ k.T) / d ** 0.5
        i, j = rows.view(-1, 1), keys.view(1, -1)
        seen = (j <= i) & ((i - j < c["window"]) | (j < c["sinks"]) if c["window"] else (j <= i))
        return torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), 1) @ v

    if c["kind"] == "rotary":
        # The rotation as a product of complex numbers.
        angle = torch.outer(double(t["positions"]), torch.tensor(_frequencies(c), dtype=torch.float64, device="cuda"))
        unit = torch.polar(torch.ones_like(angle), angle)[:, None]
        r = c["rotary"]

        def forward(x, w):
            if c["norm"]:
                x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
            head, tail = x[..., :r], x[..., r:]
            pairs = head.unflatten(-1, (r // 2, 2)) if c["interleaved"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
            turned = turned.flatten(-2) if c["interleaved"] else turned.transpose(-1, -2).flatten(-2)
            return torch.cat([turned, tail], -1)

        outs, grads = [], []
        for x, w, dy in ((t["q"], t.get("qw"), t.get("dq")), (t["k"], t.get("kw"), t.get("dk"))):
            leaves = [double(x).requires_grad_()] + ([double(w).requires_grad_()] if c["norm"] else [])
            y = forward(leaves[0], leaves[-1])
            outs.append(y.detach())
            if c["train"]:
                grads += torch.autograd.grad(y, leaves, double(dy))
        return outs + grads
    if c["kind"] == "attention":
        outs = [torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")]
        if c["train"]:
            outs += [torch.zeros(t[x].shape, dtype=torch.float64, device="cuda") for x in "qkv"]
        at = 0
        for n in map(int, c["lengths"].split()):
            pos = torch.arange(n, device="cuda")
            for i in range(h):
                rows, key = slice(at, at + n), i // (h // kv)
                leaves = [double(t[x][rows, y]).requires_grad_(c["train"]) for x, y in (("q", i), ("k", key), ("v", key))]
                if c["train"]:
                    o = softmax_rows(*leaves, pos, pos)
                    for out, g, y in zip(outs[1:], torch.autograd.grad(o, leaves, double(t["do"][rows, i])), (i, key, key)):
                        out[rows, y] += g
                else:
                    o = torch.cat([softmax_rows(leaves[0][a:a + 4096], leaves[1], leaves[2], pos[a:a + 4096], pos)
                                   for a in range(0, n, 4096)])
                outs[0][rows, i] = o.detach()
            at += n
        return outs
    if c["kind"] == "cache":
        # The largest magnitude is 127 steps of a scale that is kept in float32.
        def held(x):
            if c["type"] == "f32":
                return double(x)
            step = (double(x).abs().max(-1, keepdim=True).values / 127).float().double()
            return torch.round(double(x) / step) * step
        return [held(t["k"]), held(t["v"])]
    n, out = c["new"], torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(t["lengths"].tolist()):
        pages = t["table"][b].long()
        keys, values = double(t["kc"][pages]), double(t["vc"][pages]).transpose(2, 3)
        if c["type"] == "i8":
            keys, values = keys * double(t["ks"][pages])[..., None], values * double(t["vs"][pages])[..., None]
        pos = torch.arange(length - n, length, device="cuda")
        for j in range(kv):
            k, v = keys[:, j].reshape(-1, d)[:length], values[:, j].reshape(-1, d)[:length]
            for i in range(j * (h // kv), (j + 1) * (h // kv)):
                out[b * n:(b + 1) * n, i] = softmax_rows(double(t["q"][b * n:(b + 1) * n, i]), k, v, pos,
                                                         torch.arange(length, device="cuda"))
    return [out]


# ------------------------------------------------- bytes and operations
def _pairs(first, n, window, sinks):
    """Query-key pairs of rows at positions first .. first + n - 1, and the keys that any of them sees."""
    if not window:
        return n * first + n * (n + 1) // 2, first + n
    def upto(m):  # keys seen by rows 0 .. m - 1: the window's, and the first ones behind it
        w = min(m, window)
        near = w * (w + 1) // 2 + (m - w) * window
        behind = max(0, m - window)  # row i >= window sees min(sinks, i - window + 1) more
        s = min(behind, sinks)
        return near + s * (s + 1) // 2 + (behind - s) * sinks
    low = max(0, first - window + 1)
    return upto(first + n) - upto(first), first + n - low + min(sinks, low)


def work(case):
    c, h, kv, d = case, case["heads"], case["kv_heads"], case["dim"]
    if c["kind"] == "rotary":
        e = float(c["tokens"] * (h + kv) * d)
        back = (3 if c["norm"] else 2) if c["train"] else 0  # dy, the norm's input again, dx
        return dict(bytes=4 * e * (2 + back) + 8 * c["tokens"], flops=e * (8.0 if c["norm"] else 4.0) * (3 if c["train"] else 1))
    if c["kind"] == "attention":
        lengths = list(map(int, c["lengths"].split()))
        t, pairs = sum(lengths), sum(_pairs(0, n, c["window"], c["sinks"])[0] for n in lengths)
        q, k = t * h * d, t * kv * d
        # Forward: q, k, v, out; backward: the output's gradient, and three gradients out.
        return dict(bytes=4.0 * (2 * q + 2 * k + (2 * q + 2 * k if c["train"] else 0)),
                    flops=2.0 * pairs * h * d * (7 if c["train"] else 2))
    size = d + 4 if c["type"] == "i8" else 4 * d
    contexts = _contexts(c, 0)
    if c["kind"] == "cache":
        e = c["sequences"] * c["new"] * kv
        return dict(bytes=2.0 * e * (4 * d + 2 * size + 4 * d), flops=4.0 * e * d)
    pairs, keys = map(sum, zip(*(_pairs(n - c["new"], c["new"], c["window"], c["sinks"]) for n in contexts)))
    return dict(bytes=2.0 * keys * kv * size + 8.0 * c["sequences"] * c["new"] * h * d, flops=4.0 * pairs * h * d)
