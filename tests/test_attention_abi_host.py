"""Refusals and workspace sizes of the attention layer's calls (rotation, attention,
paged cache, attention over it): host validation, no GPU calls."""
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


def rotary(mx, freqs=(1.0, 0.1), **over):
    f = (C.c_double * max(1, len(freqs)))(*freqs)
    d = mx.RotaryDesc(3, 2, 1, 8, 2 * len(freqs), 16, 8, 8, 8, FAKE, C.cast(f, C.c_void_p), 1.0, 1e-6, 0, 1)
    d.keep = f
    for k, v in over.items():
        setattr(d, k, v)
    return d


ROTARY_BAD = [(dict(tokens=-1), "negative"), (dict(q_heads=-1), "negative"), (dict(head_dim=0), "head_dim"),
              (dict(head_dim=257), "head_dim"), (dict(rotary_dim=3), "even"), (dict(rotary_dim=10), "at most"),
              (dict(rotary_dim=-2), "rotary_dim"), (dict(tokens=1 << 31), "out of range"), (dict(frequencies=None), "null"),
              (dict(magnitude=float("nan")), "magnitude"), (dict(eps=-1.0), "eps"), (dict(eps=float("inf")), "eps")]


@pytest.mark.parametrize("over,message", ROTARY_BAD)
def test_rotary_refusals(mx, over, message):
    d = rotary(mx, **over)
    f = (C.byref(d), FAKE, FAKE, None, None, FAKE, FAKE, None)
    assert message in str(refused(mx, "mx_qk_norm_rotary_forward", *f))
    b = (C.byref(d), FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, FAKE, None, 0, None)
    assert message in str(refused(mx, "mx_qk_norm_rotary_backward", *b))


def test_rotary_buffers(mx):
    f = "mx_qk_norm_rotary_forward"
    for i in (0, 1, 4, 5):
        args = [FAKE, FAKE, None, None, FAKE, FAKE, None]
        args[i] = None
        assert "null buffer" in str(refused(mx, f, C.byref(rotary(mx)), *args))
    assert "null buffer" in str(refused(mx, f, C.byref(rotary(mx, positions=None)), FAKE, FAKE, None, None, FAKE, FAKE, None))
    assert "null descriptor" in str(refused(mx, f, None, FAKE, FAKE, None, None, FAKE, FAKE, None))
    assert "finite" in str(refused(mx, f, C.byref(rotary(mx, (float("inf"), 1.0))), FAKE, FAKE, None, None, FAKE, FAKE, None))
    b = "mx_qk_norm_rotary_backward"
    # the norm needs its input, and weights need a norm
    assert "null buffer" in str(refused(mx, b, C.byref(rotary(mx)), FAKE, FAKE, None, FAKE, None, None, FAKE, FAKE, None, None,
                                        None, 0, None))
    assert "without a norm" in str(refused(mx, b, C.byref(rotary(mx, norm=0)), FAKE, FAKE, None, None, None, None, FAKE, FAKE,
                                           FAKE, None, None, 0, None))
    big = rotary(mx, tokens=1 << 16)
    need = C.c_int64()
    mx.check(mx.lib().mx_qk_norm_rotary_workspace(C.byref(big), C.byref(need)))
    assert need.value > 0
    e = refused(mx, b, C.byref(big), FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, FAKE, FAKE, need.value - 1, None)
    assert e.status == mx.MX_ERR_WORKSPACE
    assert "null result" in str(refused(mx, "mx_qk_norm_rotary_workspace", C.byref(big), None))
    # no tokens, no heads, nothing asked for
    mx.check(mx.lib().mx_qk_norm_rotary_forward(C.byref(rotary(mx, tokens=0)), None, None, None, None, None, None, None))
    mx.check(mx.lib().mx_qk_norm_rotary_forward(C.byref(rotary(mx, q_heads=0, k_heads=0)), None, None, None, None, None, None, None))
    mx.check(mx.lib().mx_qk_norm_rotary_backward(C.byref(rotary(mx)), *[None] * 10, None, 0, None))


def attention(mx, **over):
    d = mx.AttentionDesc(10, 2, FAKE, 4, 2, 16, 64, 16, 32, 16, 32, 16, 0, 0, 0.25)
    for k, v in over.items():
        setattr(d, k, v)
    return d


ATTENTION_BAD = [(dict(tokens=-1), "negative size"), (dict(sequences=-1), "negative size"), (dict(heads=-4), "negative size"),
                 (dict(head_dim=0), "head_dim"), (dict(head_dim=129), "head_dim"), (dict(heads=3), "evenly"),
                 (dict(kv_heads=0), "evenly"), (dict(tokens=1 << 31), "out of range"), (dict(heads=65536), "out of range"),
                 (dict(sequences=1 << 22), "out of range"), (dict(tokens=1 << 27, heads=16), "out of range"), (dict(sequences=0), "no sequence"),
                 (dict(starts=None, sequences=3), "do not divide"), (dict(window=-1), "negative window"),
                 (dict(sinks=-1), "negative window"), (dict(scale=float("nan")), "scale")]


@pytest.mark.parametrize("over,message", ATTENTION_BAD)
def test_attention_refusals(mx, over, message):
    d = attention(mx, **over)
    assert message in str(refused(mx, "mx_attention_forward", C.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, None, 0, None))
    assert message in str(refused(mx, "mx_attention_backward", C.byref(d), *[FAKE] * 9, None, 0, None))
    assert message in str(refused(mx, "mx_attention_workspace", C.byref(d), 0, C.byref(C.c_int64())))


def test_attention_buffers_and_workspace(mx):
    for i in range(4):
        args = [FAKE] * 4
        args[i] = None
        assert "null buffer" in str(refused(mx, "mx_attention_forward", C.byref(attention(mx)), *args, None, None, 0, None))
    for i in range(6):
        args = [FAKE] * 9
        args[i] = None
        assert "null buffer" in str(refused(mx, "mx_attention_backward", C.byref(attention(mx)), *args, None, 0, None))
    for backward, call in ((0, "mx_attention_forward"), (1, "mx_attention_backward")):
        need = C.c_int64()
        mx.check(mx.lib().mx_attention_workspace(C.byref(attention(mx)), backward, C.byref(need)))
        assert need.value > 0
        bufs = [FAKE] * (9 if backward else 5)
        e = refused(mx, call, C.byref(attention(mx)), *bufs, FAKE, need.value - 1, None)
        assert e.status == mx.MX_ERR_WORKSPACE and str(need.value) in str(e)
        assert "aligned" in str(refused(mx, call, C.byref(attention(mx)), *bufs, FAKE + 4, need.value, None))
        assert mx.attention_workspace(0, 0, 4, 2, 16, bool(backward)) == 0
    mx.check(mx.lib().mx_attention_forward(C.byref(attention(mx, tokens=0)), *[None] * 6, 0, None))
    mx.check(mx.lib().mx_attention_forward(C.byref(attention(mx, heads=0, kv_heads=0)), *[None] * 6, 0, None))
    mx.check(mx.lib().mx_attention_backward(C.byref(attention(mx)), *[FAKE] * 6, None, None, None, None, 0, None))


def cache(mx, **over):
    c = mx.KVCacheDesc(FAKE, FAKE, FAKE, FAKE, 7, 2, 32, 16, mx.KV_I8)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def batch(mx, **over):
    b = mx.KVBatchDesc(6, 3, 4, FAKE, FAKE, FAKE)
    for k, v in over.items():
        setattr(b, k, v)
    return b


CACHE_BAD = [(dict(type=2), {}, "unknown cache type"), (dict(pages=-1), {}, "negative"), (dict(heads=-1), {}, "negative"),
             (dict(page_size=24), {}, "page_size"), (dict(page_size=0), {}, "page_size"), (dict(head_dim=20), {}, "head_dim"),
             (dict(head_dim=0), {}, "head_dim"), (dict(head_dim=144), {}, "head_dim"), (dict(pages=1 << 31), {}, "out of range"),
             ({}, dict(tokens=-1), "negative"), ({}, dict(table_width=-1), "negative"), ({}, dict(sequences=0), "no sequence"),
             ({}, dict(table_width=1 << 30), "out of range"), ({}, dict(starts=None, sequences=4), "do not divide"),
             ({}, dict(lengths=None), "null lengths"), ({}, dict(table=None), "null lengths or table"),
             (dict(k=None), {}, "null buffer of the cache"), (dict(v_scale=None), {}, "null buffer of the cache"),
             (dict(v=FAKE + 8), {}, "aligned"), (dict(k_scale=FAKE + 4), {}, "aligned")]


@pytest.mark.parametrize("c,b,message", CACHE_BAD)
def test_cache_refusals(mx, c, b, message):
    c, b = cache(mx, **c), batch(mx, **b)
    assert message in str(refused(mx, "mx_kv_cache_write", C.byref(c), C.byref(b), FAKE, 32, 16, FAKE, 32, 16, None))
    assert message in str(refused(mx, "mx_kv_cache_read", C.byref(c), C.byref(b), FAKE, FAKE, None))
    d = mx.PagedDesc(4, 64, 16, 0, 0, 0.25)
    assert message in str(refused(mx, "mx_attention_paged", C.byref(d), C.byref(c), C.byref(b), FAKE, FAKE, None, 0, None))


def test_paged_refusals(mx):
    f = "mx_attention_paged"
    call = lambda d, c=cache(mx), b=batch(mx), q=FAKE, out=FAKE: str(refused(
        mx, f, C.byref(d) if d else None, C.byref(c) if c else None, C.byref(b), q, out, None, 0, None))
    ok = mx.PagedDesc(4, 64, 16, 0, 0, 0.25)
    assert "null descriptor" in call(None) and "null cache" in call(ok, None)
    assert "evenly" in call(mx.PagedDesc(3, 64, 16, 0, 0, 0.25)) and "negative" in call(mx.PagedDesc(-2, 64, 16, 0, 0, 0.25))
    assert "window" in call(mx.PagedDesc(4, 64, 16, -1, 0, 0.25)) and "sinks" in call(mx.PagedDesc(4, 64, 16, 0, -1, 0.25))
    assert "scale" in call(mx.PagedDesc(4, 64, 16, 0, 0, float("inf")))
    assert "out of range" in call(ok, b=batch(mx, tokens=1 << 29))
    assert "null buffer" in call(ok, q=None) and "null buffer" in call(ok, out=None)
    long = batch(mx, tokens=1, sequences=1, table_width=1 << 12)
    need = C.c_int64()
    mx.check(mx.lib().mx_attention_paged_workspace(C.byref(ok), C.byref(cache(mx)), C.byref(long), C.byref(need)))
    assert need.value > 0, "one token over a long context is shared out"
    e = refused(mx, f, C.byref(ok), C.byref(cache(mx)), C.byref(long), FAKE, FAKE, FAKE, need.value - 1, None)
    assert e.status == mx.MX_ERR_WORKSPACE
    # nothing to do
    none = batch(mx, tokens=0, sequences=0, starts=None)
    mx.check(mx.lib().mx_attention_paged(C.byref(ok), C.byref(cache(mx)), C.byref(none), None, None, None, 0, None))
    mx.check(mx.lib().mx_kv_cache_write(C.byref(cache(mx)), C.byref(none), None, 0, 0, None, 0, 0, None))
    mx.check(mx.lib().mx_kv_cache_read(C.byref(cache(mx)), C.byref(none), None, None, None))


def test_python_binding_checks_shapes(mx):
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)
    plan = mx.Rotary([1.0, 0.5])
    pos = t(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="do not fit"):
        mx.qk_norm_rotary_forward(t(3, 2, 8), t(4, 2, 8), pos, plan, t(3, 2, 8), t(4, 2, 8))
    with pytest.raises(ValueError, match="positions"):
        mx.qk_norm_rotary_forward(t(3, 2, 8), None, pos.int(), plan, t(3, 2, 8), None)
    with pytest.raises(ValueError, match="positions"):
        mx.qk_norm_rotary_forward(t(3, 2, 8), None, None, plan, t(3, 2, 8), None)
    with pytest.raises(ValueError, match="q_out"):
        mx.qk_norm_rotary_forward(t(3, 2, 8), None, pos, plan, t(3, 2, 9), None)
    with pytest.raises(ValueError, match="last axis"):
        mx.qk_norm_rotary_forward(t(3, 8, 2).transpose(1, 2), None, pos, plan, t(3, 2, 8), None)
    with pytest.raises(ValueError, match="q_weight"):
        mx.qk_norm_rotary_forward(t(3, 2, 8), None, pos, plan, t(3, 2, 8), None, q_weight=t(7), eps=1e-6)
    with pytest.raises(ValueError, match="neither"):
        mx.qk_norm_rotary_forward(None, None, pos, plan, None, None)
    with pytest.raises(ValueError, match="without its output"):
        mx.qk_norm_rotary_backward(t(3, 2, 8), None, None, None, pos, plan, t(3, 2, 8), t(3, 1, 8))
    q, k = t(6, 4, 8), t(6, 2, 8)
    with pytest.raises(ValueError, match="do not fit"):
        mx.attention_forward(q, k, t(6, 1, 8), t(6, 4, 8))
    with pytest.raises(ValueError, match="starts"):
        mx.attention_forward(q, k, k, t(6, 4, 8), starts=t(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="float32"):
        mx.attention_forward(q.double(), k, k, t(6, 4, 8))
    with pytest.raises(ValueError, match="lse"):
        mx.attention_forward(q, k, k, t(6, 4, 8), lse=t(6, 4))
    with pytest.raises(ValueError, match="dv"):
        mx.attention_backward(q, q, k, k, q, t(4, 6), None, None, t(6, 4, 8))
    i8 = dict(dtype=torch.int8)
    with pytest.raises(ValueError, match="scales"):
        mx.KVCache(t(5, 2, 16, 32, **i8), t(5, 2, 32, 16, **i8))
    with pytest.raises(ValueError, match="KVCache: v"):
        mx.KVCache(t(5, 2, 16, 32), t(5, 2, 16, 32))
    with pytest.raises(ValueError, match="float32 or int8"):
        mx.KVCache(t(5, 2, 16, 32).half(), t(5, 2, 32, 16).half())
    c = mx.KVCache(t(5, 2, 16, 32), t(5, 2, 32, 16))
    with pytest.raises(ValueError, match="lengths"):
        mx.KVBatch(t(3, 2, dtype=torch.int32), t(2, dtype=torch.int32), 3)
    b = mx.KVBatch(t(3, 2, dtype=torch.int32), t(3, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="do not fit"):
        mx.kv_cache_write(c, b, t(3, 1, 32), t(3, 2, 32))
    with pytest.raises(ValueError, match="does not fit"):
        mx.attention_paged(c, b, t(4, 2, 32), t(4, 2, 32))


@pytest.mark.parametrize("kind", ["KV_F32", "KV_I8"])
@pytest.mark.parametrize("tokens", [1, 3, 700])
def test_paged_plans_of_the_largest_windows(mx, kind, tokens):
    """A window that reaches past the table is planned as none."""
    c, need = cache(mx, type=getattr(mx, kind)), C.c_int64()
    b = batch(mx, tokens=tokens, sequences=1, table_width=1 << 7)
    sizes = []
    for window in (0, 1 << 12, 1 << 40, 2 ** 63 - 200, 2 ** 63 - 1):
        for sinks in (0, 2 ** 63 - 1):
            d = mx.PagedDesc(4, 64, 16, window, sinks, 0.25)
            mx.check(mx.lib().mx_attention_paged_workspace(C.byref(d), C.byref(c), C.byref(b), C.byref(need)))
            sizes.append(need.value)
    assert sizes[0] > 0 and sizes == sizes[:1] * len(sizes)
