"""The cache in 4 bits: what is refused on the host, before anything is launched (the addresses are made up), and the tensors of a cache."""
import ctypes

import pytest
import torch

from autogptq.tvm_b200 import _lib, ops

A = 0x100000
CACHE = dict(k=A, v=A, k_scales=A, v_scales=A, dtype=0, batch=2, kv_heads=2, max_seq=40, hd=64, group=32)


def cache4(**change):
    c = _lib.Cache4(**{k: v for k, v in {**CACHE, **change}.items() if "stride" not in k})
    for n in ("k_stride", "v_stride"):
        setattr(c, n, (ctypes.c_int64 * 3)(*change.get(n, (2560, 1280, 32))))
    for n in ("k_scale_stride", "v_scale_stride"):
        setattr(c, n, (ctypes.c_int64 * 3)(*change.get(n, (320, 160, 4))))
    return c


BAD_CACHES = [(dict(dtype=2), -3), (dict(dtype=-1), -3), (dict(batch=0), -3), (dict(kv_heads=0), -3), (dict(max_seq=0), -3), (dict(hd=96), -3), (dict(group=128), -3),
              (dict(group=16), -3), (dict(batch=(1 << 29) + 1), -8), (dict(max_seq=(1 << 29) + 1), -8), (dict(k=None), -1), (dict(v_scales=None), -1),
              (dict(k=A + 8), -4), (dict(v=A + 4), -4), (dict(k_scales=A + 4), -4), (dict(k_stride=(2560, 1280, 40)), -4), (dict(v_scale_stride=(320, 160, 2)), -4),
              (dict(group=64, hd=128, k_scale_stride=(320, 160, 2)), -4)]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_caches_are_refused(change, status):
    w = _lib.CacheWriteArgs(cache=cache4(**change), k=A, v=A, pos=A, tokens=1)
    r = _lib.CacheReadArgs(cache=cache4(**change), k_out=A, v_out=A)
    assert _lib.lib.b200gptq_cache_write(ctypes.byref(w), None) == status
    assert _lib.lib.b200gptq_cache_read(ctypes.byref(r), None) == status


def test_arguments_are_refused():
    good = dict(k=A, v=A, pos=A, tokens=1)
    for change, status in [(dict(k=None), -1), (dict(v=None), -1), (dict(pos=None), -1), (dict(q=A, heads=2), -1), (dict(q_out=A), -1), (dict(cos_t=A, angles=4), -1),
                           (dict(q=A, q_out=A, heads=2), -1), (dict(tokens=0), -3), (dict(q=A, q_out=A, cos_t=A, sin_t=A, angles=4), -3), (dict(cos_t=A, sin_t=A), -3),
                           (dict(tokens=(1 << 29) + 1), -8), (dict(tokens=1 << 28), -8), (dict(k=A + 8), -4), (dict(pos=A + 4), -4), (dict(counts=A + 4), -4),
                           (dict(k_out=A + 2), -4), (dict(cos_t=A + 8, sin_t=A, angles=4), -4)]:
        a = _lib.CacheWriteArgs(cache=cache4(), **{**good, **change})
        assert _lib.lib.b200gptq_cache_write(ctypes.byref(a), None) == status, change
    a = _lib.CacheWriteArgs(cache=cache4(), **good)
    a.v_stride = (ctypes.c_int64 * 3)(64, 64, 4)
    assert _lib.lib.b200gptq_cache_write(ctypes.byref(a), None) == -4
    for change, status in [(dict(k_out=None), -1), (dict(v_out=None), -1), (dict(k_out=A + 8), -4), (dict(lengths=A + 4), -4)]:
        a = _lib.CacheReadArgs(cache=cache4(), **{**dict(k_out=A, v_out=A), **change})
        assert _lib.lib.b200gptq_cache_read(ctypes.byref(a), None) == status, change
    assert _lib.lib.b200gptq_cache_write(None, None) == -1 and _lib.lib.b200gptq_cache_read(None, None) == -1


def test_a_cache_and_its_size():
    c = ops.QuantCache.empty(2, 3, 5, 128, 64, torch.bfloat16, "cpu")
    assert c.k.shape == c.v.shape == (2, 3, 5, 64) and c.k_scales.shape == c.v_scales.shape == (2, 3, 5, 2, 2) and c.k_scales.dtype == torch.bfloat16
    assert c.nbytes == 2 * 30 * (64 + 8) and not c.k.any()
    for bad in (dict(hd=80), dict(hd=64, group=16)):
        with pytest.raises(ValueError):
            ops.QuantCache.empty(1, 1, 1, **bad)
    with pytest.raises(TypeError):
        ops.QuantCache.empty(1, 1, 1, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(RuntimeError):                       # there is no CPU path
        ops.cache_read(c)
    with pytest.raises(RuntimeError):
        ops.cache_write(c, torch.zeros(2, 1, 3, 128, dtype=torch.bfloat16), torch.zeros(2, 1, 3, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.long))


def test_attention_refuses():
    good = dict(q=A, out=A, pos=A, tokens=1, heads=4, window=8, scale=1.0)

    def arguments_of(change, cache=None):
        a = _lib.AttnCacheArgs(cache=cache4(**(cache or {})), **{**good, **{k: v for k, v in change.items() if "stride" not in k}})
        for n in ("q_stride", "out_stride"):
            setattr(a, n, (ctypes.c_int64 * 3)(*change.get(n, (256, 256, 64))))
        return ctypes.byref(a)

    def call(change, cache=None):              # (never with what is not refused: the addresses are made up, and there may be a GPU)
        return _lib.lib.b200gptq_attn_cache(arguments_of(change, cache), None, 0, None)

    def scratch(change):
        return _lib.lib.b200gptq_attn_cache_workspace_bytes(arguments_of(change))

    for change, status in [(dict(q=None), -1), (dict(out=None), -1), (dict(pos=None), -1), (dict(tokens=0), -3), (dict(heads=3), -3), (dict(heads=0), -3), (dict(window=-1), -3),
                           (dict(sinks=-1), -3), (dict(window=0, sinks=2), -3), (dict(tokens=1 << 29), -8), (dict(window=(1 << 29) + 1), -8), (dict(q=A + 8), -4), (dict(out=A + 2), -4),
                           (dict(pos=A + 4), -4), (dict(counts=A + 4), -4), (dict(status=A + 2), -4), (dict(q_stride=(256, 256, 4)), -4), (dict(out_stride=(4, 256, 64)), -4),
                           (dict(tokens=64), -5)]:
        assert call(change) == status, change
    for change, status in BAD_CACHES:
        assert call({}, change) == status, change
    assert scratch({}) == 0 and scratch(dict(tokens=64)) == 4 * 2 * 2 * 40 * 64 and scratch(dict(heads=3)) == -3
    assert _lib.lib.b200gptq_attn_cache(None, None, 0, None) == -1


def test_sampling_refuses():
    good = dict(logits=A, uniform=A, out=A, logits_stride=100, dtype=0, rows=2, vocab=100)
    for change, status in [(dict(logits=None), -1), (dict(uniform=None), -1), (dict(out=None), -1), (dict(dtype=3), -3), (dict(rows=0), -3), (dict(vocab=0), -3),
                           (dict(logits_stride=-1), -3), (dict(vocab=(1 << 18) + 1), -8), (dict(rows=(1 << 27) + 1), -8), (dict(logits=A + 1), -4), (dict(dtype=2, logits=A + 2), -4),
                           (dict(out=A + 4), -4), (dict(top_k=A + 4), -4), (dict(uniform=A + 2), -4), (dict(temperature=A + 2), -4), (dict(top_p=A + 1), -4), (dict(min_p=A + 2), -4)]:
        a = _lib.SampleArgs(**{**good, **change})
        assert _lib.lib.b200gptq_sample(ctypes.byref(a), None) == status, change
    assert _lib.lib.b200gptq_sample(None, None) == -1


def arguments(op):
    """(call, its tensors by name), of sizes that fit."""
    h = dict(dtype=torch.float16)
    if op == "sample":
        return ops.sample, dict(logits=torch.zeros(2, 40, **h), uniform=torch.zeros(2), temperature=torch.ones(2), top_k=torch.zeros(2).long(), top_p=torch.ones(2), min_p=torch.zeros(2),
                                out=torch.zeros(2).long())
    c = ops.QuantCache.empty(2, 2, 9, 64, 32, device="cpu")
    t = dict(k=c.k, v=c.v, k_scales=c.k_scales, v_scales=c.v_scales)
    rows = {n: torch.zeros(2, 1, 2, 64, **h) for n in ("k", "v", "q", "q_out", "k_out", "v_out")}
    parts = {f"cache.{n}": x for n, x in t.items()}

    def with_cache(call):
        return lambda **kw: call(cache=ops.QuantCache(*(kw.pop(f"cache.{n}") for n in t)), **kw)

    if op == "write":
        return with_cache(ops.cache_write), dict(parts, **rows, pos=torch.zeros(1).long(), cos=torch.ones(9, 32, **h), sin=torch.zeros(9, 32, **h))
    if op == "read":
        return with_cache(ops.cache_read), dict(parts, k_out=torch.zeros(2, 2, 9, 64, **h), v_out=torch.zeros(2, 2, 9, 64, **h))
    return with_cache(ops.attn_cache), dict(parts, q=torch.zeros(2, 1, 4, 64, **h), pos=torch.zeros(1).long(), out=torch.zeros(2, 1, 4, 64, **h))


FLOATS = [(op, n) for op in ("write", "read", "attend", "sample") for n, t in arguments(op)[1].items() if t.is_floating_point()]


@pytest.mark.parametrize("op,name", FLOATS)
def test_a_gradient_or_a_tangent_is_never_dropped(op, name):
    """There is no derivative: whichever tensor asks for one, the constants of a cache too, is refused (before the device is looked at)."""
    from torch.autograd import forward_ad
    call, t = arguments(op)
    plain = t[name]
    with forward_ad.dual_level():
        t[name] = forward_ad.make_dual(plain, torch.ones_like(plain))
        with torch.no_grad(), pytest.raises(RuntimeError, match="carries a tangent"):
            call(**t)
    t[name] = plain.requires_grad_()
    with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
        call(**t)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        call(**t)
