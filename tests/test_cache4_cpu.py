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
