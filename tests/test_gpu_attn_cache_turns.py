"""Attention over a cache in 4 bits whose rows are read back: in turns where there is little scratch, and only the rows that a window leaves in sight, moved together.

Bounds are those of tests/test_gpu_attn_cache.py for calls that read back (values and weights rounded to the type); turns change nothing at all.
"""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import _lib, ops
    DEV = torch.device("cuda:0")

F16, BF16 = torch.float16, torch.bfloat16


def at(*pos):
    return torch.tensor(pos, device=DEV)


def inputs(B, T, heads, kv, hd, S, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(B, T, heads + 3, hd, generator=g, device=DEV).to(dtype)[:, :, 1:heads + 1]         # (heads apart from each other's sequences)
    cache = ops.QuantCache.empty(B, kv, S, hd, 32, dtype, DEV)
    for codes, constants in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device=DEV, dtype=torch.uint8))
        constants[..., 0] = (torch.rand(constants.shape[:-1], generator=g, device=DEV) * 0.3).to(dtype)
        constants[..., 1] = (torch.rand(constants.shape[:-1], generator=g, device=DEV) * -2).to(dtype)
    return q, cache


def arguments(q, cache, pos, out, window, sinks, counts):
    def three(t):
        return (ctypes.c_int64 * 3)(*t.stride()[:3])
    c = _lib.Cache4(k=cache.k.data_ptr(), v=cache.v.data_ptr(), k_scales=cache.k_scales.data_ptr(), v_scales=cache.v_scales.data_ptr(), k_stride=three(cache.k),
                    v_stride=three(cache.v), k_scale_stride=three(cache.k_scales), v_scale_stride=three(cache.v_scales), dtype=0 if q.dtype is F16 else 1, batch=q.shape[0],
                    kv_heads=cache.k.shape[1], max_seq=cache.k.shape[2], hd=q.shape[3], group=q.shape[3] // cache.k_scales.shape[3])
    return _lib.AttnCacheArgs(cache=c, q=q.data_ptr(), out=out.data_ptr(), pos=pos.data_ptr(), counts=counts.data_ptr() if counts is not None else None, q_stride=three(q),
                              out_stride=three(out), tokens=q.shape[1], heads=q.shape[2], window=window or 0, sinks=sinks, pos_each=int(pos.numel() > 1), scale=q.shape[3] ** -0.5)


def reference(q, cache, pos, window, sinks, counts=None):
    B, T, heads, hd = q.shape
    kv, S = cache.k.shape[1:3]
    G, u = heads // kv, torch.finfo(q.dtype).eps / 2
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    d = torch.arange(hd, device=DEV)
    word, field = d % 32 // 4 * (hd // 64) + d // 64, d % 2 * 4 + d % 4 // 2 + d % 64 // 32 * 2

    def values(packed, constants):
        wide = constants.double().repeat_interleave(32, -2)
        return (packed[..., word * 4 + field // 2].long() >> 4 * (field % 2) & 15).double() * wide[..., 0] + wide[..., 1]

    j = torch.arange(S, device=DEV)[None]
    for b in range(B):
        n = T if counts is None else max(0, min(T, counts[b]))
        p = (pos[b] + torch.arange(n, device=DEV))[:, None]
        seen = (j <= p) & ((j > p - window) | (j < sinks)) if window else j <= p
        rows = seen.any(0).nonzero()[:, 0]
        if not n or not rows.numel():
            continue
        seen = seen[:, rows]
        for h in range(kv):
            K, V = values(cache.k[b, h, rows], cache.k_scales[b, h, rows]), values(cache.v[b, h, rows], cache.v_scales[b, h, rows])
            for i in range(h * G, h * G + G):
                Q = q[b, :n, i].double()
                w = torch.softmax((Q @ K.t() * hd ** -0.5).masked_fill(~seen, -torch.inf), 1).nan_to_num()
                A = w @ V.abs()
                size = ((Q.abs() @ K.abs().t()) * seen).amax(1, keepdim=True) * hd ** -0.5
                e = (hd * 2.0 ** -22 + u) * size
                m = seen.sum(1, keepdim=True)
                out[b, :n, i] = w @ V
                bound[b, :n, i] = u * out[b, :n, i].abs() + (2 * u + 2 * e + m * 2.0 ** -22 + 2.0 ** -18) * A + (m * 2.0 ** -25 * V.abs().max() if q.dtype is F16 else 0)
    return out, bound


def check(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound.clamp(min=1e-30)).max()):.3g} times the bound"


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,T,heads,kv,hd,S,window,sinks", [
    (5, 70, 6, 3, 64, 333, 0, 0),
    (2, 40, 14, 7, 128, 200, 0, 0),
    (3, 64, 5, 5, 128, 1500, 200, 7),         # rows that move up
    (7, 33, 4, 2, 64, 900, 40, 0),
    (1, 300, 8, 4, 128, 4000, 500, 130)])
def test_turns(B, T, heads, kv, hd, S, window, sinks, dtype):
    """Scratch for all of it, for one key head of one sequence, and for numbers between that divide neither the batch nor the heads: the same bits."""
    q, cache = inputs(B, T, heads, kv, hd, S, dtype)
    pos = [(S - T) * (b + 1) // B - 3 * b for b in range(B)]
    counts = [T - 5 * b % T for b in range(B)]
    pos_d, counts_d = at(*pos), at(*counts)
    want = torch.full((B, heads, T, hd + 8), 9, dtype=dtype, device=DEV).transpose(1, 2)[..., :hd]
    ops.attn_cache(q, cache, pos_d, window=window or None, sinks=sinks, counts=counts_d, out=want)
    check(torch.cat([want[b, :counts[b]] for b in range(B)]), *(torch.cat([t[b, :counts[b]] for b in range(B)]) for t in reference(q, cache, pos, window, sinks, counts)))
    rows = 4 * hd * (min(S, window + sinks + T - 1) if window else S)
    stream = torch.cuda.current_stream(DEV).cuda_stream
    a = arguments(q, cache, pos_d, want, window, sinks, counts_d)
    need = _lib.lib.b200gptq_attn_cache_workspace_bytes(ctypes.byref(a))
    assert rows * B * kv <= need <= rows * B * kv + 8 * B + 8
    for pairs in sorted({1, 2, kv - 1 or 1, kv, B, B + 1, 2 * B + 1, B * kv - 1 or 1}):
        out = torch.full_like(want, 9)
        a = arguments(q, cache, pos_d, out, window, sinks, counts_d)
        scratch = torch.full((min(need, pairs * (rows + 8) + 16),), 255, dtype=torch.uint8, device=DEV)     # (NaNs where nothing is put)
        assert _lib.lib.b200gptq_attn_cache(ctypes.byref(a), scratch.data_ptr(), scratch.numel(), stream) == 0
        assert torch.equal(out, want), pairs
        guard = torch.full((need + 4096,), 77, dtype=torch.uint8, device=DEV)                              # (nothing behind the scratch)
        assert _lib.lib.b200gptq_attn_cache(ctypes.byref(a), guard.data_ptr(), scratch.numel(), stream) == 0
        assert bool((guard[scratch.numel():] == 77).all())
    assert _lib.lib.b200gptq_attn_cache(ctypes.byref(a), scratch.data_ptr(), rows - 1, stream) == -5
    ops.check_status(DEV)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T", [64, 129])
@pytest.mark.parametrize("S,window,sinks", [(1000, 50, 0), (1000, 50, 4), (1000, 1, 0), (1000, 1, 65), (1000, 300, 200), (1000, 871, 0), (1000, 872, 0), (700, 630, 7), (5000, 64, 64)])
def test_windows_over_longer_caches(S, window, sinks, T, dtype):
    """Sequences at the beginning, where sinks and window meet and a row before and behind, in the middle and past both ends of the cache."""
    meet = sinks + window - 1
    pos = [0, 3, meet - 1, meet, meet + 1, meet + 2, S // 2, S - T - 1, S - T, S - T + 1, S - 1, S, S + window - 2, S + window + 5, 1 << 40, -3, -T, -1000]
    B = len(pos)
    q, cache = inputs(B, T, 2, 2, 64, S, dtype)
    nan = float("nan")
    want, bound = reference(q, cache, [min(p, 1 << 30) for p in pos], window, sinks)
    for b, p in enumerate(pos):                # what no token sees
        for t in (cache.k_scales, cache.v_scales):
            t[b, :, min(S, max(0, p + T)):] = nan
            t[b, :, sinks:min(S, max(sinks, p - window + 1))] = nan
            if p < 0:
                t[b, :, max(0, p + T):] = nan
    check(ops.attn_cache(q, cache, at(*pos), window=window, sinks=sinks), want, bound)
    counts = [T if b % 3 else T // 2 for b in range(B)]
    out = torch.full_like(q, 9)
    ops.attn_cache(q, cache, at(*pos), window=window, sinks=sinks, counts=at(*counts), out=out)
    for b, n in enumerate(counts):
        check(out[b, :n], want[b, :n], bound[b, :n])
        assert bool((out[b, n:] == 9).all())
    one = ops.attn_cache(q, cache, at(S // 2), window=window, sinks=sinks)          # one position for all
    check(one[6], want[6], bound[6])
    ops.check_status(DEV)


def test_what_a_call_takes():
    """Sixteen texts in caches of 131072 rows, 64 tokens and a window of 256: some 21 MB beside the output, not a cache in 16 bits."""
    B, T, kv, S = 16, 64, 2, 131072
    q, cache = inputs(1, T, kv, kv, 128, S, F16)
    q = q.expand(B, -1, -1, -1)
    cache = ops.QuantCache(*(t.expand(B, -1, -1, -1, *([-1] if t.dim() == 5 else [])) for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)))
    pos = at(*range(1000, 1000 + 7000 * B, 7000))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.attn_cache(q, cache, pos, window=256)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= out.numel() * 2 + B * kv * 319 * 128 * 4 + (1 << 20)
    want, bound = reference(q, cache, pos.tolist(), 256, 0)
    check(out, want, bound)


def test_turns_of_long_texts():
    """More than 1 GB of rows: the call makes two turns of its own, and one where it is given more than it asks for."""
    B, T, kv, S = 2, 300, 8, 131072           # (so many tokens that reading back pays)
    q, cache = inputs(1, T, kv, kv, 128, S, F16)
    q = torch.cat([q, -q])
    cache = ops.QuantCache(*(t.expand(B, -1, -1, -1, *([-1] if t.dim() == 5 else [])) for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)))
    pos = at(130000, 517)
    out = ops.attn_cache(q, cache, pos)
    other = torch.empty_like(out)
    a = arguments(q, cache, pos, other, 0, 0, None)
    rows = 4 * 128 * S
    assert _lib.lib.b200gptq_attn_cache_workspace_bytes(ctypes.byref(a)) == B * kv // 2 * rows
    scratch = torch.empty(B * kv * (rows + 8), dtype=torch.uint8, device=DEV)
    assert _lib.lib.b200gptq_attn_cache(ctypes.byref(a), scratch.data_ptr(), scratch.numel(), torch.cuda.current_stream(DEV).cuda_stream) == 0
    assert torch.equal(out, other)
    want, bound = reference(q[1:], ops.QuantCache(*(t[1:] for t in (cache.k, cache.v, cache.k_scales, cache.v_scales))), [517], 0, 0)
    check(out[1:], want, bound)
    ops.check_status(DEV)
