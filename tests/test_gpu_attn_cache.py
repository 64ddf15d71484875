"""Attention over a cache in 4 bits (ops.attn_cache), against 64 bits.

The bound, per output element, with u = half a step of the type (2^-11 fp16, 2^-8 bf16), K and V the values zero + scale code that the cache stands for,
|K|+ = |zero| + scale code, |V|+ = |zero + 8 scale| + scale |code - 8| (each as the two that are added up apart), A = sum_j w_j |V_j|+ / sum_j w_j, s the largest scale of V
and n visible keys:

    u |o|                             the result's rounding
    + 2^-11 A                         each weight times scale is rounded to fp16 before it multiplies a code less 8 (relative)
    + n 2^-25 8 s                     and below 2^-14 of the largest scale to half a step of fp16's subnormal numbers; codes less 8 are 8 at most
    + 2 d A                           d: error of a score in fp32, hd products and sums, each off by 2^-22 of the sum of |q| |K|+ at most
                                      (2^-24 for rounded sums; the tensor cores may truncate), which moves a weight and the denominator
    + (n 2^-22 + 2^-18) A             sums of n products in fp32 likewise; exp2, scale, merging of parts: a few steps of 2^-22 each

Where rows are read back first (from 64 rows per key head on at these lengths, or from 17 over many keys), K, V and the weights are rounded to the type: u sum |q| |K| more for a score, and 2 u A (and in fp16 n 2^-25 max |V|
for weights below 2^-14).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")

F16, BF16 = torch.float16, torch.bfloat16


def parts(packed, constants):
    """(scale code, zero) of each dim in 64 bits, by the header's order of the codes."""
    hd = packed.shape[-1] * 2
    words = packed.to(torch.int64).reshape(*packed.shape[:-1], hd // 8, 4)
    words = words[..., 0] | words[..., 1] << 8 | words[..., 2] << 16 | words[..., 3] << 24
    codes = torch.zeros(*packed.shape[:-1], hd, dtype=torch.float64, device=packed.device)
    for w in range(hd // 8):
        for f, e in enumerate((0, 2, 32, 34, 1, 3, 33, 35)):
            codes[..., 64 * (w % (hd // 64)) + 4 * (w // (hd // 64)) + e] = (words[..., w] >> 4 * f & 15).double()
    group = hd // constants.shape[-2]
    wide = constants.double().repeat_interleave(group, -2)
    return codes * wide[..., 0], wide[..., 1]


def reference(q, cache, pos, window=None, sinks=0, scale=None, counts=None):
    """(output, bound) in 64 bits; pos: list of positions of token 0.  Rows that a query does not see are never looked at."""
    B, T, heads, hd = q.shape
    kv, S = cache.k.shape[1], cache.k.shape[2]
    G, u = heads // kv, torch.finfo(q.dtype).eps / 2
    scale = hd ** -0.5 if scale is None else scale
    many = T * G >= 64 or (T * G > 16 and B * kv * S > 50000)
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    j = torch.arange(S, device=DEV)
    for b in range(B):
        n_tokens = T if counts is None else max(0, min(T, counts[b]))
        for h in range(kv):
            (kc, kz), (vc, vz) = parts(cache.k[b, h], cache.k_scales[b, h]), parts(cache.v[b, h], cache.v_scales[b, h])
            for t in range(n_tokens):
                p = pos[b] + t
                seen = j <= p
                if window is not None:
                    seen &= (j > p - window) | (j < sinks)
                n = int(seen.sum())
                if n == 0:
                    continue
                K, V, Kp = kc[seen] + kz[seen], vc[seen] + vz[seen], kc[seen] + kz[seen].abs()
                eight = 8 * cache.v_scales[b, h][seen][..., 0].double().repeat_interleave(hd // cache.v_scales.shape[3], -1)
                Vp = (vz[seen] + eight).abs() + (vc[seen] - eight).abs()
                Q = q[b, t, h * G:h * G + G].double()
                w = torch.softmax(Q @ K.t() * scale, dim=1)
                o, A = w @ V, w @ Vp
                d = hd * 2.0 ** -22 * (Q.abs() @ Kp.t()).amax(1, keepdim=True) * abs(scale)
                top = cache.v_scales[b, h][seen][..., 0].double().amax()
                err = u * o.abs() + n * 2.0 ** -25 * 8 * top + 2.0 ** -11 * A
                if many:
                    d = d + u * (Q.abs() @ K.abs().t()).amax(1, keepdim=True) * abs(scale)
                    err = err + 2 * u * A + (n * 2.0 ** -25 * V.abs().max() if q.dtype is F16 else 0)
                out[b, t, h * G:h * G + G], bound[b, t, h * G:h * G + G] = o, err + (2 * d + n * 2.0 ** -22 + 2.0 ** -18) * A
    return out, bound


def inputs(B, T, heads, kv, hd, S, dtype, group=32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    q, k, v = (1.5 * r(B, T, heads, hd) + 0.5).to(dtype), r(B, S, kv, hd), r(B, S, kv, hd)
    k[:, :3] += 0.5                           # the first keys lie along the queries
    v *= torch.exp2(r(B, S, kv, 1) * 2)       # rows of unlike size: scales between 2^-9 and 2^5 or so
    cache = ops.QuantCache.empty(B, kv, S, hd, group, dtype, DEV)
    ops.cache_write(cache, k.to(dtype), v.to(dtype), at(0))
    return q, cache


def check(got, want, bound):
    """(The same infinity, of infinite scales, is off by nothing: its difference is a NaN.)"""
    off = (got.double() - want).abs()
    assert bool(((off <= bound) | (got.double() == want)).all()), f"off by up to {float((off / bound.clamp(min=1e-30)).max()):.3g} times the bound"


def at(*pos):
    return torch.tensor(pos, device=DEV)


CASES = [
    # B, T, heads, kv, hd, max_seq, positions, window, sinks
    (1, 1, 4, 4, 128, 64, [0], None, 0),              # the very first token
    (1, 1, 4, 4, 128, 1, [0], None, 0),               # a cache of one row
    (1, 1, 4, 4, 128, 64, [63], 1, 0),                # sees itself alone
    (1, 1, 4, 4, 64, 64, [63], 1, 4),
    (1, 1, 32, 32, 128, 768, [700], None, 0),
    (1, 1, 8, 8, 128, 2048, [2047], None, 0),         # a cluster per head
    (3, 1, 8, 8, 128, 333, [5, 332, 100], 40, 4),     # shorter than, longer than the window
    (2, 1, 14, 2, 64, 333, [17, 332], 33, 0),         # groups of seven heads
    (2, 1, 16, 1, 128, 100, [15, 99], None, 0),       # sixteen rows
    (1, 1, 40, 2, 128, 100, [99], 64, 16),            # twenty rows
    (2, 1, 40, 1, 64, 70, [69, 3], None, 0),          # forty: two tiles
    (2, 1, 4, 4, 128, 50, [49, 10], 1000, 4),         # the window holds everything
    (2, 1, 4, 4, 128, 50, [49, 10], 8, 45),           # nearly everything is a sink
    (40, 1, 8, 8, 64, 40, list(range(40)), 9, 3),
    (2, 2, 4, 4, 128, 100, [0, 98], 5, 2),            # short runs of tokens
    (2, 5, 12, 4, 64, 100, [3, 95], None, 0),
    (1, 3, 7, 7, 128, 65, [62], 16, 16),
    (2, 33, 4, 4, 128, 100, [50, 0], 20, 4),          # two tiles of rows
    (1, 63, 2, 2, 64, 70, [7], None, 0),
    (1, 1, 2, 2, 64, 5000, [4999], None, 0),          # more keys
    (1, 1, 2, 2, 64, 5000, [4999], 4500, 130),
    (3, 1, 8, 2, 128, 4097, [4096, 0, 2000], None, 0),
    (5, 3, 6, 2, 128, 2500, [0, 2497, 31, 1200, 16], None, 0),
    (2, 2, 32, 2, 64, 2100, [2098, 1000], None, 0),   # 32 rows
    (2, 7, 10, 2, 128, 2100, [2093, 17], None, 0),    # 35 rows: two tiles
    (300, 1, 1, 1, 64, 2100, [7 * b for b in range(300)], None, 0),
    (2, 70, 4, 2, 64, 75, [0, 5], 16, 4),             # prompts and chunks of them
    (1, 129, 2, 1, 128, 300, [171], None, 0),
    (2, 257, 2, 2, 64, 300, [0, 43], None, 0),
    (1, 8, 16, 2, 128, 600, [500], 129, 1),
    (1, 17, 8, 2, 128, 9000, [8983], None, 0),        # 68 rows over few heads and many keys: not read back
    (30, 12, 32, 8, 128, 400, list(range(0, 390, 13)), None, 0),      # 48 over many heads: read back
    (1, 1, 8, 2, 128, 40000, [39000], None, 0),       # CTAs that are one text's and key head's
    (7, 1, 8, 2, 128, 20000, [3, 19999, 0, 700, 12000, 40, 9], None, 0),
    (2, 1, 2, 2, 64, 17000, [16999, 100], 16500, 130),                # even runs, from here on: with sinks
    (150, 1, 1, 1, 64, 10000, [60 * b for b in range(150)], None, 0),
    (1, 1, 16, 1, 128, 17000, [16990], None, 0),      # 16 rows
    (2, 2, 32, 2, 64, 17000, [16998, 9000], None, 0),
    (2, 7, 10, 2, 128, 17000, [16993, 17], None, 0),  # 35 rows: two tiles
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("B,T,heads,kv,hd,S,pos,window,sinks", CASES)
def test_against_64_bits(B, T, heads, kv, hd, S, pos, window, sinks, group, dtype):
    q, cache = inputs(B, T, heads, kv, hd, S, dtype, group)
    out = ops.attn_cache(q, cache, at(*pos), window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    check(out, *reference(q, cache, pos, window, sinks))
    assert torch.equal(out, ops.attn_cache(q, cache, at(*pos), window=window, sinks=sinks))      # the same bits every time
    ops.check_status(DEV)


@pytest.mark.parametrize("S", [60, 2100, 17000])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_one_position_for_all_a_scale_and_an_output(T, S):
    q, cache = inputs(3, T, 4, 2, 64, S, F16)
    pos = S - T
    out = torch.full_like(q, 9)
    got = ops.attn_cache(q, cache, at(pos), scale=-0.3, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(out, *reference(q, cache, [pos] * 3, scale=-0.3))


@pytest.mark.parametrize("S,T,window", [(50, 4, None), (50, 4, 6), (2500, 4, None), (50, 40, 6), (2500, 1, None), (17000, 4, None), (17000, 1, None)])
def test_padding_and_positions_outside(S, T, window):
    """Rows behind a sequence's end are left as they were; a query before position 0 gets zeros, one behind the cache sees what there is."""
    q, cache = inputs(8, T, 4, 2, 64, S, F16)
    pos = [0, 10, -2, S - 2, S + 3, -1000, 1 << 40, 5]
    counts = [T, 0, T, T, max(1, T - 1), T, T, -3]
    out = torch.full_like(q, 9)
    ops.attn_cache(q, cache, at(*pos), window=window, counts=at(*counts), out=out)
    want, bound = reference(q, cache, [min(p, 1 << 30) for p in pos], window, counts=counts)
    for b in range(8):
        n = max(0, counts[b])
        check(out[b, :n], want[b, :n], bound[b, :n])
        assert bool((out[b, n:] == 9).all())
    assert not out[5].any() and (window is None or not out[6].any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S,T", [(80, 1), (2300, 1), (80, 5), (2300, 5), (80, 40), (17000, 1), (17000, 5)])
def test_what_is_not_seen_does_not_matter(S, T, dtype):
    """NaN constants in rows that no query sees, and in one that some tokens see and others do not."""
    q, cache = inputs(2, T, 4, 2, 128, S, dtype)
    pos, window, sinks = [S - T - 3, 40], 12 if S < 10000 else 16600, 2
    want, bound = reference(q, cache, pos, window, sinks)
    nan = float("nan")
    for b, p in enumerate(pos):
        for t in (cache.k_scales, cache.v_scales):
            t[b, :, sinks:max(sinks, p - window + 1)] = nan
            t[b, :, p + T:] = nan
    check(ops.attn_cache(q, cache, at(*pos), window=window, sinks=sinks), want, bound)
    if T > 1:                                  # the last token's own row: the others come out as before
        cache.v_scales[0, :, pos[0] + T - 1, 0] = nan
        cache.k_scales[1, :, pos[1] + T - 1] = nan
        got = ops.attn_cache(q, cache, at(*pos), window=window, sinks=sinks)
        check(got[:, :-1], want[:, :-1], bound[:, :-1])
        group = 32
        assert torch.isnan(got[0, -1, :, :group]).all() and torch.isnan(got[1, -1]).all()
        check(got[0, -1, :, group:], want[0, -1, :, group:], bound[0, -1, :, group:])


@pytest.mark.parametrize("S,T,window", [(80, 1, None), (2300, 1, None), (2300, 5, 40), (90, 6, 20), (90, 40, None), (17000, 1, None), (17000, 5, 16600)])
def test_rows_of_an_older_text_do_not_matter(S, T, window):
    """What lies behind the last token and in front of the window: numbers as large as there are, which must not widen what weights are scaled by."""
    q, cache = inputs(2, T, 4, 2, 128, S, F16)
    pos, sinks = [S - T - 7, 37], 2 if window else 0
    want, bound = reference(q, cache, pos, window, sinks)
    for b, p in enumerate(pos):
        for t in (cache.k_scales, cache.v_scales):
            t[b, :, p + T:] = 8736.0 if t is cache.v_scales else -60000.0
            if window:
                t[b, :, sinks:max(sinks, p - window + 1)] = 8736.0
    check(ops.attn_cache(q, cache, at(*pos), window=window, sinks=sinks), want, bound)


def test_queries_and_values_of_all_sizes():
    """Scales of V from the smallest to the largest, queries from 2^-20 to 2^14 in one row and between rows."""
    for dtype in (F16, BF16):
        for S in (100, 2400, 14000):
            q, cache = inputs(1, 1, 8, 2, 128, S, dtype)
            q *= torch.exp2(torch.linspace(-6, 1, 128, device=DEV)).to(dtype)
            q[:, :, 1] *= 2.0 ** -8
            q[:, :, 5] = 0
            factor = torch.exp2(torch.linspace(-13, 9, S, device=DEV))[torch.randperm(S, generator=torch.Generator().manual_seed(1)).to(DEV)]
            cache.v_scales.mul_(factor[:, None, None].to(dtype))
            check(ops.attn_cache(q, cache, at(S - 1)), *reference(q, cache, [S - 1]))
            cache.v_scales.mul_(2.0 ** -10)
            check(ops.attn_cache(q, cache, at(S - 1)), *reference(q, cache, [S - 1]))
            cache.v_scales.zero_()
            assert not ops.attn_cache(q, cache, at(S - 1)).any()
    q, cache = inputs(1, 1, 2, 1, 64, 40, BF16)
    cache.v_scales.mul_(2.0 ** 100)            # beyond fp16's range
    check(ops.attn_cache(q, cache, at(39)), *reference(q, cache, [39]))
    q.mul_(2.0 ** 60)
    cache.k_scales.mul_(2.0 ** -60)
    check(ops.attn_cache(q, cache, at(39)), *reference(q, cache, [39]))


@pytest.mark.parametrize("S,T", [(64, 1), (2222, 2), (90, 50), (15000, 2)])
def test_views(S, T):
    """Queries out of a q|k|v, an output with rows apart, a cache cut out of a larger one."""
    B, heads, kv, hd = 2, 4, 2, 128
    g = torch.Generator(device=DEV).manual_seed(5)
    whole = ops.QuantCache.empty(B + 1, kv + 1, S + 8, hd, 32, F16, DEV)
    rows = [torch.randn(B + 1, S + 8, kv + 1, hd, generator=g, device=DEV).half() for _ in range(2)]
    ops.cache_write(whole, *rows, at(0))
    cache = ops.QuantCache(*(t[1:, :kv, 3:S + 3] for t in (whole.k, whole.v, whole.k_scales, whole.v_scales)))
    qkv = torch.randn(B, T, heads + 2 * kv, hd, generator=g, device=DEV).half()
    q = qkv[:, :, :heads]
    out = torch.zeros(B, heads, T, hd + 24, dtype=F16, device=DEV).transpose(1, 2)[..., :hd]
    ops.attn_cache(q, cache, at(S - T, 7), out=out)
    check(out, *reference(q, cache, [S - T, 7]))


@pytest.mark.parametrize("S,T", [(700, 1), (2600, 1), (700, 33), (17000, 1)])
def test_on_another_stream_and_from_a_graph(S, T):
    q, cache = inputs(2, T, 4, 2, 128, S, F16)
    pos = at(5, 100)
    want = ops.attn_cache(q, cache, pos)
    s = torch.cuda.Stream(DEV)
    s.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(s):
        other = ops.attn_cache(q, cache, pos)
    torch.cuda.current_stream(DEV).wait_stream(s)
    assert torch.equal(want, other)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.attn_cache(q, cache, pos))
    pos.copy_(at(S - T, S // 2))
    want = ops.attn_cache(q, cache, pos)
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    for _ in range(10):                        # two captured calls at once: neither holds what the other writes
        for o in outs:
            o.zero_()
        for st, gr in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream(DEV))
            with torch.cuda.stream(st):
                gr.replay()
        for st in streams:
            torch.cuda.current_stream(DEV).wait_stream(st)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_far_rows_of_a_large_cache():
    """Rows whose offsets pass 32 bits."""
    kv, hd, S, n = 3, 128, (1 << 25) + 5, 300
    cache = ops.QuantCache.empty(1, kv, S, hd, 64, F16, DEV)
    g = torch.Generator(device=DEV).manual_seed(5)
    k, v = (torch.randn(1, n, kv, hd, generator=g, device=DEV).half() for _ in range(2))
    q = torch.randn(1, 1, 2 * kv, hd, generator=g, device=DEV).half()
    ops.cache_write(cache, k, v, at(S - n))
    end = ops.QuantCache(*(t[:, :, S - n:] for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)))
    want, bound = reference(q, end, [n - 1], 256)
    check(ops.attn_cache(q, cache, at(S - 1), window=256), want, bound)


def test_refusals():
    q, cache = inputs(2, 3, 4, 2, 64, 20, F16)
    pos = at(0)
    for error, call in [
        (TypeError, lambda: ops.attn_cache(None, cache, pos)),
        (TypeError, lambda: ops.attn_cache(q.bfloat16(), cache, pos)),
        (TypeError, lambda: ops.attn_cache(q, cache, pos.int())),
        (TypeError, lambda: ops.attn_cache(q, cache, pos, window=1.5)),
        (TypeError, lambda: ops.attn_cache(q, cache, pos, scale="1")),
        (RuntimeError, lambda: ops.attn_cache(q.cpu(), cache, pos)),
        (RuntimeError, lambda: ops.attn_cache(q.clone().requires_grad_(), cache, pos)),
        (ValueError, lambda: ops.attn_cache(q[:1], cache, pos)),
        (ValueError, lambda: ops.attn_cache(q[:, :, :3], cache, pos)),
        (ValueError, lambda: ops.attn_cache(torch.zeros(2, 3, 4, 128, dtype=F16, device=DEV), cache, pos)),
        (ValueError, lambda: ops.attn_cache(q[:, :0], cache, pos)),
        (ValueError, lambda: ops.attn_cache(q, cache, at(0, 0, 0))),
        (ValueError, lambda: ops.attn_cache(q, cache, pos, window=0)),
        (ValueError, lambda: ops.attn_cache(q, cache, pos, sinks=3)),
        (ValueError, lambda: ops.attn_cache(q, cache, pos, window=4, sinks=-1)),
        (ValueError, lambda: ops.attn_cache(q, cache, pos, counts=at(1, 1))),
        (ValueError, lambda: ops.attn_cache(q, cache, pos, out=q)),
        (ValueError, lambda: ops.attn_cache(q, cache, pos, out=torch.zeros_like(q)[:1].expand(2, -1, -1, -1))),
        (ValueError, lambda: ops.attn_cache(torch.zeros(2 * 3 * 4 * 64 + 1, dtype=F16, device=DEV)[1:].view(2, 3, 4, 64), cache, pos)),
    ]:
        with pytest.raises(error):
            call()
