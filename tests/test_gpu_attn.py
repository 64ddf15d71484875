"""Attention with a window and sinks, and behind a shared prefix (ops.attn_window, ops.attn_prefix), against 64 bits.

The bound, per output element, with u = half a step of the type (2^-11 fp16, 2^-8 bf16), A = sum_j w_j |v_j| / sum_j w_j and n visible keys:

    u |o|                             the result's rounding
    + u A                             each weight is rounded to the type before it multiplies v (relative), the denominator is not
    + n 2^-25 max|v|                  fp16 only: weights below 2^-14 are subnormal, half a step of these is 2^-25 (the largest weight is 1)
    + 2 d A                           d: error of a score in fp32, hd products and sums, each off by 2^-22 of the sum of |q k| at most
                                      (2^-24 for rounded sums; the tensor cores may truncate), which moves a weight and the denominator
    + (n 2^-22 + 2^-18) A             sums of n products in fp32 likewise; exp2, scale, merging of parts: a few steps of 2^-22 each
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")

F16, BF16 = torch.float16, torch.bfloat16


def reference(q, k, v, pos, window=None, sinks=0, kp=None, vp=None, scale=None):
    """(output, bound) in 64 bits; pos: list of positions of token 0.  Rows of k and v that a query does not see are never looked at."""
    B, T, heads, hd = q.shape
    kv, S = k.shape[1], k.shape[2]
    G, u = heads // kv, torch.finfo(q.dtype).eps / 2
    scale = hd ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    if kp is not None:
        kp, vp = kp.double().cpu(), vp.double().cpu()
    for b in range(B):
        for t in range(T):
            p = pos[b] + t
            seen = [j for j in range(min(p + 1, S)) if window is None or j > p - window or j < sinks]
            for h in range(kv):
                K, V = k[b, h, seen], v[b, h, seen]
                if kp is not None:
                    K, V = torch.cat([kp[h], K]), torch.cat([vp[h], V])
                n = K.shape[0]
                if n == 0:
                    continue
                Q = q[b, t, h * G:h * G + G]
                w = torch.softmax(Q @ K.t() * scale, dim=1)
                o, A = w @ V, w @ V.abs()
                d = hd * 2.0 ** -22 * (Q.abs() @ K.abs().t()).amax(1, keepdim=True) * abs(scale)
                err = u * o.abs() + (u + 2 * d + n * 2.0 ** -22 + 2.0 ** -18) * A
                if u == 2.0 ** -11:
                    err = err + n * 2.0 ** -25 * V.abs().max()
                out[b, t, h * G:h * G + G], bound[b, t, h * G:h * G + G] = o, err
    return out, bound


def inputs(B, T, heads, kv, hd, S, dtype, seed=0, P=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=dtype)
    q, k, v = 1.5 * r(B, T, heads, hd) + 0.5, r(B, kv, S, hd), r(B, kv, S, hd)
    k[:, :, :3] += 0.5                        # the first keys lie along the queries
    return (q, k, v) if P is None else (q, k, v, r(kv, P, hd), r(kv, P, hd))


def check(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound.clamp(min=1e-30)).max()):.3g} times the bound"


def at(*pos):
    return torch.tensor(pos, device=DEV)


WINDOW = [
    # B, T, heads, kv, hd, max_seq, positions, window, sinks
    (1, 1, 4, 4, 128, 64, [0], 1, 0),                 # the very first token
    (1, 1, 4, 4, 128, 64, [63], 1, 0),                # sees itself alone
    (1, 1, 4, 4, 64, 64, [63], 1, 4),
    (1, 1, 32, 32, 128, 768, [700], 512, 4),
    (3, 1, 8, 8, 128, 333, [5, 332, 100], 40, 4),     # shorter than, longer than the window
    (2, 1, 14, 2, 64, 333, [17, 332], 33, 0),         # groups of seven heads
    (2, 1, 16, 1, 128, 100, [15, 99], 64, 7),         # sixteen rows
    (1, 1, 40, 2, 128, 100, [99], 64, 16),            # twenty rows: two tiles
    (2, 1, 4, 4, 128, 50, [49, 10], 1000, 4),         # the window holds everything
    (2, 1, 4, 4, 128, 50, [49, 10], 8, 45),           # nearly everything is a sink
    (1, 1, 2, 2, 64, 5000, [4999], 4500, 130),
    (40, 1, 8, 8, 64, 40, list(range(40)), 9, 3),
    (2, 2, 4, 4, 128, 100, [0, 98], 5, 2),            # short runs of tokens
    (2, 5, 12, 4, 64, 100, [3, 95], 17, 1),
    (1, 3, 7, 7, 128, 65, [62], 16, 16),
    (1, 33, 4, 4, 128, 100, [50], 20, 4),             # prompts and chunks of them
    (2, 70, 4, 2, 64, 75, [0, 5], 16, 4),
    (1, 129, 2, 1, 128, 300, [171], 64, 0),
    (1, 200, 6, 2, 128, 200, [0], 1, 0),
    (1, 257, 2, 2, 64, 257, [0], 300, 0),             # causal
    (1, 300, 3, 3, 128, 300, [0], 130, 140),
    (1, 130, 1, 1, 64, 1000, [800], 129, 1),
    (1, 20, 32, 1, 128, 90, [60], 50, 2),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(map(str, c[:6] + c[7:])))
def test_window(case, dtype):
    B, T, heads, kv, hd, S, pos, window, sinks = case
    q, k, v = inputs(B, T, heads, kv, hd, S, dtype, seed=T + S)
    got = ops.attn_window(q, k, v, at(*pos), window, sinks)
    assert got.shape == q.shape and got.dtype == dtype
    check(got, *reference(q, k, v, pos, window, sinks))
    assert torch.equal(got, ops.attn_window(q, k, v, at(*pos), window, sinks))


PREFIX = [
    # B, T, heads, kv, hd, max_seq, positions, P
    (1, 1, 4, 4, 128, 16, [0], 0),
    (2, 1, 4, 4, 128, 16, [3, 15], 1),
    (3, 1, 8, 8, 64, 33, [0, 32, 7], 17),
    (4, 1, 4, 4, 128, 40, [-1, 0, 39, 20], 500),      # nothing of its own
    (16, 1, 2, 2, 128, 20, list(range(16)), 129),
    (17, 1, 2, 2, 128, 20, list(range(17)), 128),     # one row more than a tile
    (33, 1, 2, 2, 64, 40, list(range(33)), 300),
    (5, 1, 14, 2, 128, 40, [1, 2, 3, 4, 39], 1000),
    (70, 1, 4, 1, 128, 8, [i % 8 for i in range(70)], 260),
    (130, 1, 2, 2, 64, 8, [i % 8 for i in range(130)], 1500),
    (2, 3, 4, 2, 128, 30, [0, 27], 77),
    (2, 40, 4, 4, 64, 60, [0, 20], 200),
    (3, 70, 6, 2, 128, 70, [0, 0, 0], 333),
    (1, 150, 2, 1, 128, 180, [20], 128),
    (2, 131, 1, 1, 64, 140, [0, 9], 3),
    (1, 1, 32, 1, 128, 64, [40], 700),
    # so much that it goes before, in parts: up to 8, 16, 32, 128, 256 and more rows per key head
    (2, 1, 2, 2, 128, 40, [0, 39], 40001),
    (12, 1, 1, 1, 128, 40, list(range(12)), 6100),
    (8, 1, 6, 2, 64, 40, list(range(8)), 10007),
    (70, 1, 4, 4, 64, 8, [i % 8 for i in range(70)], 1500),
    (130, 1, 2, 2, 64, 8, [i % 8 - 1 for i in range(130)], 600),
    (11, 3, 10, 2, 128, 40, list(range(11)), 3333),
    (90, 1, 4, 1, 128, 5, [i % 5 for i in range(90)], 1111),
    (5, 60, 1, 1, 64, 70, list(range(5)), 40000),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", PREFIX, ids=lambda c: "-".join(map(str, c[:6] + c[7:])))
def test_prefix(case, dtype):
    B, T, heads, kv, hd, S, pos, P = case
    q, k, v, kp, vp = inputs(B, T, heads, kv, hd, S, dtype, seed=B + P, P=P)
    got = ops.attn_prefix(q, kp, vp, k, v, at(*pos))
    check(got, *reference(q, k, v, pos, kp=kp, vp=vp))
    assert torch.equal(got, ops.attn_prefix(q, kp, vp, k, v, at(*pos)))


@pytest.mark.parametrize("T", [1, 4, 150])
def test_queries_outside_the_cache(T):
    """Before position 0: nothing is seen, zeros.  Behind the cache's end: what the window still has of it, and the sinks."""
    q, k, v = inputs(4, T, 4, 2, 64, 40, F16)
    pos = [-1, 40, 45, -(1 << 40)]
    got = ops.attn_window(q, k, v, at(*pos), 8, 3)
    check(got, *reference(q, k, v, pos[:3] + [-10 ** 6], 8, 3))
    assert bool((got[0, 0] == 0).all()) and bool((got[3] == 0).all())
    far = ops.attn_window(q, k, v, at(1 << 40), 8, 0)
    assert bool((far == 0).all())


@pytest.mark.parametrize("prefix", [None, 30])
@pytest.mark.parametrize("T,G", [(1, 1), (3, 2), (140, 2)])
def test_padding_is_left_alone(T, G, prefix):
    B = 4
    case = inputs(B, T, 2 * G, 2, 64, T + 20, F16, P=prefix)
    counts = [T, 0, 1, (T + 1) // 2]
    out = torch.full_like(case[0], 7.0)
    if prefix is None:
        r = ops.attn_window(case[0], case[1], case[2], at(4), 10, 2, counts=at(*counts), out=out)
        want, bound = reference(*case, [4] * B, 10, 2)
    else:
        r = ops.attn_prefix(case[0], case[3], case[4], case[1], case[2], at(4), counts=at(*counts), out=out)
        want, bound = reference(*case[:3], [4] * B, kp=case[3], vp=case[4])
    assert r is out
    for b, n in enumerate(counts):
        check(out[b, :n], want[b, :n], bound[b, :n])
        assert bool((out[b, n:] == 7).all())


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("T,window,sinks", [(1, 20, 4), (4, 20, 4), (1, 300, 0), (150, 20, 4), (150, 300, 0)])
def test_rows_that_are_not_seen_do_not_matter(T, window, sinks, junk):
    """NaN and infinities behind the last position, between the sinks and the window, and, for tokens of one call, in a row that only the later
    ones see."""
    S, p = 400, 200
    q, k, v = inputs(2, T, 4, 2, 128, S, F16)
    want, bound = reference(q, k, v, [p, p], window, sinks)
    k[:, :, p + T:], v[:, :, p + T:] = junk, junk
    if p - window + 1 > sinks:
        k[:, :, sinks:p - window + 1], v[:, :, sinks:p - window + 1] = junk, junk
    check(ops.attn_window(q, k, v, at(p), window, sinks), want, bound)
    if T > 1:
        late = p + T // 2                     # seen from there on, while the window holds it
        k[:, :, late], v[:, :, late] = junk, junk
        got = ops.attn_window(q, k, v, at(p), window, sinks)
        sees = [t for t in range(T) if late <= p + t and (late > p + t - window)]
        rest = [t for t in range(T) if t not in sees]
        check(got[:, rest], want[:, rest], bound[:, rest])
        assert bool(got[:, sees].isnan().any()) or junk == -math.inf


@pytest.mark.parametrize("T", [1, 5, 150, 3000])
def test_nan_that_is_seen_is_passed_on(T):
    """A NaN in one query, in one key or in one dim of one value: those rows and dims are NaN, and no others."""
    S, p, W = T + 300, 200, 40
    q, k, v = inputs(1, T, 2, 1, 64, S, F16)
    clean = ops.attn_window(q, k, v, at(p), W, 2)
    bad = q.clone()
    bad[0, T // 2, 1, 7] = math.nan
    got = ops.attn_window(bad, k, v, at(p), W, 2)
    assert bool(got[0, T // 2, 1].isnan().all())
    got[0, T // 2, 1] = clean[0, T // 2, 1]
    assert torch.equal(got, clean)
    j = p + T // 2
    sees = torch.tensor([j <= p + t < j + W for t in range(T)])
    bad = k.clone()
    bad[0, 0, j, 3] = math.nan
    got = ops.attn_window(q, bad, v, at(p), W, 2)[0].cpu()
    assert bool(got[sees].isnan().all()) and not bool(got[~sees].isnan().any())
    bad = v.clone()
    bad[0, 0, j, 3] = math.inf
    got = ops.attn_window(q, k, bad, at(p), W, 2)[0].cpu()
    assert bool((got[sees][..., 3] == math.inf).all()) and bool(torch.isfinite(got[~sees]).all())
    assert bool(torch.isfinite(got[..., :3]).all()) and bool(torch.isfinite(got[..., 4:]).all())
    assert bool(ops.attn_window(q * math.nan, k, v, at(p), W, 2).isnan().all())


@pytest.mark.parametrize("T", [1, 140])
def test_caches_that_repeat(T):
    """Batches and heads that are one (stride 0), which a tensor map cannot say."""
    q, k, v = inputs(3, T, 4, 2, 64, 200, F16)
    k, v = k[:1, :1].expand(3, 2, 200, 64), v[:1].expand(3, 2, 200, 64)
    check(ops.attn_window(q, k, v, at(3, 9, 40), 30, 2), *reference(q, k, v, [3, 9, 40], 30, 2))
    kp, vp = inputs(1, 1, 1, 1, 64, 99, F16, seed=5)[1:]
    kp, vp = kp[0].expand(2, 99, 64), vp[0].expand(2, 99, 64)
    check(ops.attn_prefix(q, kp, vp, k, v, at(3, 9, 40)), *reference(q, k, v, [3, 9, 40], kp=kp, vp=vp))
    check(ops.attn_prefix(q[:1].expand(3, T, 4, 64), kp, vp, k, v, at(3, 9, 40)), *reference(q[:1].expand(3, T, 4, 64), k, v, [3, 9, 40], kp=kp, vp=vp))


def test_junk_behind_the_own_rows_with_a_prefix():
    for T in (1, 5, 140):
        q, k, v, kp, vp = inputs(3, T, 4, 2, 128, 200, F16, P=100)
        want, bound = reference(q, k, v, [0, 9, 30], kp=kp, vp=vp)
        for b, p in enumerate([0, 9, 30]):
            k[b, :, p + T:], v[b, :, p + T:] = math.nan, math.inf
        check(ops.attn_prefix(q, kp, vp, k, v, at(0, 9, 30)), want, bound)


@pytest.mark.parametrize("T", [1, 6, 140])
def test_strided_views(T):
    """q out of a packed q|k|v, caches laid out [batch, position, head, dim] and cut out of larger ones, out with room between its rows."""
    B, heads, kv, hd, S = 2, 4, 2, 64, 200
    g = torch.Generator(device=DEV).manual_seed(3)
    packed = torch.randn(B, T, 3, heads, hd, generator=g, device=DEV, dtype=F16)
    q = packed[:, :, 0]
    k = torch.randn(B, S + 9, kv + 1, 2 * hd, generator=g, device=DEV, dtype=F16)[:, 5:5 + S, 1:, hd:].permute(0, 2, 1, 3)
    v = torch.randn(kv, B, S, hd, generator=g, device=DEV, dtype=F16).transpose(0, 1)
    room = torch.zeros(B, T, heads, 2 * hd, device=DEV, dtype=F16)
    out = room[..., hd:]
    pos = [30, 33]
    ops.attn_window(q, k, v, at(*pos), 25, 3, out=out)
    check(out, *reference(q, k, v, pos, 25, 3))
    assert bool((room[..., :hd] == 0).all())
    kp = torch.randn(100, kv, hd, generator=g, device=DEV, dtype=F16).transpose(0, 1)
    vp = torch.randn(kv, 120, hd, generator=g, device=DEV, dtype=F16)[:, 11:111]
    ops.attn_prefix(q, kp, vp, k, v, at(*pos), out=out)
    check(out, *reference(q, k, v, pos, kp=kp, vp=vp))


@pytest.mark.parametrize("T", [1, 140])
def test_offsets_past_32_bits(T):
    """A cache whose rows lie 2^25 elements apart, 200 of them: offsets up to 13 GB, past 2^32 elements."""
    S, hd, step = 200, 64, 1 << 25
    buf = torch.zeros(S * step, device=DEV, dtype=F16)
    q, k0, v0 = inputs(1, T, 2, 1, hd, S, F16)
    k, v = (buf.as_strided((1, 1, S, hd), (S * step, S * step, step, 1), o) for o in (0, 1024))
    k.copy_(k0)
    v.copy_(v0)
    check(ops.attn_window(q, k, v, at(S - T), 150, 4), *reference(q, k0, v0, [S - T], 150, 4))
    check(ops.attn_prefix(q, k[0], v[0], k0, v0, at(3)), *reference(q, k0, v0, [3], kp=k0[0], vp=v0[0]))


@pytest.mark.parametrize("T", [1, 140])
def test_scale(T):
    q, k, v = inputs(1, T, 2, 2, 64, 200, F16)
    for scale in (0.0, -0.1, 0.5):
        check(ops.attn_window(q, k, v, at(50), 40, 4, scale=scale), *reference(q, k, v, [50], 40, 4, scale=scale))


def test_large_scores():
    """Scores of several thousand: weights of all but one key vanish."""
    for T in (1, 140):
        q, k, v = inputs(1, T, 2, 2, 128, 300, F16)
        check(ops.attn_window(30 * q, 10 * k, v, at(100), 120, 4), *reference(30 * q, 10 * k, v, [100], 120, 4))


@pytest.mark.parametrize("T", [1, 140])
def test_other_streams_and_graphs(T):
    """On a side stream; captured, with positions that move on between replays; two graphs that share nothing, replayed side by side."""
    B, S, P = 3, 400, 300
    q, k, v, kp, vp = inputs(B, T, 4, 2, 128, S, F16, P=P)
    pos = at(10, 20, 30)
    want = [ops.attn_window(q, k, v, pos + i, 50, 4) for i in range(3)], [ops.attn_prefix(q, kp, vp, k, v, pos + i) for i in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = ops.attn_window(q, k, v, pos, 50, 4), ops.attn_prefix(q, kp, vp, k, v, pos)
    side.synchronize()
    assert torch.equal(a, want[0][0]) and torch.equal(b, want[1][0])
    graphs = []
    for _ in range(2):
        p, gr = pos.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            x, y = ops.attn_window(q, k, v, p, 50, 4), ops.attn_prefix(q, kp, vp, k, v, p)
            p.add_(1)
        graphs.append((gr, x, y, torch.cuda.Stream(), p))        # (the graph reads p where it lies)
    for i in range(3):
        for gr, _, _, s, _ in graphs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                gr.replay()
        for _, x, y, s, _ in graphs:
            s.synchronize()
            assert torch.equal(x, want[0][i]) and torch.equal(y, want[1][i])


@pytest.mark.parametrize("T", [1, 4, 140])
def test_a_chain_of_calls_sees_what_was_written_just_before(T):
    """Keys written by the operation in front of the call, outputs read by the one behind it, again and again without a synchronisation."""
    B, S = 2, 400
    q, k, v, kp, vp = inputs(B, T, 4, 4, 128, S, F16, P=200)
    steps = [torch.randn_like(k) for _ in range(8)]
    got = []
    for s in steps:
        k.copy_(s)
        x = ops.attn_prefix(q, kp, vp, k, v, at(7))
        got.append(ops.attn_window(x, k, v, at(99), 64, 2))
    for s, g in zip(steps, got):
        x = ops.attn_prefix(q, kp, vp, s, v, at(7))
        torch.cuda.synchronize()
        assert torch.equal(g, ops.attn_window(x, s, v, at(99), 64, 2))


def test_refusals():
    q, k, v, kp, vp = inputs(2, 1, 4, 2, 64, 40, F16, P=16)
    p = at(3)
    W = lambda *a, **kw: ops.attn_window(*a, **kw)
    for bad, error in [
        (lambda: W(q.float(), k, v, p, 4), TypeError), (lambda: W(q, k.bfloat16(), v, p, 4), TypeError),
        (lambda: W(q[..., :32], k[..., :32], v[..., :32], p, 4), ValueError), (lambda: W(q[:, :, :3], k, v, p, 4), ValueError),
        (lambda: W(q, k[:1], v[:1], p, 4), ValueError), (lambda: W(q, k, v[:, :, :30], p, 4), ValueError),
        (lambda: W(q, k, v, p.int(), 4), TypeError), (lambda: W(q, k, v, at(1, 2, 3), 4), ValueError),
        (lambda: W(q, k, v, p, 0), ValueError), (lambda: W(q, k, v, p, -1), ValueError), (lambda: W(q, k, v, p, 4, -1), ValueError),
        (lambda: W(q, k, v, p, 1 << 40), ValueError), (lambda: W(q, k, v, p, 4.5), TypeError), (lambda: W(q, k, v, p, 4, scale="x"), TypeError),
        (lambda: W(q, k, v, p, 4, counts=at(1, 1)), ValueError), (lambda: W(q, k, v, p, 4, counts=at(1), out=torch.empty_like(q)), ValueError),
        (lambda: W(q, k, v, p, 4, out=q), ValueError), (lambda: W(q, k, v, p, 4, out=torch.empty_like(q)[:, :, :2]), ValueError),
        (lambda: W(q, k, v, p, 4, out=torch.empty(1, 1, 4, 64, device=DEV, dtype=F16).expand(2, 1, 4, 64)), ValueError),
        (lambda: W(q[0], k, v, p, 4), ValueError), (lambda: W(q[:0], k[:0], v[:0], p, 4), ValueError), (lambda: W(q[:, :0], k, v, p, 4), ValueError),
        (lambda: W(q, k.cpu(), v, p, 4), RuntimeError), (lambda: W(q, k, v, p.cpu(), 4), RuntimeError), (lambda: W(q, k, None, p, 4), TypeError),
        (lambda: W(q.requires_grad_(), k, v, p, 4), RuntimeError),
        (lambda: ops.attn_prefix(q.detach(), kp, None, k, v, p), TypeError), (lambda: ops.attn_prefix(q.detach(), kp[:1], vp[:1], k, v, p), ValueError),
        (lambda: ops.attn_prefix(q.detach(), kp, vp[:, :4], k, v, p), ValueError), (lambda: ops.attn_prefix(q.detach(), kp.float(), vp, k, v, p), TypeError),
    ]:
        with pytest.raises(error):
            bad()
    q = q.detach()
    flat = torch.zeros(2 * 4 * 64 + 8, device=DEV, dtype=F16)
    with pytest.raises(ValueError, match="16 bytes"):
        W(flat[1:1 + 2 * 4 * 64].view(2, 1, 4, 64), k, v, p, 4)
    with pytest.raises(ValueError, match="16 bytes"):
        W(q, k[:, :, :, :].as_strided(k.shape, (40 * 2 * 64, 40 * 64, 63, 1)), v, p, 4)
    with torch.no_grad():
        W(q.clone().requires_grad_(), k, v, p, 4)


def test_a_given_output_counts_a_write():
    q, k, v = inputs(1, 1, 2, 2, 64, 40, F16)
    out = torch.empty_like(q)
    before = out._version
    ops.attn_window(q, k, v, at(3), 4, out=out)
    assert out._version == before + 1


@pytest.mark.parametrize("strides", [(256, 256, 32, 1), (256, 256, 0, 1), (64, 256, 64, 1), (128, 256, 64, 1)])
def test_an_output_whose_rows_share_memory_is_refused(strides):
    q, k, v = inputs(3, 1, 4, 2, 64, 40, F16)
    out = torch.zeros(2000, device=DEV, dtype=F16).as_strided(q.shape, strides)
    with pytest.raises(ValueError, match="overlap"):
        ops.attn_window(q, k, v, at(3), 4, out=out)


def test_outputs_in_any_order_of_dimensions_are_taken():
    q, k, v = inputs(3, 5, 4, 2, 64, 40, F16)
    want = ops.attn_window(q, k, v, at(3), 9, 1)
    for order in ((0, 1, 2), (2, 0, 1), (1, 2, 0), (2, 1, 0)):
        shape = [q.shape[i] for i in order]
        out = torch.zeros(*shape, 72, device=DEV, dtype=F16)[..., :64].permute(*(order.index(i) for i in range(3)), 3)
        assert torch.equal(ops.attn_window(q, k, v, at(3), 9, 1, out=out), want)


def microseconds(call, n=5):
    for _ in range(2):
        call()
    e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    torch.cuda.synchronize()
    e[0].record()
    for _ in range(n):
        call()
    e[1].record()
    e[1].synchronize()
    return e[0].elapsed_time(e[1]) * 1000 / n


@pytest.mark.parametrize("dtype,junk", [(F16, math.nan), (BF16, math.nan), (F16, math.inf), (F16, -math.inf)])
@pytest.mark.parametrize("T,B", [(4096, 1), (1, 32)])
def test_one_value_that_is_not_finite_does_not_slow_a_call_down(T, B, dtype, junk):
    """In one dim of a sink's value, which every row sees: that dim is it in every row, and the call takes about as long as without.  (Where each row
    is done again key by key it takes hundreds of times as long; the bound of ten leaves room for other users of the machine.)"""
    q, k, v = inputs(B, T, 8, 8, 128, 4096, dtype)
    pos = at(4096 - T)
    clean = ops.attn_window(q, k, v, pos, 2000, 4)
    before = microseconds(lambda: ops.attn_window(q, k, v, pos, 2000, 4))
    v[:, :, 0, 77] = junk
    got = ops.attn_window(q, k, v, pos, 2000, 4)
    assert bool((got[..., 77].isnan() if math.isnan(junk) else got[..., 77] == junk).all())
    rest = [d for d in range(128) if d != 77]
    assert torch.equal(got[..., rest], clean[..., rest])
    assert microseconds(lambda: ops.attn_window(q, k, v, pos, 2000, 4)) < 10 * before
