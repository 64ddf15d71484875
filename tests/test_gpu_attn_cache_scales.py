"""Attention over a cache in 4 bits whose scales of V differ by group, by key and by weight: what a small weight or another group or row has to do with is the
values, not how large a scale stands beside them.

The bound, per output element, in the terms of tests/test_gpu_attn_cache.py (u half a step of the type, A = sum_j w_j |V_j|+ / sum_j w_j, d error of a score), but with
T = max_j w_j s_j / sum_j w_j over the row's own visible keys, s_j the scale of the element's own group:

    u |o| + 2^-11 A                   the result's rounding; each weight times scale rounded to fp16 (relative)
    + n 2^-31 8 T                     weights times scales are held so that the largest so far lies between 2^6 and 2^16: what is below 2^-14 is off by 2^-25 at most, codes
                                      less 8 are 8 at most
    + (2 d + n 2^-22 + 2^-18) A       as there

All calls here have fewer than 64 rows per key head and few key heads, so none of them is read back.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")

F16, BF16 = torch.float16, torch.bfloat16


def parts(packed, constants):
    """(code, scale, zero) of each dim in 64 bits."""
    hd = packed.shape[-1] * 2
    d = torch.arange(hd, device=packed.device)
    word = d % 32 // 4 * (hd // 64) + d // 64
    field = d % 2 * 4 + d % 4 // 2 + d % 64 // 32 * 2
    codes = packed[..., word * 4 + field // 2].long() >> 4 * (field % 2) & 15
    wide = constants.double().repeat_interleave(hd // constants.shape[-2], -2)
    return codes.double(), wide[..., 0], wide[..., 1]


def reference(q, cache, pos, window=None, sinks=0):
    B, T, heads, hd = q.shape
    kv, S = cache.k.shape[1:3]
    G, u, scale = heads // kv, torch.finfo(q.dtype).eps / 2, hd ** -0.5
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    j = torch.arange(S, device=DEV)
    for b in range(B):
        for h in range(kv):
            (kc, ks, kz), (vc, vs, vz) = parts(cache.k[b, h], cache.k_scales[b, h]), parts(cache.v[b, h], cache.v_scales[b, h])
            K, Kp = kz + ks * kc, kz.abs() + ks * kc
            V, Vp = vz + vs * vc, (vz + 8 * vs).abs() + vs * (vc - 8).abs()
            for t in range(T):
                p = pos[b] + t
                seen = (j <= p) & ((j > p - window) | (j < sinks)) if window is not None else j <= p
                Q = q[b, t, h * G:h * G + G].double()
                w = torch.softmax(Q @ K[seen].t() * scale, dim=1)
                A = w @ Vp[seen]
                top = (w[:, :, None] * vs[seen][None]).amax(1)
                d = hd * 2.0 ** -22 * (Q.abs() @ Kp[seen].t()).amax(1, keepdim=True) * scale
                n = int(seen.sum())
                out[b, t, h * G:h * G + G] = o = w @ V[seen]
                bound[b, t, h * G:h * G + G] = u * o.abs() + n * 2.0 ** -31 * 8 * top + (2.0 ** -11 + 2 * d + n * 2.0 ** -22 + 2.0 ** -18) * A
    return out, bound


def check(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound.clamp(min=1e-30)).max()):.3g} times the bound"


def made(B, S, kv, hd, group, dtype, log2_weights, seed=0):
    """A cache whose key j has a score of log2_weights[j] for queries of ones (in units of log 2), with random codes in V, scales of 0.1 and zeros of -0.5 .. 0.3."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = ops.QuantCache.empty(B, kv, S, hd, group, dtype, DEV)
    # scores are sums of hd equal products; in bf16 as in fp16 whole and half numbers are exact
    cache.k_scales[..., 1] = (log2_weights.double() * 0.6931471805599453 * hd ** -0.5).to(dtype)[:, None]
    cache.v.copy_(torch.randint(0, 256, cache.v.shape, generator=g, device=DEV, dtype=torch.uint8))
    cache.v_scales[..., 0] = 0.1
    cache.v_scales[..., 1] = (torch.rand(cache.v_scales.shape[:-1], generator=g, device=DEV) * 0.8 - 0.5).to(dtype)
    return cache


def queries(B, T, heads, hd, dtype):
    return torch.ones(B, T, heads, hd, dtype=dtype, device=DEV)


def at(*pos):
    return torch.tensor(pos, device=DEV)


# heads of one key head: 1, 2 and 4 tiles of eight rows; clusters of one and of more CTAs; runs
SIZES = [(heads, S) for heads in (1, 13, 30) for S in (70, 4096, 20000)]


def long_tail(S):
    """A weight of 1 for every 64th key, so that each warp has some, and 2^-10.2 for the others, a third of the sum and a row's share of half of it."""
    where = torch.full((S,), -10.2, device=DEV)
    where[5::64] = 0
    return where


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,group", [(64, 32), (128, 32), (128, 64)])
@pytest.mark.parametrize("heads,S", SIZES)
def test_a_group_of_larger_scales(heads, S, hd, group, dtype):
    """In one group of each row the scale is 40000 times the others'; the tail's codes all lie above 8."""
    cache = made(1, S, 1, hd, group, dtype, long_tail(S))
    cache.v |= 0x88
    cache.v_scales[:, :, :, -1, 0] = 4000
    q = queries(1, 1, heads, hd, dtype)
    check(ops.attn_cache(q, cache, at(S - 1)), *reference(q, cache, [S - 1]))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("place", [0, 7, 63])
@pytest.mark.parametrize("below", [30, 60, 100])
@pytest.mark.parametrize("heads,S", SIZES)
def test_a_key_of_little_weight_and_a_large_scale(heads, S, below, place, dtype):
    """Visible keys (in each warp's part) of weight 2^-below whose values are 80000 times the others'."""
    where = long_tail(S)
    where[place::64] = -below
    cache = made(1, S, 1, 128, 32, dtype, where)
    cache.v |= 0x88
    cache.v_scales[:, :, place::64, :, 0] = 8000
    q = queries(1, 1, heads, 128, dtype)
    check(ops.attn_cache(q, cache, at(S - 1)), *reference(q, cache, [S - 1]))


@pytest.mark.parametrize("S,window", [(1000, 900), (4096, 3000), (20000, 18000)])
@pytest.mark.parametrize("T,heads", [(2, 1), (6, 2), (7, 4)])
def test_a_large_scale_that_other_rows_see(T, heads, S, window):
    """What the first tokens see ends before, and what the last ones see begins behind, keys of the largest values: these come out as without them."""
    cache = made(1, S, 1, 128, 32, F16, long_tail(S))
    cache.v |= 0x88
    pos = S - T
    cache.v_scales[:, :, S - 1, :, 0] = 4000                  # seen by the last token alone
    cache.v_scales[:, :, pos - window + 1, 1, 0] = 4000       # and by the first one alone
    q = queries(1, T, heads, 128, F16)
    check(ops.attn_cache(q, cache, at(pos), window=window), *reference(q, cache, [pos], window))


@pytest.mark.parametrize("heads,S", SIZES)
def test_scores_that_climb_and_scales_that_fall(heads, S):
    """Each key has half the scale and 1.5 times the weight of the one before it: what weights are scaled by follows both."""
    steps = torch.arange(S, device=DEV)
    cache = made(1, S, 1, 128, 32, BF16, steps % 97 * 0.5849625)
    cache.v_scales[..., 0] = torch.exp2(40 - (steps % 97).float()).to(BF16)[:, None]
    cache.v_scales[..., 1] = 0
    q = queries(1, 1, heads, 128, BF16)
    check(ops.attn_cache(q, cache, at(S - 1)), *reference(q, cache, [S - 1]))
    cache.v_scales[..., 0] = torch.exp2((steps % 97).float() - 90).to(BF16)[:, None]
    check(ops.attn_cache(q, cache, at(S - 1)), *reference(q, cache, [S - 1]))


@pytest.mark.parametrize("S", [50, 20000])
def test_the_largest_and_smallest_scales(S):
    """Scales of 2^120 beside 2^-80 by group, and weights that pass fp16's range in both directions."""
    where = torch.zeros(S, device=DEV)
    where[S // 2:] = -20
    where[-1] = 30
    cache = made(2, S, 2, 128, 32, BF16, where)
    cache.v_scales[:, :, :, 0, 0] = 2.0 ** 120
    cache.v_scales[:, :, :, 1, 0] = 2.0 ** -80
    cache.v_scales[:, :, :, 1, 1] = 0
    q = queries(2, 1, 4, 128, BF16)
    check(ops.attn_cache(q, cache, at(S - 1, S - 7)), *reference(q, cache, [S - 1, S - 7]))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S,window", [(40, 1), (3000, None), (20000, None)])
@pytest.mark.parametrize("heads,group", [(1, 32), (13, 64), (30, 32)])
def test_the_largest_weight_is_not_rounded(heads, group, S, window, dtype):
    """A row whose weight lies all on one key comes out as that key's value: the largest weight is a power of two, and times a scale of 16 bits has no rounding.

    u |o| is left, and 2^-17 A for zeros and codes added up in fp32 and the scale's exp2 (a few steps of 2^-22 each).
    """
    g = torch.Generator(device=DEV).manual_seed(3)
    where = torch.full((S,), -60.0, device=DEV)
    where[S - 1] = 0
    cache = made(1, S, 1, 128, group, dtype, where)
    cache.k_scales[..., 1] += cache.k_scales.new_tensor(0.37)                 # (scores that are no whole numbers)
    cache.v_scales[..., 0] = (0.1 + torch.rand(cache.v_scales.shape[:-1], generator=g, device=DEV)).to(dtype)
    q = queries(1, 1, heads, 128, dtype)
    code, scale, zero = (t[0, 0, S - 1] for t in parts(cache.v, cache.v_scales))
    want = (zero + scale * code)[None, None, None].expand(q.shape)
    A = (zero.abs() + 16 * scale)[None, None, None]
    check(ops.attn_cache(q, cache, at(S - 1), window=window), want, torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -17 * A)
