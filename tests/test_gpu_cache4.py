"""The cache in 4 bits: ops.cache_write and ops.cache_read against the format's definition.

Codes and constants are compared exactly with the definition in fp32 on the CPU (whose sums and divisions are rounded as the GPU's), where rows are not
rotated.  Values are held to bounds, with u = half a step of the type (2^-11 fp16, 2^-8 bf16), scale s, zero z and m = the row's largest |x|:

    |value - x| <= s / 2 + 15 u s + u |value| + tiny      nearest code; a scale off by u s, 15 of which pile up at the upper end; the value's own rounding; scales
                                                          below the type's normal numbers are off by half its smallest step, tiny = 15 of these

A rotated element is one rounding (u) of a sum of two exact products that fp32 rounds once (2^-24), relative to |x0| + |x1|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")

F16, BF16 = torch.float16, torch.bfloat16


def dims_of_fields(hd):
    """Dim of field f of word w, as the header has it."""
    return [[64 * (w % (hd // 64)) + 4 * (w // (hd // 64)) + e for e in (0, 2, 32, 34, 1, 3, 33, 35)] for w in range(hd // 8)]


def codes_of(packed):
    """Codes [..., hd] of rows of bytes [..., hd / 2]."""
    hd = packed.shape[-1] * 2
    words = packed.cpu().to(torch.int64).reshape(*packed.shape[:-1], hd // 8, 4)
    words = words[..., 0] | words[..., 1] << 8 | words[..., 2] << 16 | words[..., 3] << 24
    out = torch.zeros(*packed.shape[:-1], hd, dtype=torch.int64)
    for w, dims in enumerate(dims_of_fields(hd)):
        for f, d in enumerate(dims):
            out[..., d] = words[..., w] >> 4 * f & 15
    return out


def defined(x, group):
    """(codes, scales, zeros) of rows [..., hd] in their type, by the definition."""
    g = x.cpu().float().reshape(*x.shape[:-1], -1, group)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).to(x.dtype).float()
    good = torch.isfinite(g).all(-1, keepdim=True) & torch.isfinite(scale)
    codes = torch.where((scale > 0) & good, torch.clamp(torch.round((g - lo) / scale), 0, 15), 0.0)
    nan = torch.tensor(float("nan"))
    return codes.long().reshape(x.shape), torch.where(good, scale, nan)[..., 0], torch.where(good, lo, nan)[..., 0]


def values(cache, which):
    """What the cache stands for, in 64 bits."""
    packed, constants = (cache.k, cache.k_scales) if which == "k" else (cache.v, cache.v_scales)
    codes, c = codes_of(packed).double(), constants.double().cpu()
    g = codes.reshape(*c.shape[:-1], -1)
    return (c[..., 1:] + c[..., :1] * g).reshape(codes.shape)


def rounded(x, dtype):
    """Values as they come out: rounded, and held to the type's largest number."""
    top = torch.finfo(dtype).max
    return x.float().clamp(-top, top).to(dtype).double()


def rows(*shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*shape, generator=g, device=DEV)
    x[..., 3] *= 20                            # a dim that is larger than the others
    return x.to(dtype)


def at(*pos):
    return torch.tensor(pos, device=DEV)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) and torch.equal(torch.isnan(a), torch.isnan(b))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,T,kv,S,pos", [(1, 1, 1, 1, [0]), (1, 1, 32, 40, [39]), (3, 7, 5, 33, [0, 26, 11]), (2, 130, 2, 131, [1]), (70, 2, 3, 9, [4])])
def test_codes_and_constants(B, T, kv, S, pos, hd, group, dtype):
    cache = ops.QuantCache.empty(B, kv, S, hd, group, dtype, DEV)
    k, v = rows(B, T, kv, hd, dtype=dtype), rows(B, T, kv, hd, dtype=dtype, seed=1)
    k_out, v_out = torch.empty_like(k), torch.empty_like(v)
    assert ops.cache_write(cache, k, v, at(*pos), k_out=k_out, v_out=v_out) is None
    u, tiny = torch.finfo(dtype).eps / 2, 15 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    first = (pos * B)[:B] if len(pos) == 1 else pos
    back = ops.cache_read(cache)
    for x, out, packed, constants, name, read in ((k, k_out, cache.k, cache.k_scales, "k", back[0]), (v, v_out, cache.v, cache.v_scales, "v", back[1])):
        codes, scale, zero = defined(x, group)
        stands = values(cache, name)
        assert same(read.double().cpu(), rounded(stands, dtype))
        untouched = torch.ones(B, S, dtype=torch.bool)
        for b, p in enumerate(first):
            untouched[b, p:p + T] = False
            assert torch.equal(codes_of(packed)[b, :, p:p + T], codes[b].transpose(0, 1))
            assert torch.equal(constants[b, :, p:p + T, :, 0].cpu().float(), scale[b].transpose(0, 1))
            assert torch.equal(constants[b, :, p:p + T, :, 1].cpu().float(), zero[b].transpose(0, 1))
            got = stands[b, :, p:p + T].transpose(0, 1)
            assert same(out[b].double().cpu(), rounded(got, dtype))
            s = scale[b].double().repeat_interleave(group, -1)
            off = (out[b].double().cpu() - x[b].double().cpu()).abs()
            assert bool((off <= s / 2 + 15 * u * s + u * got.abs() + tiny).all())
        assert not packed.cpu().transpose(1, 2)[untouched].any() and not constants.cpu().transpose(1, 2)[untouched].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,heads,kv", [(128, 4, 2), (64, 7, 1)])
def test_rotation_on_the_way(hd, heads, kv, dtype):
    """From the columns of one q|k|v, where q, k and v are views."""
    B, T, S, p = 2, 9, 50, [0, 38]
    x = rows(B, T, heads + 2 * kv, hd, dtype=dtype)
    q, k, v = x[:, :, :heads], x[:, :, heads:heads + kv], x[:, :, heads + kv:]
    angle = torch.arange(S, device=DEV)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, device=DEV).double() / hd)
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    cache = ops.QuantCache.empty(B, kv, S, hd, 32, dtype, DEV)
    q_out, k_out, v_out = torch.zeros(B, T, heads, hd, dtype=dtype, device=DEV), *(torch.zeros(B, T, kv, hd, dtype=dtype, device=DEV) for _ in range(2))
    assert ops.cache_write(cache, k, v, at(*p), cos=cos, sin=sin, q=q, q_out=q_out, k_out=k_out, v_out=v_out) is q_out
    u = torch.finfo(dtype).eps / 2
    for b in range(B):
        c, s = (t[p[b]:p[b] + T].double().cpu()[:, None] for t in (cos, sin))
        turned = []
        for y in (q[b], k[b]):
            y = y.double().cpu()
            e, o = y[..., 0::2], y[..., 1::2]
            turned.append(torch.stack([e * c - o * s, e * s + o * c], -1).flatten(-2))
        size = (q[b].double().cpu()[..., 0::2].abs() + q[b].double().cpu()[..., 1::2].abs()).repeat_interleave(2, -1)
        assert bool(((q_out[b].double().cpu() - turned[0]).abs() <= u * turned[0].abs() + 2.0 ** -23 * size + 2.0 ** -25).all())
        # the keys' codes are those of rows that are rounded like the queries: rotated by this very call as queries, they have to come out the same
        again = torch.zeros(1, T, kv, hd, dtype=dtype, device=DEV)
        other = ops.QuantCache.empty(1, kv, S, hd, 32, dtype, DEV)
        ops.cache_write(other, k[b:b + 1], v[b:b + 1], at(p[b]), cos=cos, sin=sin, q=k[b:b + 1], q_out=again)
        codes, scale, zero = defined(again[0], 32)
        assert torch.equal(codes_of(cache.k)[b, :, p[b]:p[b] + T], codes.transpose(0, 1))
        codes, scale, zero = defined(v[b], 32)
        assert torch.equal(codes_of(cache.v)[b, :, p[b]:p[b] + T], codes.transpose(0, 1))
        assert torch.equal(cache.v_scales[b, :, p[b]:p[b] + T, :, 0].cpu().float(), scale.transpose(0, 1))
    assert same(k_out.double().cpu()[1], rounded(values(cache, "k")[1, :, p[1]:p[1] + T].transpose(0, 1), dtype))


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_ranges_at_the_edges(dtype, group):
    """Equal values, the type's smallest and largest, zeros of both signs, ties between codes, NaN and infinities."""
    hd, top, tiny = 128, torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x = torch.zeros(12, hd)
    x[0], x[1], x[2, ::2] = 3.25, -top, -0.0
    x[3] = torch.arange(hd) % 3 * tiny                      # a scale that rounds to zero or to the smallest number
    x[4] = torch.arange(hd) % 16 * tiny
    x[5], x[5, 5], x[5, 70] = 1.0, top if dtype is F16 else 1e38, -top if dtype is F16 else -1e38
    x[6] = torch.arange(hd) % 31 * 0.5                      # halves of a step of one: ties
    x[7], x[7, 40] = 2.0, float("nan")
    x[8], x[8, 3], x[8, 100] = 1.0, float("inf"), -float("inf")
    x[9], x[9, 0], x[9, 1] = 1.0, float("inf"), -float("inf")
    x[10] = torch.randn(hd, generator=torch.Generator().manual_seed(3)) * 1e-6
    x[11, 0::2], x[11, 1::2] = (top, -top)                  # bf16: the range passes fp32
    x = x.to(dtype).to(DEV)[None, :, None]
    cache = ops.QuantCache.empty(1, 1, 12, hd, group, dtype, DEV)
    out = torch.empty_like(x)
    ops.cache_write(cache, x, x, at(0), k_out=out, v_out=torch.empty_like(x))
    codes, scale, zero = defined(x, group)
    bad = torch.isnan(scale).repeat_interleave(group, -1)
    for packed, constants in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        assert torch.equal(codes_of(packed)[0, 0].masked_fill(bad[0, :, 0], 0), codes[0, :, 0])
        assert same(constants[0, 0, ..., 0].cpu().float(), scale[0, :, 0]) and same(constants[0, 0, ..., 1].cpu().float(), zero[0, :, 0])
    assert torch.equal(torch.isnan(out).cpu(), bad) and bad[0, 7].sum() == group and bad.sum() == group * 4 + (hd if dtype is BF16 else 0)
    assert torch.equal(out.double().cpu()[~bad], rounded(values(cache, "k")[:, 0, :, None], dtype)[~bad]) and bool(torch.isfinite(out.cpu()[~bad]).all())
    if dtype is F16:
        assert torch.equal(out[0, 11], x[0, 11])            # -top + 15 scales is above top: held there
    assert torch.equal(out[0, :3].cpu(), x[0, :3].cpu())     # one value, or two zeros


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_near_the_largest_number(dtype, group):
    """A scale that was rounded up puts the last code above the type's largest number; what comes out is that number."""
    top = torch.finfo(dtype).max
    x = torch.zeros(40, 128)
    for i in range(40):
        x[i] = top * torch.linspace(0.02 * i, 1, 128)
    x = x.to(dtype).to(DEV)[None, :, None]
    cache, out = ops.QuantCache.empty(1, 1, 40, 128, group, dtype, DEV), torch.empty_like(x)
    ops.cache_write(cache, x, -x, at(0), k_out=out, v_out=torch.empty_like(x))
    assert bool(torch.isfinite(out).all()) and torch.equal(out[0, :, 0].double().cpu(), rounded(values(cache, "k")[0, 0], dtype))
    assert float((values(cache, "k") > top).double().sum()) > 0                # (there are such)
    assert torch.equal(codes_of(cache.k)[0, 0], defined(x, group)[0][0, :, 0]) and torch.equal(codes_of(cache.v)[0, 0], defined(-x, group)[0][0, :, 0])
    assert all(bool(torch.isfinite(t).all()) for t in ops.cache_read(cache))


def test_padding_and_positions_outside():
    B, T, kv, hd, S = 6, 4, 2, 64, 10
    k, v = rows(B, T, kv, hd, dtype=F16), rows(B, T, kv, hd, dtype=F16, seed=1)
    angle = torch.ones(8, hd // 2, dtype=F16, device=DEV)
    big = 1 << 62
    pos, counts = [0, 8, -2, big, -big, 5], [2, 4, 4, 4, 9, 0]
    for tables in (False, True):
        cache = ops.QuantCache.empty(B, kv, S, hd, dtype=F16, device=DEV)
        for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
            t.fill_(7)
        k_out, v_out, q_out = (torch.full_like(k, 5) for _ in range(3))
        extra = dict(cos=angle, sin=angle, q=k, q_out=q_out) if tables else {}
        ops.cache_write(cache, k, v, at(*pos), counts=at(*counts), k_out=k_out, v_out=v_out, **extra)
        end = 8 if tables else S
        for b in range(B):
            written = [pos[b] + t for t in range(T) if t < counts[b] and 0 <= pos[b] + t < end]
            for j in range(S):
                left = bool((cache.k[b, :, j] == 7).all() and (cache.v[b, :, j] == 7).all() and (cache.k_scales[b, :, j] == 7).all())
                assert left == (j not in written)
            for t in range(T):
                for o in (k_out, v_out) + ((q_out,) if tables else ()):
                    assert bool((o[b, t] == 5).all()) == (pos[b] + t not in written or t >= counts[b])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_reading_back_some_rows_of_views(hd, group, dtype):
    B, kv, S = 3, 2, 37
    whole = ops.QuantCache.empty(B + 1, kv + 1, S + 5, hd, group, dtype, DEV)
    cut = ops.QuantCache(*(t[1:, :kv, 2:S + 2] for t in (whole.k, whole.v, whole.k_scales, whole.v_scales)))
    x, y = rows(B, S, kv, hd, dtype=dtype), rows(B, S, kv, hd, dtype=dtype, seed=2)
    ops.cache_write(cut, x, y, at(0))
    assert not whole.k[0].any() and not whole.k[:, kv].any() and not whole.v[:, :, :2].any() and not whole.k_scales[:, :, S + 2:].any()
    lengths = [0, 17, 99]
    outs = [torch.full((B, S, kv, hd + 8), 9.0, dtype=dtype, device=DEV)[..., :hd].transpose(1, 2) for _ in range(2)]
    k, v = ops.cache_read(cut, lengths=at(*lengths), k_out=outs[0], v_out=outs[1])
    assert k.data_ptr() == outs[0].data_ptr() and v.data_ptr() == outs[1].data_ptr()
    for got, name in ((k, "k"), (v, "v")):
        want = rounded(values(cut, name), dtype)
        for b, n in enumerate(lengths):
            assert torch.equal(got[b, :, :n].double().cpu(), want[b, :, :n]) and bool((got[b, :, n:] == 9).all())


def test_written_in_place_on_another_stream_and_from_a_graph():
    B, T, kv, hd, S = 2, 1, 4, 128, 6
    cache = ops.QuantCache.empty(B, kv, S, hd, device=DEV)
    pos, k, v = at(0), rows(B, T, kv, hd, dtype=F16), rows(B, T, kv, hd, dtype=F16, seed=1)
    before = cache.k._version, cache.v_scales._version
    s = torch.cuda.Stream(DEV)
    s.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(s):
        ops.cache_write(cache, k, v, pos)
    torch.cuda.current_stream(DEV).wait_stream(s)
    assert cache.k._version > before[0] and cache.v_scales._version > before[1]
    assert torch.equal(codes_of(cache.k)[:, :, 0], defined(k, 32)[0][:, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_write(cache, k, v, pos)
        back = ops.cache_read(cache)
        pos.add_(1)
    for i in range(2, 5):
        k.copy_(rows(B, T, kv, hd, dtype=F16, seed=10 + i))
        pos.fill_(i)
        graph.replay()
        assert torch.equal(codes_of(cache.k)[:, :, i], defined(k, 32)[0][:, 0]) and int(pos) == i + 1
        assert torch.equal(back[0].double().cpu(), rounded(values(cache, "k"), F16))


def test_far_rows_of_a_large_cache():
    """Offsets that pass 32 bits, in bytes and in elements."""
    kv, hd, S = 1, 128, (1 << 25) + 5                       # 2.1 GB of codes; a row of values out of cache_read would be 8.6 GB
    cache = ops.QuantCache.empty(1, 3 * kv, S, hd, 64, device=DEV)
    k, v = rows(1, 3, 3, hd, dtype=F16), rows(1, 3, 3, hd, dtype=F16, seed=1)
    ops.cache_write(cache, k, v, at(S - 3))
    codes, scale, zero = defined(k, 64)
    assert torch.equal(codes_of(cache.k[:, :, S - 3:]), codes.transpose(1, 2))
    assert torch.equal(cache.k_scales[0, :, S - 3:, :, 1].cpu().float(), zero[0].transpose(0, 1))
    assert not cache.k[:, :, :S - 3].any() and not cache.v[:, :, :S - 3].any()


def test_refusals():
    B, T, kv, hd, S = 2, 3, 2, 64, 10
    cache = ops.QuantCache.empty(B, kv, S, hd, device=DEV)
    k, v, pos = rows(B, T, kv, hd, dtype=F16), rows(B, T, kv, hd, dtype=F16), at(0)
    angle = torch.ones(S, hd // 2, dtype=F16, device=DEV)

    def parts(**change):
        return ops.QuantCache(**{**{n: getattr(cache, n) for n in ("k", "v", "k_scales", "v_scales")}, **change})

    for error, call in [
        (TypeError, lambda: ops.cache_write(cache, None, v, pos)),
        (TypeError, lambda: ops.cache_write(cache, k.float(), v, pos)),
        (TypeError, lambda: ops.cache_write(cache, k, v.bfloat16(), pos)),
        (TypeError, lambda: ops.cache_write(cache, k, v, at(0).int())),
        (TypeError, lambda: ops.cache_write(parts(k=cache.k.to(torch.int8)), k, v, pos)),
        (TypeError, lambda: ops.cache_write(parts(v_scales=cache.v_scales.bfloat16()), k, v, pos)),
        (TypeError, lambda: ops.cache_write(parts(k_scales=cache.k_scales.float()), k, v, pos)),
        (RuntimeError, lambda: ops.cache_write(cache, k.cpu(), v, pos)),
        (RuntimeError, lambda: ops.cache_write(parts(v=cache.v.cpu()), k, v, pos)),
        (RuntimeError, lambda: ops.cache_write(cache, k.clone().requires_grad_(), v, pos)),
        (ValueError, lambda: ops.cache_write(cache, k[:1], v, pos)),
        (ValueError, lambda: ops.cache_write(cache, k, v[:, :2], pos)),
        (ValueError, lambda: ops.cache_write(cache, k[..., :32], v[..., :32], pos)),
        (ValueError, lambda: ops.cache_write(cache, k, v, at(0, 1, 2))),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, counts=at(1))),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, cos=angle)),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, cos=angle, sin=angle[:4])),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, cos=angle[:, ::2], sin=angle[:, ::2])),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, q=k, q_out=torch.empty_like(k))),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, cos=angle, sin=angle, q=k)),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, cos=angle, sin=angle, q=k, q_out=k)),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, k_out=k, v_out=torch.empty_like(v))),
        (ValueError, lambda: ops.cache_write(cache, k, v, pos, k_out=torch.empty_like(k))),
        (ValueError, lambda: ops.cache_write(parts(v=cache.k), k, v, pos)),
        (ValueError, lambda: ops.cache_write(parts(k=cache.k[:1].expand(B, -1, -1, -1)), k, v, pos)),
        (ValueError, lambda: ops.cache_write(parts(k=cache.k[:, :1]), k, v, pos)),
        (ValueError, lambda: ops.cache_write(parts(k_scales=cache.k_scales[..., :1]), k, v, pos)),
        (ValueError, lambda: ops.cache_write(cache, torch.zeros(B * T * kv * hd + 1, dtype=F16, device=DEV)[1:].view(B, T, kv, hd), v, pos)),
        (ValueError, lambda: ops.cache_read(cache, lengths=at(1, 1))),
        (ValueError, lambda: ops.cache_read(cache, k_out=torch.empty(B, kv, S, hd, dtype=F16, device=DEV))),
        (ValueError, lambda: ops.cache_read(cache, lengths=at(1), k_out=torch.empty(B, kv, S, hd, dtype=F16, device=DEV), v_out=torch.empty(B, kv, S, hd, dtype=F16, device=DEV))),
        (ValueError, lambda: ops.cache_read(cache, k_out=torch.empty(B, kv, S - 1, hd, dtype=F16, device=DEV), v_out=torch.empty(B, kv, S, hd, dtype=F16, device=DEV))),
        (TypeError, lambda: ops.cache_read(cache, k_out=torch.empty(B, kv, S, hd, device=DEV), v_out=torch.empty(B, kv, S, hd, device=DEV))),
    ]:
        with pytest.raises(error):
            call()
    assert not cache.k.any() and not cache.v_scales.any()
