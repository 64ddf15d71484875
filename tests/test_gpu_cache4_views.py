"""Caches in 4 bits whose parts alternate in one allocation, and outputs that alternate with inputs: no byte is shared, and each is taken; what does share one is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")

F16 = torch.float16
B, KV, S, HD, T = 3, 2, 40, 64, 5


def at(*pos):
    return torch.tensor(pos, device=DEV)


def interleaved(where):
    """A cache made of views of one allocation per kind: keys and values side by side in dimension `where` of [batch, kv_heads, max_seq, ..]."""
    def pair(*tail, dtype):
        shape = [B, KV, S, *tail]
        shape.insert(where, 2)
        whole = torch.zeros(shape, dtype=dtype, device=DEV)
        return whole.select(where, 0), whole.select(where, 1)
    (k, v), (ks, vs) = pair(HD // 2, dtype=torch.uint8), pair(HD // 32, 2, dtype=F16)
    return ops.QuantCache(k, v, ks, vs)


def in_rows():
    """Codes and constants of keys, then of values, in each row of one allocation of bytes: 32 + 8 (+ 8 to a multiple of 16), twice."""
    rows = torch.zeros(B, KV, S, 2, 48, dtype=torch.uint8, device=DEV)
    constants = rows.view(F16)[..., 16:20].unflatten(-1, (2, 2))
    return ops.QuantCache(rows[..., 0, :32], rows[..., 1, :32], constants[..., 0, :, :], constants[..., 1, :, :])


@pytest.mark.parametrize("make", [lambda: interleaved(0), lambda: interleaved(1), lambda: interleaved(2), lambda: interleaved(3), in_rows])
def test_parts_of_one_allocation(make):
    g = torch.Generator(device=DEV).manual_seed(0)
    qkv = torch.randn(B, T, 8, HD, generator=g, device=DEV).half()
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    plain, cache = ops.QuantCache.empty(B, KV, S, HD), make()
    angle = torch.rand(S, HD // 2, generator=g, device=DEV).half()
    pos = at(0, 7, S - T)
    outs = []
    for c in (plain, cache):
        together = torch.zeros(B, T, 2, KV, HD, dtype=F16, device=DEV)            # what goes in and comes out, each in one allocation
        both = torch.zeros(B, T, 4, 2, HD, dtype=F16, device=DEV)
        both[..., 0, :] = q
        rotated = ops.cache_write(c, k, v, pos, cos=angle, sin=angle, q=both[..., 0, :], q_out=both[..., 1, :], k_out=together[:, :, 0], v_out=together[:, :, 1])
        read = torch.zeros(B, KV, S, 2, HD, dtype=F16, device=DEV)
        ops.cache_read(c, k_out=read[..., 0, :], v_out=read[..., 1, :])
        attended = torch.zeros(B, T, 4, 2, HD, dtype=F16, device=DEV)
        attended[..., 0, :] = rotated
        ops.attn_cache(attended[..., 0, :], c, pos, out=attended[..., 1, :])
        outs.append([both, together, read, attended, c.k.contiguous(), c.v.contiguous(), c.k_scales.contiguous(), c.v_scales.contiguous()])
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    assert torch.equal(outs[0][0][..., 0, :], q) and outs[0][2].any() and outs[0][3][..., 1, :].any()


def test_shared_bytes_are_refused():
    k, v = (torch.zeros(B, T, KV, HD, dtype=F16, device=DEV) for _ in range(2))
    pos = at(0)
    whole = torch.zeros(B, KV, S, 2 * HD, dtype=torch.uint8, device=DEV)
    constants = torch.zeros(B, KV, S + 1, 2, 2, 2, dtype=F16, device=DEV)
    good = ops.QuantCache(whole[..., :32], whole[..., 64:96], constants[:, :, :S, 0], constants[:, :, :S, 1])
    ops.cache_write(good, k, v, pos)
    for bad in (ops.QuantCache(whole[..., :32], whole[..., 16:48], good.k_scales, good.v_scales),
                ops.QuantCache(whole[..., :32], whole[..., :32], good.k_scales, good.v_scales),
                ops.QuantCache(good.k, good.v, good.k_scales, constants[:, :, 1:, 0]),                # (a row further on)
                ops.QuantCache(good.k, good.v, good.k_scales, whole.view(F16)[..., 4:8].unflatten(-1, (2, 2)))):          # (in the keys' codes)
        with pytest.raises(ValueError, match="overlap"):
            ops.cache_write(bad, k, v, pos)
    wide = torch.zeros(B, T, 3 * KV, HD, dtype=F16, device=DEV)
    with pytest.raises(ValueError, match="overlap"):          # (a head in common)
        ops.cache_write(good, k, v, pos, k_out=wide[:, :, :KV], v_out=wide[:, :, KV - 1:2 * KV - 1])
    with pytest.raises(ValueError, match="overlap"):          # (the heads that follow, of the same token, but one token's fewer)
        ops.cache_write(good, wide[:, :, :KV], v, pos, k_out=wide[:, :, 1:1 + KV], v_out=wide[:, :, 2 * KV:])
    ops.cache_write(good, wide[:, :, :KV], v, pos, k_out=wide[:, :, KV:2 * KV], v_out=wide[:, :, 2 * KV:])
    q = torch.zeros(B, T, 2 * KV, HD, dtype=F16, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.attn_cache(q[:, :, :KV], good, pos, out=q[:, :, 1:1 + KV])
    with pytest.raises(ValueError, match="overlap"):          # (by tokens: each lies in the other's span, one token further on)
        line = torch.zeros(B, T + 1, KV, HD, dtype=F16, device=DEV)
        ops.attn_cache(line[:, 1:], good, pos, out=line[:, :T])
    read = torch.zeros(B, KV, S, 2 * HD, dtype=F16, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_read(good, k_out=read[..., :HD], v_out=read[..., HD // 2:HD // 2 + HD])
