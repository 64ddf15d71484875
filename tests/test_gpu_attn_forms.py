"""The forms of b200gptq_attn that only larger calls take, each with padding, junk, strides, streams and graphs, against 64 bits:

* two tiles of rows per CTA (more tiles of 128 rows than the device has SMs): both product warps share each unit of keys, of which either tile may see a part,
  the second tile may be empty, rows are stored straight from the tile;
* a prefix that goes before in parts (scratch is asked for): the prefix launch, each sequence's own rows beside it, a third launch that adds up.

The bound per output element is that of test_gpu_attn.py, whose terms stand there."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import _lib, ops
    DEV = torch.device("cuda:0")
    SMS = torch.cuda.get_device_properties(0).multi_processor_count
else:
    SMS = 148

F16, BF16 = torch.float16, torch.bfloat16


def enough(T, heads, kv):
    """Sequences for more tiles of 128 rows than SMs."""
    return SMS // (-(-T * (heads // kv) // 128) * kv) + 1


def two(T, heads, kv, hd, **more):
    return dict(B=enough(T, heads, kv), T=T, heads=heads, kv=kv, hd=hd, parts=False, **more)


def apart(B, T, heads, kv, hd, P):
    return dict(B=B, T=T, heads=heads, kv=kv, hd=hd, P=P, parts=True)


FORMS = {
    "two-window-odd": two(257, 8, 8, 64, W=40, S=3),               # three tiles: the last CTA's second one is empty
    "two-window-groups": two(129, 6, 2, 128, W=70, S=5),
    "two-window-sinks-meet": two(300, 4, 4, 128, W=130, S=140),
    "two-window-itself": two(200, 14, 2, 64, W=1, S=0),
    "two-window-all": two(400, 4, 4, 128, W=1000, S=0),
    "two-prefix": two(140, 4, 4, 128, P=100),
    "two-prefix-groups": two(131, 16, 2, 64, P=333),
    "parts-tiles": apart(70, 1, 4, 4, 64, 1500),
    "parts-tiles-groups": apart(50, 2, 8, 2, 128, 1000),
    "parts-rows": apart(12, 1, 1, 1, 128, 6100),
    "parts-rows-runs": apart(5, 3, 4, 2, 128, 8200),
}
every_form = pytest.mark.parametrize("name", FORMS)


class Call:
    """The tensors of a call and the call."""

    def __init__(self, name, dtype=F16, seed=0):
        f = FORMS[name]
        self.B, self.T, self.heads, self.kv, self.hd = (f[n] for n in ("B", "T", "heads", "kv", "hd"))
        self.W, self.S, self.P, self.room = f.get("W"), f.get("S", 0), f.get("P"), self.T + 60
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=dtype)
        self.q = 1.5 * r(self.B, self.T, self.heads, self.hd) + 0.5
        self.k, self.v = r(self.B, self.kv, self.room, self.hd), r(self.B, self.kv, self.room, self.hd)
        self.k[:, :, :3] += 0.5
        self.kp = self.vp = None
        if self.P:
            self.kp, self.vp = r(self.kv, self.P, self.hd), r(self.kv, self.P, self.hd)
        # positions of token 0; one sequence begins before its cache, one of a window ends behind it
        self.at = [7 * b % 59 for b in range(self.B)]
        self.at[1 % self.B] = -1 if self.P else -5
        if self.W:
            self.at[2 % self.B] = self.room - self.T // 2
        self.pos = torch.tensor(self.at, device=DEV)
        a = _lib.AttnArgs(dtype=0 if dtype == F16 else 1, batch=self.B, tokens=self.T, heads=self.heads, kv_heads=self.kv, hd=self.hd, max_seq=self.room,
                          window=self.W or 0, sinks=self.S, prefix=self.P or 0, scale=1.0)
        for n, t in (("k_stride", self.k), ("v_stride", self.v)):
            setattr(a, n, (ctypes.c_int64 * 3)(*t.stride()[:3]))
        for n, t in (("k_prefix_stride", self.kp), ("v_prefix_stride", self.vp)):
            setattr(a, n, (ctypes.c_int64 * 2)(*(t.stride()[:2] if t is not None else (0, 0))))
        scratch = _lib.lib.b200gptq_attn_workspace_bytes(ctypes.byref(a))
        tiles = -(-self.T * (self.heads // self.kv) // 128) * self.kv * self.B
        if f["parts"] is not None:
            assert scratch > 0 if f["parts"] else scratch == 0 and tiles > SMS and self.T * self.heads // self.kv >= 64

    def __call__(self, pos=None, **more):
        t = {n: more.pop(n, getattr(self, n)) for n in ("q", "k", "v", "kp", "vp")}
        pos = self.pos if pos is None else pos
        if self.P:
            return ops.attn_prefix(t["q"], t["kp"], t["vp"], t["k"], t["v"], pos, **more)
        return ops.attn_window(t["q"], t["k"], t["v"], pos, self.W, self.S, **more)

    def sees(self, b):
        """[T, room]: what the tokens of a sequence see of its own cache."""
        p = self.at[b] + torch.arange(self.T, device=DEV)[:, None]
        j = torch.arange(self.room, device=DEV)[None]
        seen = j <= p
        return seen & ((j > p - self.W) | (j < self.S)) if self.W else seen

    def reference(self):
        """(output, bound) in 64 bits."""
        G, u = self.heads // self.kv, torch.finfo(self.q.dtype).eps / 2
        out, bound = (torch.zeros(self.q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
        scale = self.hd ** -0.5
        for b in range(self.B):
            seen = self.sees(b)
            if self.P:
                seen = torch.cat([torch.ones(self.T, self.P, dtype=torch.bool, device=DEV), seen], 1)
            hidden = ~seen.repeat_interleave(G, 0)
            n = seen.sum(1).repeat_interleave(G)[:, None]
            for h in range(self.kv):
                K, V = self.k[b, h].double(), self.v[b, h].double()
                if self.P:
                    K, V = torch.cat([self.kp[h].double(), K]), torch.cat([self.vp[h].double(), V])
                Q = self.q[b, :, h * G:h * G + G].double().reshape(-1, self.hd)
                w = torch.softmax((Q @ K.t() * scale).masked_fill(hidden, -math.inf), 1).masked_fill(n == 0, 0)
                o, A = w @ V, w @ V.abs()
                d = self.hd * 2.0 ** -22 * (Q.abs() @ K.abs().t()).masked_fill(hidden, 0).amax(1, keepdim=True) * scale
                err = u * o.abs() + (u + 2 * d + n * 2.0 ** -22 + 2.0 ** -18) * A
                if u == 2.0 ** -11:
                    err = err + n * 2.0 ** -25 * V.abs().max()
                out[b, :, h * G:h * G + G], bound[b, :, h * G:h * G + G] = (x.reshape(self.T, G, self.hd) for x in (o, err))
        return out, bound


def check(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound.clamp(min=1e-30)).max()):.3g} times the bound"


@pytest.mark.parametrize("dtype", [F16, BF16])
@every_form
def test_against_64_bits(name, dtype):
    c = Call(name, dtype)
    got = c()
    check(got, *c.reference())
    assert torch.equal(got, c())
    ops.check_status(DEV)


@every_form
def test_padding(name):
    """Sequences without a token, the last among them, with one, with half and with all of them."""
    c = Call(name)
    want, bound = c.reference()
    counts = [(c.T, 0, 1, (c.T + 1) // 2)[b % 4] for b in range(c.B)]
    counts[-1] = 0
    out = torch.full_like(c.q, 7.0)
    assert c(counts=torch.tensor(counts, device=DEV), out=out) is out
    for b, n in enumerate(counts):
        check(out[b, :n], want[b, :n], bound[b, :n])
        assert bool((out[b, n:] == 7).all())


@pytest.mark.parametrize("junk", [math.nan, math.inf])
@every_form
def test_rows_that_no_token_sees(name, junk):
    c = Call(name)
    want, bound = c.reference()
    for b in range(c.B):
        never = ~c.sees(b).any(0)
        c.k[b, :, never], c.v[b, :, never] = junk, junk
    check(c(), want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@every_form
def test_values_that_some_tokens_see(name, dtype):
    """An infinity in dim 3 of one row and a NaN in dim 5 of another: the tokens that see them have them there, all else is as without."""
    c = Call(name, dtype)
    want, bound = c.reference()
    rows = [min(max(0, p + c.T // 2), c.room - 1) for p in c.at]
    others = [min(max(0, p + c.T // 3 + 1), c.room - 1) for p in c.at]
    for b in range(c.B):
        c.v[b, :, rows[b], 3], c.v[b, :, others[b], 5] = math.inf, math.nan
    got = c()
    some = False
    for b in range(c.B):
        seen = c.sees(b)
        inf, nan = seen[:, rows[b]], seen[:, others[b]]
        some = some or bool(inf.any()) and not bool(inf.all())
        assert bool((got[b, inf][..., 3] == math.inf).all()) and bool(got[b, nan][..., 5].isnan().all())
        check(got[b, ~inf][..., 3], want[b, ~inf][..., 3], bound[b, ~inf][..., 3])
        check(got[b, ~nan][..., 5], want[b, ~nan][..., 5], bound[b, ~nan][..., 5])
    assert some or c.T == 1
    rest = [d for d in range(c.hd) if d not in (3, 5)]
    check(got[..., rest], want[..., rest], bound[..., rest])


@every_form
def test_keys_and_queries_that_are_nan(name):
    """A NaN in a key makes the rows that see it NaN, one in a query its own."""
    c = Call(name)
    want, bound = c.reference()
    b, t = c.B - 1, c.T // 2
    j = max(0, c.at[b] + t)
    c.k[b, :, j, 2] = math.nan
    c.q[0, 0, 0, 1] = math.nan
    got = c()
    bad = torch.zeros(got.shape[:3], dtype=torch.bool, device=DEV)
    bad[b, c.sees(b)[:, j]] = True
    bad[0, 0, 0] |= bool(c.P) or bool(c.sees(0)[0].any())
    assert bool(got[bad].isnan().all())
    check(got[~bad], want[~bad], bound[~bad])


@pytest.mark.parametrize("name", [n for n in FORMS if "P" in FORMS[n]])
def test_a_nan_in_a_value_of_the_prefix_is_everywhere(name):
    c = Call(name)
    clean = c()
    c.vp[:, c.P // 2, 9] = math.nan
    got = c()
    assert bool(got[..., 9].isnan().all())
    got[..., 9] = clean[..., 9]
    assert torch.equal(got, clean)


@every_form
def test_strides(name):
    """q out of a packed q|k|v, caches laid out [batch, position, head, dim] with room, the prefix [position, head, dim], out with room between its rows."""
    c = Call(name)
    want = c()
    packed = torch.zeros(c.B, c.T, 3, c.heads, c.hd, device=DEV, dtype=F16)
    packed[:, :, 1] = c.q
    k = torch.full((c.B, c.room + 3, c.kv + 1, 2 * c.hd), math.nan, device=DEV, dtype=F16)[:, 2:2 + c.room, 1:, c.hd:]
    k.copy_(c.k.permute(0, 2, 1, 3))
    v = c.v.transpose(0, 1).contiguous().transpose(0, 1)
    more = dict(q=packed[:, :, 1], k=k.permute(0, 2, 1, 3), v=v)
    if c.P:
        more.update(kp=c.kp.transpose(0, 1).contiguous().transpose(0, 1), vp=torch.cat([c.vp, c.vp], 2)[..., c.hd:])
    room = torch.zeros(c.B, c.T, c.heads, 2 * c.hd, device=DEV, dtype=F16)
    c(out=room[..., c.hd:], **more)
    assert torch.equal(room[..., c.hd:], want) and bool((room[..., :c.hd] == 0).all())


@every_form
def test_caches_that_repeat(name):
    """Every sequence and head has the same keys (stride 0): what no tensor map can say."""
    c = Call(name)
    c.k, c.v = c.k[:1, :1].expand(c.B, c.kv, -1, -1), c.v[:1].expand(c.B, -1, -1, -1)
    if c.P:
        c.kp, c.vp = c.kp[:1].expand(c.kv, -1, -1), c.vp[:1].expand(c.kv, -1, -1)
    check(c(), *c.reference())


@every_form
def test_a_chain_of_calls(name):
    """q, keys and positions written by the operation in front of the call and overwritten by the one behind it, calls of other forms and sizes in between, scratch
    used again by each, and never a synchronisation."""
    c, o = Call(name), Call("parts-tiles" if name != "parts-tiles" else "parts-rows-runs", seed=1)
    steps = [tuple(torch.randn_like(t) for t in (c.q, c.k)) + (c.pos + i % 3,) for i in range(6)]
    torch.cuda.synchronize()
    got, other = [], []
    for q, k, p in steps:
        c.q.copy_(q)
        c.k.copy_(k)
        c.pos.copy_(p)
        got.append(c())
        other.append(o())
        got.append(c())
        c.q.fill_(math.nan)
        c.k.fill_(math.nan)
        c.pos.fill_(1 << 40)
    want = []
    for q, k, p in steps:
        torch.cuda.synchronize()
        want.append(c(q=q, k=k, pos=p))
        torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert torch.equal(got[2 * i], w) and torch.equal(got[2 * i + 1], w)
    assert all(torch.equal(other[0], x) for x in other)


@every_form
def test_streams_and_graphs(name):
    """On a side stream beside the same call on the usual one; from two graphs that are replayed side by side, with positions that move on."""
    c = Call(name)
    want = [c(pos=c.pos + i) for i in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pairs = []
    for i in range(3):
        p = c.pos + i
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x = c(pos=p)
        pairs.append((x, c(pos=p), p))
    torch.cuda.synchronize()
    for w, (x, y, _) in zip(want, pairs):
        assert torch.equal(x, w) and torch.equal(y, w)
    graphs = []
    for _ in range(2):
        p, g = c.pos.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x = c(pos=p)
            y = c(pos=p)
            p.add_(1)
        graphs.append((g, x, y, p, torch.cuda.Stream()))
    for w in want:
        for g, _, _, _, s in graphs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, x, y, _, _ in graphs:
            assert torch.equal(x, w) and torch.equal(y, w)
    ops.check_status(DEV)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("at,W", [(-1000, 14), (-130, 14), (5000, 14)])
def test_tiles_that_see_nothing(at, W, hd):
    """Whole tiles of rows before position 0, or so far behind the cache that the window has left it: zeros.  (The queries are more than the L2 holds, so
    that the warps of a tile get theirs at different times.)"""
    B, T, heads = 400, 257, 8
    q = torch.full((B, T, heads, hd), 3.0, device=DEV, dtype=F16)
    k = torch.ones(B, heads, 1, hd, device=DEV, dtype=F16)
    p = at + torch.arange(T, device=DEV)
    empty = (p < 0) | (p >= W)
    for _ in range(6):
        got = ops.attn_window(q, k, k, torch.tensor([at], device=DEV), W, 0)
        assert bool((got[:, empty] == 0).all()) and bool((got[:, ~empty] == 1).all())


SMALL = {"one-token": dict(B=40, T=1, heads=2, kv=2), "few-tokens": dict(B=40, T=5, heads=4, kv=2), "twenty-rows": dict(B=3, T=5, heads=8, kv=2), "one-tile": dict(B=3, T=70, heads=2, kv=1)}


@pytest.mark.parametrize("name", [*FORMS, *SMALL])
def test_values_at_the_end_of_fp16(name, monkeypatch):
    """All values are the largest fp16 number or its negative, dim by dim (as where activations are held to the type's range), and a mean of them is that number.
    Weights of 1 and, fifteen times as many, of 0.5 (1 + 1.2 2^-11), which fp16 holds as 0.5 (1 + 2^-10): with their sum not rounded the mean is 3.4 10^-4 more,
    where fp16 has infinity.  The bound: half a step for the weights, half a step for the result."""
    monkeypatch.setitem(FORMS, "here", dict(SMALL.get(name, {}), hd=128, W=60, S=2, parts=None))
    c = Call(name if name in FORMS else "here")
    top = torch.finfo(F16).max
    sign = torch.where(torch.arange(c.hd, device=DEV) % 3 > 0, top, -top).to(F16)
    c.q.zero_()
    c.q[..., 0] = 1
    for k, v in ((c.k, c.v), (c.kp, c.vp)):
        if k is not None:
            k.zero_()
            k[..., 0] = -1
            k[..., ::16, 0] = 0
            v.copy_(sign.expand_as(v))
    got = c(scale=(1 - math.log2(1 + 1.2 * 2.0 ** -11)) * math.log(2))
    some = torch.stack([c.sees(b).any(1) for b in range(c.B)]) | bool(c.P)
    assert bool((got[~some] == 0).all()) and bool(torch.isfinite(got).all())
    assert bool(((got[some].double() - sign.double()).abs() <= 2 * 2.0 ** -11 * top).all())


@every_form
def test_a_negative_scale_is_that_of_the_negated_queries(name):
    """Bit for bit, as a sign changes no rounding; and a scale of zero is that of queries of zero."""
    c = Call(name)
    assert torch.equal(c(scale=-0.1), c(q=-c.q, scale=0.1))
    assert torch.equal(c(scale=0.0), c(q=torch.zeros_like(c.q), scale=0.1))


@every_form
def test_numbers_far_out_of_range(name):
    """Positions and counts at the ends of 64 bits are held to what there is."""
    c = Call(name)
    ends = torch.tensor([(1 << 63) - 1, -(1 << 63)], device=DEV)
    out = torch.full_like(c.q, 7.0)
    c(counts=ends[1].expand(c.B).contiguous(), out=out)
    assert bool((out == 7).all())
    want = c()
    assert torch.equal(c(counts=ends[0].expand(c.B).contiguous(), out=out), want)
    c.at = [-(1 << 40)] * c.B
    check(c(pos=ends[1:]), *c.reference())
    c.at = [1 << 40] * c.B
    check(c(pos=ends[:1]), *c.reference())


@pytest.mark.parametrize("W,S", [(1 << 29, 0), (1 << 29, 1 << 29), (1, 1 << 29), (30, 61)])
@pytest.mark.parametrize("name", [*(n for n in FORMS if "P" not in FORMS[n]), *SMALL])
def test_the_largest_windows_and_sinks(name, W, S, monkeypatch):
    monkeypatch.setitem(FORMS, "here", dict(SMALL.get(name, {}), hd=64, W=60, S=2, parts=None))
    c = Call(name if name in FORMS else "here")
    c.W, c.S = W, S
    check(c(), *c.reference())
