"""ops.adjust_logits against 64 bits, row by row from the definition.

The bound, per value: half a step of the type for the result (fp32: 2^-24), and in fp32 one rounding each (2^-24 of the value at hand, all of which are at most
M = |x r| + |x / r| + frequency n + presence + |bias| + |x|) for the product or quotient, frequency * n, the two subtractions and the sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def make(R, V, L, N, mask, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    s = {"logits": (4 * torch.randn(R, V, generator=g)).to(dtype)}
    s["history"] = (V * torch.rand(R, L, generator=g) ** 3).long().clamp(max=V - 1)
    if L > 3:
        s["history"][:, 1::7] = -1            # padding, and tokens of no vocabulary
        s["history"][:, 2::11] = V
        s["history"][:, 3::13] = 1 << 40
    s["lengths"] = torch.randint(0, L + 1, (R,), generator=g)
    s["lengths"][0] = L
    s["prompt_lens"] = s["lengths"] // 2
    s["repetition"] = 0.8 + torch.rand(R, generator=g)
    s["frequency"], s["presence"] = torch.randn(R, generator=g), torch.randn(R, generator=g)
    if N:
        s["bias_tokens"] = torch.randint(-1, V + 1, (R, N), generator=g)
        s["bias_tokens"][:, N // 2:] = s["bias_tokens"][:, :N - N // 2]          # the same tokens again
        s["bias_values"] = 3 * torch.randn(R, N, generator=g)
    if mask:
        s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (R, -(-V // 32)), generator=g).int()
        s["mask"][-1] = 0                     # a row that leaves nothing
        if R > 2:
            s["mask"][1] = -1
    return s


def reference(s):
    x, (R, V) = s["logits"].double(), s["logits"].shape
    M = x.abs()
    for b in range(R):
        if "history" in s:
            n, m = (int(s[k][b]) if k in s else 0 for k in ("lengths", "prompt_lens"))
            n = max(0, min(n, s["history"].shape[1]))
            text = s["history"][b, :n].tolist()
            r, f, p = (float(s[k][b]) if k in s else d for k, d in (("repetition", 1), ("frequency", 0), ("presence", 0)))
            made = {}
            for t in text[max(0, m):]:
                made[t] = made.get(t, 0) + 1
            for t in set(text):
                if 0 <= t < V:
                    M[b, t] += abs(float(x[b, t]) / r) + abs(float(x[b, t]) * r)
                    x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
                    if t in made:
                        x[b, t] -= f * made[t] + p
                        M[b, t] += abs(f * made[t]) + abs(p)
        if "bias_tokens" in s:
            for t, w in dict(zip(s["bias_tokens"][b].tolist(), s["bias_values"][b].tolist())).items():
                if 0 <= t < V:
                    x[b, t] += w
                    M[b, t] += abs(w)
        if "mask" in s:
            row = s["mask"][b if s["mask"].shape[0] > 1 else 0]
            for t in range(V):
                if not (int(row[t // 32]) >> (t % 32)) & 1:
                    x[b, t] = -math.inf
    return x, M


def check(got, s):
    want, M = reference(s)
    fine = torch.isfinite(want)
    got = got.double().cpu()
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(got[~fine], want[~fine])
    u = torch.finfo(s["logits"].dtype).eps / 2
    err = 5 * 2.0 ** -24 * M
    bound = u * (want.abs() + err) + err + (2.0 ** -25 if s["logits"].dtype == torch.float16 else 0)
    assert bool(((got - want).abs() <= bound)[fine].all())


def call(s, **more):
    return ops.adjust_logits(**{k: t.to(DEV) for k, t in s.items()}, **more)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,L,N,mask", [(1, 1, 1, 0, False), (1, 31, 5, 1, True), (3, 1000, 200, 30, True), (2, 1023, 0, 3, False),
                                          (4, 1025, 64, 0, True), (1, 5003, 3000, 300, True), (700, 2051, 9, 2, False),
                                          (2, 40000, 1500, 40, False), (300, 5000, 20, 0, False)])
def test_rules(R, V, L, N, mask, dtype):
    s = make(R, V, L, N, mask, dtype, seed=V)
    got = call(s)
    check(got, s)
    x = s["logits"].to(DEV)                   # in place
    rest = {k: t for k, t in s.items() if k != "logits"}
    assert ops.adjust_logits(x, **{k: t.to(DEV) for k, t in rest.items()}, out=x) is x
    assert torch.equal(x, got)


@pytest.mark.parametrize("keys", [(), ("history", "lengths"), ("history", "lengths", "repetition"), ("history", "lengths", "frequency"),
                                  ("history", "lengths", "prompt_lens", "presence"), ("bias_tokens", "bias_values"), ("mask",)])
def test_any_rule_alone(keys):
    s = make(3, 1500, 100, 20, True, torch.float16)
    s = {k: s[k] for k in ("logits",) + keys}
    check(call(s), s)
    if not keys:
        assert torch.equal(call(s).cpu(), s["logits"])


def test_lengths_out_of_range_are_held_to_the_history():
    s = make(4, 300, 50, 0, False, torch.float32)
    s["lengths"], s["prompt_lens"] = torch.tensor([-5, 1 << 40, 50, 0]), torch.tensor([-3, -(1 << 40), 1 << 40, 5])
    got = call(s)
    s["lengths"], s["prompt_lens"] = torch.tensor([0, 50, 50, 0]), torch.tensor([0, 0, 50, 5])
    check(got, s)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_that_are_not_aligned(dtype):
    """Rows of odd length and distance, output aligned otherwise than the input, one mask for all rows, a history cut out of a longer one."""
    s = make(5, 1999, 70, 4, True, dtype)
    s["mask"] = s["mask"][:1]
    d = {k: t.to(DEV) for k, t in s.items()}
    room = torch.zeros(5, 2111, dtype=dtype, device=DEV)
    d["logits"] = room[:, 3:3 + 1999].copy_(d["logits"])
    d["history"] = torch.nn.functional.pad(d["history"], (1, 4))[:, 1:71]
    for out in (None, torch.zeros(5, 2003, dtype=dtype, device=DEV)[:, 1:2000], d["logits"]):
        check(ops.adjust_logits(**d, out=out), s)
    assert bool((room[:, :3] == 0).all()) and bool((room[:, 2002:] == 0).all())


def test_infinities_and_nan():
    """-infinity and the type's lowest value stay what they are or round to it; NaN passes, except where the mask forbids it."""
    low = torch.finfo(torch.float16).min
    x = torch.tensor([[math.inf, -math.inf, low, math.nan, math.nan, 1.0]], dtype=torch.float16)
    s = {"logits": x, "history": torch.arange(6)[None], "lengths": torch.tensor([6]), "repetition": torch.tensor([1.5]),
         "presence": torch.tensor([0.5]), "mask": torch.tensor([[0b101111]], dtype=torch.int32)}
    got = call(s)[0].cpu()
    assert got[0] == math.inf and got[1] == -math.inf and got[2] == -math.inf and bool(got[3].isnan()) and got[4] == -math.inf
    one = torch.tensor(1.0) / 1.5 - 0.5
    assert abs(float(got[5]) - float(one)) <= 2.0 ** -11 * float(one)
    s["frequency"] = torch.tensor([math.inf])
    s["lengths"] = torch.tensor([0])          # no token: nothing is multiplied by the infinity
    assert float(call(s)[0, 5]) == 1.0


@pytest.mark.parametrize("L,N", [(65535, 32767), (65536, 20), (70, 32768), (66000, 33000)])
def test_long_texts_and_long_lists(L, N):
    """Counts and entries that fit a token's word just so, and those that have words of their own."""
    s = make(2, 3000, L, N, True, torch.float32, seed=L)
    s["history"][:, ::3] = 1234
    s["bias_tokens"][:, -1] = 77              # the last entry of all
    check(call(s), s)


def test_same_token_throughout():
    s = {"logits": torch.ones(2, 5000, dtype=torch.float32), "history": torch.full((2, 100000), 4321), "lengths": torch.tensor([100000, 99999]),
         "prompt_lens": torch.tensor([1, 0]), "frequency": torch.tensor([0.25, 0.5]), "presence": torch.tensor([1.0, 2.0])}
    got = call(s).cpu()
    assert got[0, 4321] == 1 - 0.25 * 99999 - 1 and got[1, 4321] == 1 - 0.5 * 99999 - 2
    got[:, 4321] = 1
    assert bool((got == 1).all())


def test_graph_and_stream():
    s = {k: t.to(DEV) for k, t in make(8, 3001, 300, 10, True, torch.float16).items()}
    want = [ops.adjust_logits(**dict(s, lengths=(s["lengths"] + i))) for i in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.adjust_logits(**s)
    side.synchronize()
    assert torch.equal(got, want[0])
    s = dict(s, lengths=s["lengths"].clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.adjust_logits(**s)
        s["lengths"].add_(1)
    for w in want:
        g.replay()
        assert torch.equal(y, w)


def test_refusals():
    s = {k: t.to(DEV) for k, t in make(3, 100, 20, 4, True, torch.float16).items()}
    x = s["logits"]
    for change, error in [
        ({"logits": x.double()}, TypeError), ({"logits": x[0]}, ValueError), ({"logits": x[:, ::2]}, ValueError), ({"logits": x[:0]}, ValueError),
        ({"lengths": None}, ValueError), ({"history": None}, ValueError), ({"history": None, "lengths": None}, ValueError),
        ({"history": s["history"].int()}, TypeError), ({"history": s["history"][:2]}, ValueError), ({"lengths": s["lengths"][:2]}, ValueError),
        ({"lengths": s["lengths"].int()}, TypeError), ({"repetition": s["repetition"].half()}, TypeError), ({"repetition": s["repetition"][:1]}, ValueError),
        ({"bias_values": None}, ValueError), ({"bias_tokens": s["bias_tokens"][:, :2]}, ValueError), ({"bias_values": s["bias_values"].half()}, TypeError),
        ({"mask": s["mask"].long()}, TypeError), ({"mask": s["mask"][:, :3]}, ValueError), ({"mask": s["mask"][:2]}, ValueError), ({"mask": s["mask"].cpu()}, RuntimeError),
        ({"out": x.float()}, TypeError), ({"out": x[:, :50]}, ValueError), ({"out": x.flip(0)[:2]}, ValueError), ({"out": x[:1].expand(3, 100)}, ValueError),
        ({"logits": x.clone().requires_grad_()}, RuntimeError),
    ]:
        with pytest.raises(error):
            ops.adjust_logits(**dict(s, **change))
    wide = torch.zeros(3, 200, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.adjust_logits(**dict(s, logits=wide[:, :100], out=wide[:, 1:101]))
