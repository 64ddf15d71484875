"""Sampling (ops.sample) against the definition in 64 bits, whole numbers: no tolerance.

A token may only differ from the definition's where a random number, a share of top-p or min-p falls within rounding of a border.  The kernel's weights are off by
2^-32 of themselves and half a unit of 2^-F each (F is 45 at 100000 tokens), so two sums differ by 2^-31 of themselves
and 2^-46 per token at most, and 64 bits by 2^-52 relative; the reference says for each row whether any decision lay within 2^-30 of a
border, and such rows are not drawn: the seeds here have none (asserted).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def reference(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, how far from a border the nearest decision was, relative) with one row at a time on the CPU."""
    tokens, nearest = [], math.inf
    for b in range(x.shape[0]):
        row = x[b].double().cpu()
        row = torch.where(torch.isnan(row), -math.inf, row)
        t = 1.0 if temperature is None else float(temperature[b])
        top = row.max()
        if not t >= 1e-18 or (top_k is not None and int(top_k[b]) == 1) or top == -math.inf:
            tokens.append(int((row == top).nonzero()[0]))
            continue
        w = torch.where(row == top, 1.0, torch.exp((row - top) / t) if top < math.inf else 0.0)
        w = torch.nan_to_num(w, nan=0.0)
        order = torch.sort(row, descending=True, stable=True).indices
        n = row.numel()
        if top_k is not None and int(top_k[b]) > 0:
            n = min(n, int(top_k[b]))
        if top_p is not None and float(top_p[b]) < 1:
            sums = torch.cumsum(w[order[:n]], 0)
            goal = max(float(top_p[b]), 0.0) * sums[-1]
            if goal > 0:
                nearest = min(nearest, float(((sums[:-1] - goal).abs() / sums[-1]).min()) if n > 1 else math.inf)
            n = min(n, 1 + int((sums < goal).sum()))
        if min_p is not None and float(min_p[b]) > 0:
            kept = w[order[:n]]
            if n > 1 and float(min_p[b]) < 1:
                nearest = min(nearest, float((kept[1:][kept[1:] < 1] - float(min_p[b])).abs().min()) if (kept[1:] < 1).any() else math.inf)
            n = max(1, int((kept >= float(min_p[b])).sum()))
        chosen = torch.sort(order[:n]).values
        sums = torch.cumsum(w[chosen], 0)
        goal = min(max(float(u[b]), 0.0), 1 - 2.0 ** -60) * sums[-1]
        if 0 < float(u[b]) < 1:
            nearest = min(nearest, float(((sums - goal).abs() / sums[-1]).min()))
        at = int((sums <= goal).sum())
        if float(u[b]) >= 1:
            at = int((w[chosen] > 2.0 ** -44).nonzero()[-1])
        tokens.append(int(chosen[min(at, n - 1)]))
    return torch.tensor(tokens), nearest


def numbers(rows, seed=0, kind="all"):
    g = torch.Generator().manual_seed(seed)
    r = lambda: torch.rand(rows, generator=g)
    out = {"temperature": (0.4 + 1.2 * r()).to(DEV)}
    k, p, m = torch.randint(0, 60, (rows,), generator=g), 0.3 + 0.7 * r(), 0.1 * r()
    if kind in ("k", "all"):
        out["top_k"] = k.to(DEV)
    if kind in ("p", "all"):
        out["top_p"] = p.to(DEV)
    if kind in ("m", "all"):
        out["min_p"] = m.to(DEV)
    return r().to(DEV), out


def check(x, u, margin=2.0 ** -30, **kw):
    want, nearest = reference(x, u, **kw)
    assert nearest > margin
    got = ops.sample(x, u, **kw)
    assert got.dtype == torch.int64 and got.shape == (x.shape[0],)
    assert torch.equal(got.cpu(), want), (got.cpu() != want).nonzero().flatten().tolist()
    assert torch.equal(got, ops.sample(x, u, **kw))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("kind", ["none", "k", "p", "m", "all"])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (5, 31), (2, 1000), (1, 32000), (4, 50272), (300, 257), (33, 4099), (3, 100003)])
def test_against_64_bits(rows, V, kind, dtype):
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (3 * torch.randn(rows, V, generator=g, device=DEV)).to(dtype)
    u, kw = numbers(rows, seed=V, kind=kind)
    check(x, u, **kw)


def test_a_vocabulary_of_the_largest_size():
    g = torch.Generator(device=DEV).manual_seed(0)
    x = 3 * torch.randn(2, 1 << 18, generator=g, device=DEV)
    u, kw = numbers(2, seed=1, kind="p")
    check(x, u, **kw)
    check(x.half(), u, **kw)
    with pytest.raises(ValueError):
        ops.sample(torch.zeros(1, (1 << 18) + 1, device=DEV), u[:1])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_border_among_equal_logits(dtype):
    """All the same, and few values: which of them are kept goes by the token."""
    V = 5000
    u = (torch.arange(16, device=DEV) + 0.37) / 16
    same = torch.full((16, V), -2.5, dtype=dtype, device=DEV)
    for kw in ({}, dict(top_k=torch.arange(1, 17, device=DEV) * 37), dict(top_p=torch.linspace(0.003, 0.9771, 16, device=DEV))):
        # All weights are 1 and all sums whole numbers, exact on both sides: only p * 5000 and u * n are rounded (2^-53), and only in the reference
        check(same, u, margin=2.0 ** -50, **kw)
    few = (torch.randint(0, 4, (16, V), generator=torch.Generator().manual_seed(2)) * 1.5).to(dtype).to(DEV)
    for kw in ({}, dict(top_k=torch.arange(1, 17, device=DEV) * 137), dict(top_p=torch.linspace(0.003, 0.9771, 16, device=DEV)),
               dict(top_k=torch.arange(1, 17, device=DEV) * 237, top_p=torch.linspace(0.103, 0.9571, 16, device=DEV))):
        check(few, u, **kw)


@pytest.mark.parametrize("dtype,V", [(F32, 1 << 18), (F32, 150001), (F16, 1 << 18), (F16, 9000)])
def test_a_crowd_of_equal_logits_below_the_largest(dtype, V):
    """Sums of one number many times over, whose bits do not end: nothing passes over in the bins."""
    x = torch.full((6, V), -1.2345, device=DEV)
    x[:, 77], x[:, 4001] = 0.0, -0.3
    x[5, ::2] = -1.5
    u = torch.tensor([0.1234, 0.5555, 0.91, 0.3, 0.77, 0.6], device=DEV)
    p = torch.tensor([0.5, 0.31, 0.9, 0.777, 0.123, 0.66], device=DEV)
    k = torch.tensor([V // 2, V // 3, 5000, V - 3, 100, V - V // 3], device=DEV)
    x = x.to(dtype)
    check(x, u, top_p=p)
    check(x, u, top_k=k)
    check(x, u, top_p=p, top_k=k, temperature=torch.full((6,), 0.9, device=DEV))


def test_values_around_zero_and_of_all_sizes():
    """The bits of x between two close values span many powers of two near zero."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(24, 3000, generator=g) * torch.exp2(torch.randint(-40, 1, (24, 3000), generator=g).float())
    x[::2] *= 0.01
    x[1::4] -= 1000
    u, kw = numbers(24, seed=5)
    kw["top_k"] = torch.randint(2, 2500, (24,), generator=g).to(DEV)
    kw["min_p"] = torch.zeros(24, device=DEV)
    kw["temperature"][:8] = torch.tensor([1e-3, 1e-2, 10.0, 1e3, 1e6, 1e-1, 30.0, 1e10], device=DEV)
    check(x.to(DEV), u, **kw)
    check(x.half().to(DEV), u, **kw)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_the_edges(dtype):
    inf, nan = math.inf, math.nan
    x = torch.zeros(20, 40)
    x[0] = -inf
    x[1], x[1, 7] = -inf, -3.0
    x[2] = nan
    x[3], x[3, 5], x[3, 9] = nan, 1.0, 1.0
    x[4, 11] = x[4, 30] = inf
    x[5, 3], x[5, 17] = nan, 5.0
    x[6] = torch.arange(40) % 2 * 50.0
    x[7, 20:] = -inf
    x[8:] = torch.randn(12, 40, generator=torch.Generator().manual_seed(1))
    x = x.to(dtype).to(DEV)
    u = torch.full((20,), 0.6180339, device=DEV)
    u[12:16] = torch.tensor([0.0, 1.0, -1.0, 2.0])
    t = torch.ones(20, device=DEV)
    t[8:12] = torch.tensor([0.0, -1.0, nan, 1e-30])
    check(x, u, temperature=t)
    got = ops.sample(x, u, temperature=t).cpu()
    assert got[0] == 0 and got[1] == 7 and got[2] == 0 and got[3] == 9 and got[4] == 30 and got[12] == got[14] == 0 and got[13] == got[15] == 39
    assert torch.equal(got[8:12], x[8:12].float().cpu().argmax(1))
    p = torch.full((20,), 0.9, device=DEV)
    p[:8:2] = 0.0
    p[16:] = torch.tensor([nan, 1.0, 5.0, -2.0])
    k = torch.full((20,), 30, device=DEV)
    k[16:] = torch.tensor([-5, 0, 1 << 40, 1])
    m = torch.tensor([0.0, 1.0, 0.05, 2.0] * 5, device=DEV)
    check(x, u, top_p=torch.nan_to_num(p, nan=1.0))
    assert torch.equal(ops.sample(x, u, top_p=p), ops.sample(x, u, top_p=torch.nan_to_num(p, nan=1.0)))
    check(x, u, top_p=torch.nan_to_num(p, nan=1.0), top_k=k)
    check(x, u, min_p=m, top_k=k)
    big = x.clone()
    big[8:] = torch.finfo(dtype).max * torch.linspace(-1, 1, 40, device=DEV).to(dtype)
    check(big, u, temperature=torch.full((20,), 1e38, device=DEV), top_k=k)
    assert torch.equal(ops.sample(torch.zeros_like(x), u, temperature=torch.full((20,), inf, device=DEV)), ops.sample(torch.zeros_like(x), u))


def test_distribution():
    """A hundred thousand rows of one distribution: each token's share within five standard deviations."""
    x = torch.tensor([0.3, -1.0, 2.0, 0.3, -inf_(), 1.1], device=DEV).expand(100000, 6)
    n = x.shape[0]
    u = torch.rand(n, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV)
    for kw, kept in (({}, [0, 1, 2, 3, 5]), (dict(top_k=torch.full((n,), 3, device=DEV)), [0, 2, 5]), (dict(top_p=torch.full((n,), 0.6, device=DEV)), [2, 5])):
        p = torch.zeros(6, dtype=torch.float64)
        p[kept] = torch.softmax(x[0].cpu().double()[kept], 0)
        share = torch.bincount(ops.sample(x, u, **kw).cpu(), minlength=6).double() / n
        assert bool(((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt() + (p > 0) / n).all())


def inf_():
    return math.inf


def test_views_streams_graphs_and_the_output():
    g = torch.Generator(device=DEV).manual_seed(3)
    wide = torch.randn(5, 2 * 1001 + 3, generator=g, device=DEV).half()
    x = wide[1:, 3:1004]                                    # rows at odd places
    u, kw = numbers(4, seed=9)
    check(x, u, **kw)
    out = torch.zeros(4, dtype=torch.long, device=DEV)
    assert ops.sample(x, u, out=out, **kw).data_ptr() == out.data_ptr() and out._version > 0
    s = torch.cuda.Stream(DEV)
    s.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(s):
        other = ops.sample(x, u, **kw)
    torch.cuda.current_stream(DEV).wait_stream(s)
    assert torch.equal(out, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(x, u, out=out, **kw)
    for i in range(5):
        wide.copy_(torch.randn(wide.shape, generator=g, device=DEV))
        u.copy_(torch.rand(4, generator=g, device=DEV))
        graph.replay()
        assert torch.equal(out.cpu(), reference(x, u, **kw)[0])


def test_refusals():
    x, u = torch.zeros(3, 10, device=DEV), torch.zeros(3, device=DEV)
    k = torch.zeros(3, dtype=torch.long, device=DEV)
    for error, call in [
        (TypeError, lambda: ops.sample(None, u)), (TypeError, lambda: ops.sample(x, None)), (TypeError, lambda: ops.sample(x.double(), u)),
        (TypeError, lambda: ops.sample(x, u.double())), (TypeError, lambda: ops.sample(x, u, top_k=k.int())), (TypeError, lambda: ops.sample(x, u, temperature=1.0)),
        (TypeError, lambda: ops.sample(x, u, out=k.int())), (RuntimeError, lambda: ops.sample(x.cpu(), u)), (RuntimeError, lambda: ops.sample(x, u.cpu())),
        (RuntimeError, lambda: ops.sample(x.clone().requires_grad_(), u)), (ValueError, lambda: ops.sample(x[0], u)), (ValueError, lambda: ops.sample(x[:, :0], u)),
        (ValueError, lambda: ops.sample(x.t(), torch.zeros(10, device=DEV))), (ValueError, lambda: ops.sample(x, u[:2])), (ValueError, lambda: ops.sample(x, u, top_p=u[:1])),
        (ValueError, lambda: ops.sample(x, u, top_k=k[:, None])), (ValueError, lambda: ops.sample(x, u, out=k[:2])), (ValueError, lambda: ops.sample(x, u, top_k=k, out=k)),
    ]:
        with pytest.raises(error):
            call()
