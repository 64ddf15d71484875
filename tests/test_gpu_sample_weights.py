"""How far the weights of ops.sample are off, and that none is lost at the end of the bins: no tolerance but the header's.

A weight w, the largest being 1, is a whole number of units of 2^-49 here (up to 8192 tokens) and off by half a unit and 2^-32 of itself at most.  64 bits are off by 2^-52.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import ops
    DEV = torch.device("cuda:0")


def exp(x):
    """By numpy: torch's on the CPU was off by 2^-28 in a part of the numbers, in the first call of a process and in no other."""
    return torch.from_numpy(np.exp(x.numpy()))


@pytest.mark.parametrize("seed", range(3))
def test_weights_are_off_by_what_the_header_says(seed):
    """Two tokens, the second of weight 1: the first is drawn if its weight is more than u / (1 - u).  The random numbers are next to that, between 2^-32 and 2^-28 of a weight away."""
    g = torch.Generator().manual_seed(seed)
    n = 1 << 21
    x = -(torch.rand(n, generator=g, dtype=torch.float64) * 14 + 0.01).float()
    t = (torch.rand(n, generator=g, dtype=torch.float64) * 0.8 + 0.6).float()
    w = exp(x.double() / t.double())
    u = (w / (1 + w)).float()
    border = u.double() / (1 - u.double())
    off = (w - border).abs()
    near = (off > 2.0 ** -32 * w + 2.0 ** -50 * (1 + 2.0 ** -10)) & (off < 2.0 ** -28 * w)
    x, t, u, first = x[near], t[near], u[near], (w > border)[near]
    assert x.numel() > 20000
    logits = torch.stack([x, torch.zeros_like(x)], 1)
    out = ops.sample(logits.to(DEV), u.to(DEV), temperature=t.to(DEV)).cpu()
    assert int((out != (~first).long()).sum()) == 0


def test_a_crowd_of_equal_weights():
    """8000 tokens of the same small weight: their errors are one error, which the sum shows."""
    n = 12000
    g = torch.Generator().manual_seed(9)
    x = -(torch.rand(n, generator=g, dtype=torch.float64) * 9 + 0.01).float()
    w = exp(x.double())
    u = (8000 * w / (1 + 8000 * w)).float()                   # the last token, of weight 1, or one of the crowd
    border = u.double() / (1 - u.double())
    off = (8000 * w - border).abs()
    sure = off > 8000 * (2.0 ** -32 * w + 2.0 ** -50 * (1 + 2.0 ** -10))
    near = sure & (off < 2.0 ** -25 * 8000 * w)
    assert int(near.sum()) > 300
    logits = x[near][:, None].expand(-1, 8001).clone()
    logits[:, 8000] = 0
    out = ops.sample(logits.to(DEV), u[near].to(DEV)).cpu()
    assert torch.equal(out == 8000, (8000 * w < border)[near])


def at_the_end():
    """Temperatures and largest logits for which a logit of 0 has a little more than half a unit of weight and 1024 bins, counted in fp32, end before it."""
    found = []
    for t in np.linspace(0.5, 2, 3000).astype(np.float32):
        step = 1.4426950408889634 / float(t)
        per_half = np.float32(step * 2048 / 50)
        near = np.float32(50 / step)
        for k in range(-6, 7):
            top = (np.array([near]).view(np.int32) + k).view(np.float32)[0]
            if 1e-6 < 50 - float(top) * step and np.float32(0.5) * top * per_half >= 1024:
                found.append((50 - float(top) * step, float(t), float(top)))
    return sorted(found, reverse=True)[:20]


def test_top_k_counts_the_smallest_weights():
    """Of 998 tokens with half a unit of weight and more, all unlike, top-k keeps the two largest beside the top one, and with no random number the lowest that is kept is drawn."""
    rows = at_the_end()
    assert len(rows) == 20
    small = torch.arange(1, 999, dtype=torch.float64) * 2.0 ** -60
    logits = torch.stack([torch.cat([small, torch.tensor([top], dtype=torch.float64)]) for _, _, top in rows]).float()
    temperature = torch.tensor([t for _, t, _ in rows])
    assert all(0.5 < 2.0 ** 49 * math.exp((float(row[0]) - float(row[-1])) / t) < 0.51 for row, (_, t, _) in zip(logits, rows))
    k = torch.full((20,), 3, dtype=torch.long)
    out = ops.sample(logits.to(DEV), torch.zeros(20, device=DEV), temperature=temperature.to(DEV), top_k=k.to(DEV)).cpu()
    assert bool((out >= 996).all()), out
