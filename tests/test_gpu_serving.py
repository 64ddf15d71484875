"""GPTQDecoder with a window and sinks, with a prefix that a batch shares, and with rules on the logits: each against the same model without it, eager against
captured, and all that go together in one run."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from autogptq.tvm_b200 import decoder, ops
    DEV = torch.device("cuda:0")


def config(arch="llama", heads=4, hidden=256, **more):
    return decoder.DecoderConfig(arch=arch, layers=2, hidden=hidden, heads=heads, inter=512, vocab=1003, bits=4, group_size=128, desc_act=arch == "opt",
                                 **{"max_seq": 96, **more})


def prompt_of(batch, n, seed=1, vocab=1003):
    return torch.randint(0, vocab, (batch, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def close(a, b, what):
    """Logits of two models that compute the same function in other orders: the output contract of the path, on the vocabulary projection."""
    tol = 1e-2 * float(b.last_hidden.float().norm(dim=-1).min()) * float(b.lm_head.float().abs().max())
    x, y = (m.last_logits.float()[:, :m.cfg.vocab] for m in (a, b))
    assert bool(torch.isfinite(x).all()) and float((x - y).abs().max()) <= tol, what


def step(models, first):
    tokens = first.tokens.clone()
    for m in models:
        m.tokens.copy_(tokens)
        m.decode(1)


@pytest.mark.parametrize("arch,heads,hidden,window,sinks,batch", [("llama", 4, 256, 7, 2, 1), ("llama", 2, 256, 20, 4, 3), ("opt", 4, 256, 7, 0, 2),
                                                                  ("llama", 4, 256, 1, 1, 1), ("opt", 2, 256, 500, 3, 1)])
def test_window_fused_and_framework_paths_agree(arch, heads, hidden, window, sinks, batch):
    cfg = config(arch, heads, hidden, window=window, sinks=sinks)
    a, b = (decoder.GPTQDecoder(cfg, batch=batch, device=DEV, fused=f) for f in (True, False))
    prompt = prompt_of(batch, 33)
    for m in (a, b):
        m.prefill(prompt)
    close(a, b, "prompt")
    for i in range(6):
        step((b, a), b)
        close(a, b, f"step {i}")


def test_a_window_that_holds_everything_is_no_window():
    cfg, whole = config(window=96), config()
    a, b = decoder.GPTQDecoder(cfg, batch=2, device=DEV), decoder.GPTQDecoder(whole, batch=2, device=DEV)
    for m in (a, b):
        m.prefill(prompt_of(2, 40))
    for i in range(5):
        close(a, b, f"step {i}")
        step((b, a), b)


@pytest.mark.parametrize("arch,batch,P,n", [("llama", 3, 30, 17), ("opt", 2, 21, 9), ("llama", 1, 1, 50), ("llama", 12, 47, 3), ("opt", 40, 5, 1)])
def test_a_shared_prefix_is_the_same_text(arch, batch, P, n):
    cfg = config(arch)
    prefix, prompt = prompt_of(1, P, 7)[0], prompt_of(batch, n)
    a, b = decoder.GPTQDecoder(cfg, batch=batch, device=DEV), decoder.GPTQDecoder(cfg, batch=batch, device=DEV)
    a.share_prefix(prefix)
    a.prefill(prompt)
    b.prefill(torch.cat([prefix.expand(batch, P), prompt], 1))
    close(a, b, "prompt")
    for i in range(5):
        step((b, a), b)
        close(a, b, f"step {i}")
    assert int(a.pos) == n + 5
    a.share_prefix(None)                      # and back
    a.prefill(prompt)
    b.prefill(prompt)
    close(a, b, "without")
    step((b, a), b)
    close(a, b, "a step without")


def test_a_prefix_longer_than_the_caches():
    cfg, long = config(max_seq=40), config(max_seq=200)
    prefix, prompt = prompt_of(1, 120, 3)[0], prompt_of(2, 11)
    a, b = decoder.GPTQDecoder(cfg, batch=2, device=DEV), decoder.GPTQDecoder(long, batch=2, device=DEV)
    a.share_prefix(prefix)
    a.prefill(prompt)
    b.prefill(torch.cat([prefix.expand(2, 120), prompt], 1))
    for i in range(4):
        close(a, b, f"step {i}")
        step((b, a), b)


def ruled(base, history, prompt_len, rules, i):
    x = base.double().clone()
    text = history[i]
    r, f, p = (v[i] if isinstance(v, list) else v for v in (rules.repetition or 1.0, rules.frequency or 0.0, rules.presence or 0.0))
    for t in set(text):
        x[t] = x[t] / r if x[t] > 0 else x[t] * r
    for t in set(text[prompt_len:]):
        x[t] -= f * text[prompt_len:].count(t) + p
    for t, w in (rules.bias[i] if isinstance(rules.bias, list) else rules.bias or {}).items():
        x[t] += w
    if rules.mask is not None:
        m = rules.mask[i % rules.mask.shape[0]].tolist()
        for t in range(len(x)):
            if not m[t // 32] >> (t % 32) & 1:
                x[t] = -math.inf
    return x


@pytest.mark.parametrize("batch,prefix", [(1, 0), (3, 0), (3, 13)])
def test_rules(batch, prefix):
    """The logits that the pick sees are the rules' of those of the same model without rules, with the whole text as history."""
    cfg = config()
    V, words = cfg.vocab, -(-cfg.vocab // 32)
    mask = torch.randint(-2 ** 31, 2 ** 31, (batch, words), generator=torch.Generator().manual_seed(5)).int()
    rules = decoder.LogitRules(repetition=[1.3 - 0.2 * i for i in range(batch)], frequency=0.4, presence=[0.1 * i for i in range(batch)],
                               bias=[{5 * i + 1: 9.0, 17: -3.0} for i in range(batch)], mask=mask)
    a, b = decoder.GPTQDecoder(cfg, batch=batch, device=DEV), decoder.GPTQDecoder(cfg, batch=batch, device=DEV)
    front, prompt = prompt_of(1, prefix, 7)[0], prompt_of(batch, 12)
    for m in (a, b):
        m.share_prefix(front if prefix else None)
    a.set_rules(rules)
    for m in (a, b):
        m.prefill(prompt)
    text = [front.tolist() + prompt[i].tolist() for i in range(batch)]
    for _ in range(12):
        base, got = b.last_logits.half(), a.last_logits.float().cpu()
        for i in range(batch):
            want = ruled(base[i, :V].cpu(), text, prefix + 12, rules, i)
            fine = torch.isfinite(want)
            assert torch.equal(torch.isfinite(got[i, :V]), fine)
            # one rounding to fp16, and a few in fp32 of numbers below 32
            assert bool(((got[i, :V].double() - want).abs()[fine] <= 2.0 ** -11 * want.abs()[fine] + 2.0 ** -16).all())
            assert int(a.tokens[i]) == int(got[i, :V].argmax())
            text[i].append(int(a.tokens[i]))
        step((b, a), a)


def test_everything_together_eager_and_captured():
    """A shared prefix, unlike requests with rules (a grammar that changes from step to step), tokens one by one, eager and from a graph; then rules with a window."""
    batch, steps = 3, 10
    for cfg, prefix in ((config(), prompt_of(1, 19, 7)[0]), (config(window=9, sinks=2), None)):
        words = -(-cfg.vocab // 32)
        g = torch.Generator().manual_seed(2)
        masks = [torch.randint(-2 ** 31, 2 ** 31, (batch, words), generator=g).int().to(DEV) for _ in range(steps)]
        runs = []
        for captured in (False, True):
            m = decoder.GPTQDecoder(cfg, batch=batch, device=DEV)
            m.share_prefix(prefix)
            mask = masks[0].clone()
            m.set_rules(decoder.LogitRules(repetition=1.2, frequency=[0.0, 0.3, -0.2], presence=0.5, bias={3: 2.0}, mask=mask))
            m.prefill(prompt_of(batch, 14))
            if captured:
                m.capture()
            out = []
            for k in masks:
                mask.copy_(k)
                out.append(m.decode(1).clone())
                for i in range(batch):        # what was picked is what the grammar allows
                    t = int(m.tokens[i])
                    assert int(k[i, t // 32]) >> (t % 32) & 1
            runs.append((torch.cat(out), m.last_logits.float().clone(), m.history[:, :60].clone()))
        assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
        done = (0 if prefix is None else 19) + 14 + steps
        assert torch.equal(runs[0][2][:, :done], runs[1][2][:, :done])
    ops.check_status(DEV)


def test_rules_leave_when_they_are_taken_back():
    cfg = config()
    a, b = decoder.GPTQDecoder(cfg, batch=1, device=DEV), decoder.GPTQDecoder(cfg, batch=1, device=DEV)
    a.set_rules(decoder.LogitRules(bias={7: 1000.0}))
    for m in (a, b):
        m.prefill(prompt_of(1, 5))
    assert int(a.tokens) == 7
    assert torch.equal(a.decode(3).cpu(), torch.full((3, 1), 7))
    a.set_rules(None)
    a.prefill(prompt_of(1, 5))
    assert torch.equal(a.decode(6), b.decode(6))


def test_refusals():
    m = decoder.GPTQDecoder(config(window=5), batch=2, device=DEV)
    t = prompt_of(1, 5)[0]
    with pytest.raises(ValueError):
        m.share_prefix(t)                     # window and prefix
    m = decoder.GPTQDecoder(config("opt"), batch=2, device=DEV)
    for bad in (t[None], t.int(), prompt_of(1, 96)[0]):
        with pytest.raises(ValueError):
            m.share_prefix(bad)
    m.share_prefix(prompt_of(1, 90)[0])
    with pytest.raises(ValueError):
        m.prefill(prompt_of(2, 7))            # past the learned positions
    m.prefill(prompt_of(2, 4))
    with pytest.raises(ValueError):
        m.decode(3)
    m.decode(2)
    for rules in (decoder.LogitRules(repetition=0.0), decoder.LogitRules(repetition=[1.0]), decoder.LogitRules(frequency=math.nan),
                  decoder.LogitRules(bias={1003: 1.0}), decoder.LogitRules(bias=[{}]), decoder.LogitRules(mask=torch.zeros(2, 31, dtype=torch.int32)),
                  decoder.LogitRules(mask=torch.zeros(2, 32))):
        with pytest.raises(ValueError):
            m.set_rules(rules)
    with pytest.raises(ValueError):
        decoder.GPTQDecoder(config(window=0), device=DEV)
    unfused = decoder.GPTQDecoder(config(), device=DEV, fused=False)
    with pytest.raises(ValueError):
        unfused.share_prefix(t)
