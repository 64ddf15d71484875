"""GPTQDecoder with caches of 4 bits and with sampling: against a plain model whose keys and values are rounded by the format's definition, eager against captured, and
all that goes together in one run."""
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


def held(packed, constants):
    """What rows of a cache of 4 bits stand for, in 32 bits."""
    hd = packed.shape[-1] * 2
    words = packed.to(torch.int64).reshape(*packed.shape[:-1], hd // 8, 4)
    words = words[..., 0] | words[..., 1] << 8 | words[..., 2] << 16 | words[..., 3] << 24
    codes = torch.zeros(*packed.shape[:-1], hd, device=packed.device)
    for w in range(hd // 8):
        for f, e in enumerate((0, 2, 32, 34, 1, 3, 33, 35)):
            codes[..., 64 * (w % (hd // 64)) + 4 * (w // (hd // 64)) + e] = (words[..., w] >> 4 * f & 15).float()
    wide = constants.float().repeat_interleave(hd // constants.shape[-2], -2)
    return codes * wide[..., 0] + wide[..., 1]


class Plain:
    """The model's layers as plain expressions around its linears.  Keys and values are what the model's caches stand for (a value in the middle between two codes may
    fall either way with the last bit of a sum in front of it, which moves the logits by more than rounding does); those of the first layer, before they are quantised,
    are kept, to be compared with them."""

    def __init__(self, model):
        self.m, self.k, self.v, self.at = model, [], [], 0

    def run(self, tokens):
        """Logits of the last of ``tokens`` [B, S], which follow what was run before.  The model has run them already."""
        m, cfg = self.m, self.m.cfg
        B, S = tokens.shape
        idx = torch.arange(self.at, self.at + S, device=DEV)
        x = m._embed(tokens, idx)
        for i, L in enumerate(m.layers):
            qkv = L.qkv(m._norm(x, L.norm1_w, L.norm1_b).reshape(B * S, cfg.hidden)).reshape(B, S, 3, cfg.heads, cfg.head_dim)
            q, k, v = (t.transpose(1, 2) for t in qkv.unbind(2))
            if cfg.arch == "llama":
                cos, sin = m.cos[idx].float(), m.sin[idx].float()
                q, k = (m._rope(t.float(), cos, sin).half() for t in (q, k))
            if i == 0:
                self.k.append(k)
                self.v.append(v)
            rows = slice(0, self.at + S)
            K, V = held(L.cache.k[:, :, rows], L.cache.k_scales[:, :, rows]), held(L.cache.v[:, :, rows], L.cache.v_scales[:, :, rows])
            j = torch.arange(K.shape[2], device=DEV)[None, :]
            seen = j <= idx[:, None]
            if cfg.window is not None:
                seen &= (j > idx[:, None] - cfg.window) | (j < cfg.sinks)
            w = torch.softmax((q.double() @ K.double().transpose(2, 3) / math.sqrt(cfg.head_dim)).masked_fill(~seen, -math.inf), -1)
            att = (w @ V.double()).half().transpose(1, 2).reshape(B * S, cfg.hidden)
            x = x + L.o(att).reshape(B, S, cfg.hidden)
            u = L.up(m._norm(x, L.norm2_w, L.norm2_b).reshape(B * S, cfg.hidden))
            act = torch.nn.functional.silu(u[:, :cfg.inter]) * u[:, cfg.inter:] if cfg.arch == "llama" else torch.relu(u)
            x = x + L.down(act.contiguous()).reshape(B, S, cfg.hidden)
        self.at += S
        self.h = m._norm(x[:, -1], m.final_norm_w, m.final_norm_b)
        return m._project(self.h).float()[:, :cfg.vocab]


def close(m, plain, logits, what):
    """The output contract of the path, on the vocabulary projection."""
    tol = 1e-2 * float(plain.h.float().norm(dim=-1).min()) * float(m.lm_head.float().abs().max())
    x = m.last_logits.float()[:, :m.cfg.vocab]
    assert bool(torch.isfinite(x).all()) and float((x - logits).abs().max()) <= tol, what


@pytest.mark.parametrize("arch,heads,hidden,batch,n,more", [
    ("llama", 4, 256, 1, 33, {}), ("llama", 2, 256, 3, 80, dict(cache_group=64)), ("opt", 4, 256, 2, 70, {}), ("opt", 2, 256, 1, 5, {}),
    ("llama", 4, 256, 2, 33, dict(window=7, sinks=2)), ("llama", 2, 256, 2, 90, dict(max_seq=2300)), ("llama", 4, 256, 12, 1, {})])
def test_against_a_plain_model(arch, heads, hidden, batch, n, more):
    cfg = config(arch, heads, hidden, cache_bits=4, **more)
    m = decoder.GPTQDecoder(cfg, batch=batch, device=DEV)
    plain, prompt = Plain(m), prompt_of(batch, n)
    m.prefill(prompt)
    close(m, plain, plain.run(prompt), "prompt")
    for i in range(6):
        token = m.tokens.clone()
        m.decode(1)
        close(m, plain, plain.run(token[:, None]), f"step {i}")
    # The first layer's rows: half a scale, 15 roundings of it (2^-11), and what the model's own linears and rotation are off by (2^-8 of a value and 1e-3)
    c = m.layers[0].cache
    for got, scales, want in zip(ops.cache_read(c), (c.k_scales, c.v_scales), (plain.k, plain.v)):
        want = torch.cat(want, 2).float()
        steps = scales[:, :, :n + 6, :, 0].float().repeat_interleave(cfg.cache_group, -1)
        assert bool(((got[:, :, :n + 6].float() - want).abs() <= (0.5 + 15 * 2.0 ** -11) * steps + 2.0 ** -8 * want.abs() + 1e-3).all())
        assert not got[:, :, n + 6:].any()


def test_the_caches_are_smaller():
    a, b = (decoder.GPTQDecoder(config(cache_bits=bits), batch=2, device=DEV) for bits in (4, 16))
    assert a.layers[0].k_cache is None and b.layers[0].cache is None
    whole = 2 * b.layers[0].k_cache.numel() * 2
    assert a.layers[0].cache.nbytes * 3.2 == whole


def test_drawn_tokens_are_the_definitions():
    """Every token, of the prompt's pick and of the steps, follows from the logits that the model shows and the random number of its position."""
    batch, vocab = 3, 1003
    for more in ({}, dict(cache_bits=4)):
        m = decoder.GPTQDecoder(config(**more), batch=batch, device=DEV)
        m.set_sampling(decoder.Sampling(temperature=[0.5, 2.0, 0.0], top_k=[40, 0, 5], top_p=0.9, min_p=0.01, seed=3))
        for n in (7, 11):
            m.prefill(prompt_of(batch, n))
            for i in range(5):
                u = m._uniform[n - 1 + i]
                want = ops.sample(m.last_logits[:, :vocab], u, **m._sampling_arguments)
                assert torch.equal(want, m.tokens) and int(m.pos) == n + i
                assert int(m.tokens[2]) == int(m.last_logits[2, :vocab].float().argmax())
                m.decode(1)


def test_same_seed_same_text_and_back_to_greedy():
    a, b = (decoder.GPTQDecoder(config(), batch=2, device=DEV) for _ in range(2))
    texts = []
    for m, seed in ((a, 5), (b, 5), (b, 6)):
        m.set_sampling(decoder.Sampling(temperature=30.0, seed=seed))
        for _ in range(2):
            m.prefill(prompt_of(2, 9))
            texts.append(m.decode(20))
    assert torch.equal(texts[0], texts[2]) and torch.equal(texts[1], texts[3])
    assert not torch.equal(texts[0], texts[1]) and not torch.equal(texts[0], texts[4])
    a.set_sampling(None)
    fresh = decoder.GPTQDecoder(config(), batch=2, device=DEV)
    for m in (a, fresh):
        m.prefill(prompt_of(2, 9))
    assert torch.equal(a.decode(5), fresh.decode(5))
    b.set_sampling(decoder.Sampling(temperature=0.0))
    b.prefill(prompt_of(2, 9))
    fresh.prefill(prompt_of(2, 9))
    assert torch.equal(b.decode(5), fresh.decode(5))


def test_everything_together_eager_and_captured():
    """Caches of 4 bits, rules with a grammar that changes from step to step, sampling; with and without a window; eager and from a graph."""
    batch, steps = 3, 10
    for cfg in (config(cache_bits=4), config(cache_bits=4, cache_group=64, window=9, sinks=2, max_seq=2200)):
        words = -(-cfg.vocab // 32)
        g = torch.Generator().manual_seed(2)
        masks = [torch.randint(-2 ** 31, 2 ** 31, (batch, words), generator=g).int().to(DEV) for _ in range(steps)]
        runs = []
        for captured in (False, True):
            m = decoder.GPTQDecoder(cfg, batch=batch, device=DEV)
            mask = masks[0].clone()
            m.set_rules(decoder.LogitRules(repetition=1.2, frequency=[0.0, 0.3, -0.2], presence=0.5, bias={3: 2.0}, mask=mask))
            m.set_sampling(decoder.Sampling(temperature=[5.0, 1.0, 20.0], top_k=200, top_p=[0.9, 1.0, 0.99], seed=1))
            m.prefill(prompt_of(batch, 14))
            if captured:
                m.capture()
            out = []
            for k in masks:
                mask.copy_(k)
                out.append(m.decode(1).clone())
                for i in range(batch):        # what was drawn is what the grammar allows
                    t = int(m.tokens[i])
                    assert int(k[i, t // 32]) >> (t % 32) & 1
            runs.append((torch.cat(out), m.last_logits.float().clone(), [L.cache.k.clone() for L in m.layers]))
        assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
        # (the capture's warm-up steps ran past the prompt and were overwritten; rows behind the text are scratch)
        assert all(torch.equal(x[:, :, :14 + steps], y[:, :, :14 + steps]) for x, y in zip(runs[0][2], runs[1][2]))
    ops.check_status(DEV)


def test_refusals():
    for bad in (dict(cache_bits=8), dict(cache_bits=4, cache_group=128), dict(cache_bits=4, heads=8)):
        with pytest.raises(ValueError):
            decoder.GPTQDecoder(config(**bad), device=DEV)
    with pytest.raises(ValueError):
        decoder.GPTQDecoder(config(cache_bits=4), device=DEV, fused=False)
    m = decoder.GPTQDecoder(config(cache_bits=4), batch=2, device=DEV)
    with pytest.raises(ValueError):
        m.share_prefix(prompt_of(1, 5)[0])
    m.share_prefix(None)
    with pytest.raises(ValueError):
        m.prefill(prompt_of(2, 97))
    m.prefill(prompt_of(2, 90))
    with pytest.raises(ValueError):
        m.decode(7)
