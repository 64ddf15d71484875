"""Serving operators of a decoder beside its linears, as a list of cases with their inputs, cost and plain form.

* ``window``  attention whose queries see the last ``window`` positions and the first ``sinks``: ``ops.attn_window``, for the
              single tokens of a decode step and for prompts or chunks of them;
* ``prefix``  attention of a batch whose texts begin alike: the keys and values of the common part are held once
              (``ops.attn_prefix``), the rest in each sequence's own cache; single tokens and the prompts that follow the common part;
* ``logits``  penalties for repeated tokens, biases and grammar masks on the logits before the pick: ``ops.adjust_logits``.

``run`` computes the plain form in 32 bits, or makes the package's calls where ``own`` is set.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _window(name, B, T, heads, kv, hd, pos, spread, max_seq, window, sinks, dtype="fp16", ragged=False):
    """``T`` new tokens for each of ``B`` sequences, the first of them at position ``pos`` (shortest text) to ``pos + spread``."""
    c = dict(op="window", B=B, T=T, heads=heads, kv=kv, hd=hd, pos=pos, spread=spread, max_seq=max_seq, window=window, sinks=sinks,
             dtype=dtype, ragged=ragged)
    return dict(c, name=name) if name else c


def _prefix(name, B, T, heads, kv, hd, prefix, pos, spread, max_seq, dtype="fp16", ragged=False):
    """``T`` new tokens for each of ``B`` sequences behind ``prefix`` common ones and ``pos`` to ``pos + spread`` of their own."""
    c = dict(op="prefix", B=B, T=T, heads=heads, kv=kv, hd=hd, prefix=prefix, pos=pos, spread=spread, max_seq=max_seq, dtype=dtype,
             ragged=ragged)
    return dict(c, name=name) if name else c


def _logits(name, B, V, history, bias, mask, dtype="fp16"):
    """``B`` rows over a vocabulary of ``V``, up to ``history`` tokens each so far, ``bias`` biased tokens per row."""
    c = dict(op="logits", B=B, V=V, history=history, bias=bias, mask=mask, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One sequence of the Llama-7B architecture in the middle of its cache, one token: launch and latency.
        _window("window_decode_b1_h32_w512", 1, 1, 32, 32, 128, 700, 0, 768, 512, 4),
        # A decode step of sixteen long texts with shared key heads.
        _window("window_decode_b16_h32kv8_w4096", 16, 1, 32, 8, 128, 900, 15000, 16384, 4096, 4),
        # Three short prompts of unlike lengths, padded to the longest; narrow heads, an odd window.
        _window("window_prompt_b3_t333_hd64_w100", 3, 333, 12, 12, 64, 0, 0, 400, 100, 5, "bf16", True),
        # The next 512 tokens of two long prompts, with the heads of an OPT-66B layer.
        _window("window_chunk_b2_t512_h72_w1024", 2, 512, 72, 72, 128, 3500, 77, 4224, 1024, 4),
        # A long prompt at once.
        _window("window_prompt_b1_t8192_h32kv8_w4096", 1, 8192, 32, 8, 128, 0, 0, 8192, 4096, 4),
        # Four answers to one short instruction, one token each: latency.
        _prefix("prefix_decode_b4_p500", 4, 1, 32, 32, 128, 500, 20, 9, 256),
        # A decode step of 32 requests behind a long system text, shared key heads.
        _prefix("prefix_decode_b32_h32kv8_p8192", 32, 1, 32, 8, 128, 8192, 17, 480, 640),
        # 64 continuations of one document, the Llama-7B head layout.
        _prefix("prefix_decode_b64_h32_p16384", 64, 1, 32, 32, 128, 16384, 1, 250, 256),
        # Five questions of unlike lengths about one text, as prompts; narrow heads.
        _prefix("prefix_prompt_b5_t203_hd64_p2011", 5, 203, 12, 4, 64, 2011, 0, 0, 256, "bf16", True),
        # One answer with a penalty for repetition.
        _logits("logits_b1_v32000", 1, 32000, 768, 0, False),
        # A batch with biases and a grammar each, the vocabulary of OPT-66B.
        _logits("logits_b64_v50272_mask", 64, 50272, 2048, 300, True),
        # A large batch over a vocabulary of odd size, long texts, logits in 32 bits.
        _logits("logits_b128_v100003_fp32", 128, 100003, 4096, 17, True, "fp32"),
    ]


def _between(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng):
    kv = rng.choice([1, 2, 4, 8, 12, 32])
    group = rng.choice([1, 1, 2, 4, 7, 8])
    return min(kv * group, 40) // kv * kv, kv


def draw(rng):
    """Costs are held below those of the largest listed case of the same kind."""
    kind = rng.random()
    dtype, hd = rng.choice(["fp16", "fp16", "bf16"]), rng.choice([64, 128, 128])
    if kind < 0.25:                            # a decode step, window
        heads, kv = _draw_heads(rng)
        window = _between(rng, 1, 4096)
        max_seq = _between(rng, 64, 16384)
        B = min(_between(rng, 1, 48), max(1, (1 << 31) // (kv * max_seq * hd * 4)), max(1, 600000 // (kv * min(window, max_seq))))
        T = rng.choice([1, 1, 1, 1, 2, 5])
        pos = rng.randint(0, max_seq - T)
        return _window(None, B, min(T, max_seq), heads, kv, hd, pos, rng.randint(0, max_seq - T - pos), max_seq, window, rng.choice([0, 1, 4, 4, 16, 130]), dtype)
    if kind < 0.45:                            # a prompt or a chunk of one, window
        heads, kv = _draw_heads(rng)
        T = _between(rng, 2, 4000)
        B = min(rng.randint(1, 6), max(1, 80000000 // (heads * T * T)))
        before = rng.choice([0, 0, rng.randint(1, 2000)])
        heads, kv = (heads, kv) if heads * T * (T + before) < 1 << 29 else (kv, kv) if kv * T * (T + before) < 1 << 29 else (1, 1)
        return _window(None, B, T, heads, kv, hd, before, rng.choice([0, 0, 31]), before + T + 31 + rng.randint(0, 200),
                       _between(rng, 1, 5000), rng.choice([0, 1, 4, 4, 16, 130]), dtype, rng.random() < 0.5)
    if kind < 0.65:                            # a decode step behind a common part
        heads, kv = _draw_heads(rng)
        P = _between(rng, 1, 16384)
        max_seq = _between(rng, 8, 1024)
        B = min(_between(rng, 1, 96), max(1, 400000 // (kv * max_seq)))
        T = rng.choice([1, 1, 1, 1, 2, 5])
        pos = rng.randint(0, max_seq - T)
        return _prefix(None, B, T, heads, kv, hd, P, pos, rng.randint(0, max_seq - T - pos), max_seq, dtype)
    if kind < 0.75:                            # prompts behind a common part
        heads, kv = _draw_heads(rng)
        T, B, P = _between(rng, 6, 600), rng.randint(1, 8), _between(rng, 1, 6000)
        heads, kv = (heads, kv) if B * heads * T * (T + P) < 1 << 28 else (kv, kv) if B * kv * T * (T + P) < 1 << 28 else (1, 1)
        return _prefix(None, B, T, heads, kv, hd, P, 0, 0, T + rng.randint(0, 100), dtype, rng.random() < 0.5)
    V = _between(rng, 1000, 100000)
    B = min(_between(rng, 1, 128), max(1, 10000000 // V))
    return _logits(None, B, V, _between(rng, 1, 4096), rng.choice([0, 1, 30, 300]), rng.random() < 0.5, rng.choice(["fp16", "bf16", "fp32"]))


# ---- sizes that follow from a case alone -----------------------------------------------------------------------------------
def _positions(c):
    return [c["pos"] + c["spread"] * b // max(1, c["B"] - 1) for b in range(c["B"])]


def _counts(c):
    return [c["T"] - (b * 7919 % (c["T"] // 2 + 1) if c["ragged"] else 0) for b in range(c["B"])]


def _visible(c):
    """Per sequence (query-key pairs, keys that any query sees) of its own cache, for one head."""
    out = []
    for p, n in zip(_positions(c), _counts(c)):
        if c["op"] == "prefix":
            out.append((n * (p + 1) + n * (n - 1) // 2, p + n))
            continue
        W, S = c["window"], c["sinks"]
        first = max(0, p - W + 1)
        pairs = sum(min(W, i + 1) + min(S, max(0, i + 1 - W)) for i in range(p, p + n))
        out.append((pairs, p + n - first + min(S, first)))
    return out


def work(case):
    c = case
    if c["op"] == "logits":
        size = 4 if c["dtype"] == "fp32" else 2
        rows = 2 * c["V"] * size + sum(_lengths(c)) * 8 / c["B"] + c["bias"] * 12 + (math.ceil(c["V"] / 32) * 4 if c["mask"] else 0)
        return {"bytes": c["B"] * rows, "flops": c["B"] * c["V"]}
    seen, tokens = _visible(c), sum(_counts(c))
    per_key = 2 * c["kv"] * c["hd"] * 2
    P = c.get("prefix", 0)
    return {"bytes": 2 * tokens * c["heads"] * c["hd"] * 2 + per_key * (P + sum(k for _, k in seen)),
            "flops": 4 * c["hd"] * c["heads"] * (P * tokens + sum(n for n, _ in seen))}


def _lengths(c):
    L = c["history"]
    return [L - (L // 2) * b // max(1, c["B"] - 1) if c["B"] > 1 else L for b in range(c["B"])]


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[c["dtype"]]
    if c["op"] == "logits":
        return _prepare_logits(c, g, t, dev)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=t)

    B, T, heads, kv, hd = c["B"], c["T"], c["heads"], c["kv"], c["hd"]
    s = {"op": c["op"], "keys": max(_positions(c)) + T}
    # queries have a direction in common, and the first keys lie along it: these collect a large share of the softmax
    s["q"] = rand(B, T, heads, hd) * 1.5 + 0.5
    s["k"], s["v"] = rand(B, kv, c["max_seq"], hd), rand(B, kv, c["max_seq"], hd)
    s["pos"] = torch.tensor(_positions(c), device=dev)
    s["counts"] = torch.tensor(_counts(c), device=dev) if c["ragged"] else None
    s["out"] = torch.zeros_like(s["q"]) if c["ragged"] else None
    first = 12.0 / hd ** 0.5
    if c["op"] == "window":
        s["window"], s["sinks"] = c["window"], c["sinks"]
        s["k"][:, :, :c["sinks"]] += first
    else:
        s["kp"], s["vp"] = rand(kv, c["prefix"], hd), rand(kv, c["prefix"], hd)
        s["kp"][:, :2] += first
    return s


def _prepare_logits(c, g, t, dev):
    B, V, L = c["B"], c["V"], c["history"]
    s = {"op": "logits", "logits": (3 * torch.randn(B, V, generator=g, device=dev)).to(t)}
    # a text repeats its common tokens
    s["history"] = (V * torch.rand(B, L, generator=g, device=dev) ** 3).long().clamp_(max=V - 1)
    s["lengths"] = torch.tensor(_lengths(c), device=dev)
    s["prompt_lens"] = s["lengths"] // 3
    s["repetition"] = 1 + 0.3 * torch.rand(B, generator=g, device=dev)
    s["frequency"] = 0.5 * torch.rand(B, generator=g, device=dev)
    s["presence"] = 0.5 * torch.rand(B, generator=g, device=dev)
    s["bias_tokens"] = s["bias_values"] = s["mask"] = None
    if c["bias"]:
        s["bias_tokens"] = torch.randint(0, V, (B, c["bias"]), generator=g, device=dev)
        s["bias_values"] = 5 * torch.randn(B, c["bias"], generator=g, device=dev)
    if c["mask"]:
        words = [torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g, device=dev) for _ in range(2)]
        s["mask"] = (words[0] & words[1]).to(torch.int32)       # a quarter of the tokens may come next
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from autogptq.tvm_b200 import ops
        if s["op"] == "window":
            return ops.attn_window(s["q"], s["k"], s["v"], s["pos"], s["window"], s["sinks"], counts=s["counts"], out=s["out"])
        if s["op"] == "prefix":
            return ops.attn_prefix(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["pos"], counts=s["counts"], out=s["out"])
        return ops.adjust_logits(s["logits"], s["history"], s["lengths"], prompt_lens=s["prompt_lens"], repetition=s["repetition"],
                                 frequency=s["frequency"], presence=s["presence"], bias_tokens=s["bias_tokens"],
                                 bias_values=s["bias_values"], mask=s["mask"])
    return _plain_logits(s) if s["op"] == "logits" else _plain_attention(s)


def _plain_attention(s):
    q, B, T = s["q"].float(), s["q"].shape[0], s["q"].shape[1]
    heads, hd, kv = q.shape[2], q.shape[3], s["k"].shape[1]
    G, N = heads // kv, s["keys"]
    q = q.reshape(B, T, kv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, G * T, hd) * hd ** -0.5
    k, v = s["k"][:, :, :N].float(), s["v"][:, :, :N].float()
    at = (s["pos"][:, None] + torch.arange(T, device=q.device))[:, :, None]              # position of each query
    j = torch.arange(N, device=q.device)
    hidden = j > at
    if s["op"] == "window":
        hidden = hidden | ((j <= at - s["window"]) & (j >= s["sinks"]))
    scores = (q @ k.transpose(2, 3)).reshape(B, kv, G, T, N).masked_fill_(hidden[:, None, None], -math.inf).reshape(B, kv, G * T, N)
    top = scores.amax(-1, keepdim=True)
    if s["op"] == "prefix":
        P = s["kp"].shape[1]
        rows = q.transpose(0, 1).reshape(kv, B * G * T, hd)
        front = (rows @ s["kp"].float().transpose(1, 2)).reshape(kv, B, G * T, P).transpose(0, 1)
        top = torch.maximum(top, front.amax(-1, keepdim=True))
        front = front.sub(top).exp_()
    scores = scores.sub_(top).exp_()
    total, mixed = scores.sum(-1, keepdim=True), scores @ v
    if s["op"] == "prefix":
        total = total + front.sum(-1, keepdim=True)
        front = front.transpose(0, 1).reshape(kv, B * G * T, P) @ s["vp"].float()
        mixed = mixed + front.reshape(kv, B, G * T, hd).transpose(0, 1)
    out = (mixed / total).reshape(B, kv, G, T, hd).permute(0, 3, 1, 2, 4).reshape(B, T, heads, hd).to(s["q"].dtype)
    if s["counts"] is not None:
        out = torch.where((torch.arange(T, device=q.device) < s["counts"][:, None])[:, :, None, None], out, s["out"])
    return out


def _plain_logits(s):
    x, V, tokens = s["logits"].float(), s["logits"].shape[1], s["history"]
    at = torch.arange(tokens.shape[1], device=x.device)
    used = at < s["lengths"][:, None]
    made = used & (at >= s["prompt_lens"][:, None])
    seen = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, tokens, used.int()) > 0
    count = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, tokens, made.int())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_tokens"] is not None:                # of several values for one token the last one counts
        entry = torch.arange(s["bias_tokens"].shape[1], device=x.device).expand_as(s["bias_tokens"])
        last = torch.full(x.shape, -1, device=x.device).scatter_reduce_(1, s["bias_tokens"], entry, "amax")
        x = x + torch.where(last >= 0, s["bias_values"].gather(1, last.clamp(min=0)), 0.0)
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=x.device)) & 1
        x = x.masked_fill(bits.reshape(x.shape[0], -1)[:, :V] == 0, -math.inf)
    return x.to(s["logits"].dtype)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "logits":
        return _exact_logits(c, s)
    B, heads, kv, hd = c["B"], c["heads"], c["kv"], c["hd"]
    G = heads // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (p, n) in enumerate(zip(_positions(c), _counts(c))):
        query = torch.arange(p, p + n, device="cuda")[:, None]
        key = torch.arange(p + n, device="cuda")[None]
        sees = key <= query
        if c["op"] == "window":
            sees = sees & ((query - key < c["window"]) | (key < c["sinks"]))
        for h in range(kv):
            K, W = s["k"][b, h, :p + n].double(), s["v"][b, h, :p + n].double()
            sight = sees
            if c["op"] == "prefix":
                K, W = torch.cat([s["kp"][h].double(), K]), torch.cat([s["vp"][h].double(), W])
                sight = torch.cat([torch.ones(n, c["prefix"], dtype=torch.bool, device="cuda"), sees], 1)
            for i in range(h * G, h * G + G):
                a = torch.einsum("td,nd->tn", s["q"][b, :n, i].double(), K) / math.sqrt(hd)
                a = torch.softmax(a.where(sight, torch.tensor(-math.inf, dtype=torch.float64, device="cuda")), 1)
                out[b, :n, i] = a @ W
    return out


def _exact_logits(c, s):
    out = s["logits"].double()
    V = c["V"]
    for b, n in enumerate(_lengths(c)):
        row, m = out[b], n // 3
        seen = torch.bincount(s["history"][b, :n], minlength=V) > 0
        made = torch.bincount(s["history"][b, m:n], minlength=V).double()
        r = s["repetition"][b].double()
        row = torch.where(seen, row * torch.where(row > 0, 1 / r, r), row)
        row = row - made * s["frequency"][b].double() - made.clamp(max=1) * s["presence"][b].double()
        if c["bias"]:
            chosen = dict(zip(s["bias_tokens"][b].tolist(), s["bias_values"][b].double().tolist()))
            row[torch.tensor(list(chosen), device="cuda")] += torch.tensor(list(chosen.values()), dtype=torch.float64, device="cuda")
        if c["mask"]:
            token = torch.arange(V, device="cuda")
            allowed = torch.bitwise_and(torch.bitwise_right_shift(s["mask"][b].long()[token // 32], token % 32), 1)
            row[allowed == 0] = -math.inf
        out[b] = row
    return out
