"""A cache held in 4 bits, attention over it, and sampling, as a list of cases with their inputs, cost and plain form.

* ``write``   new keys and values of a step or a prompt are rotated, quantised and packed into the cache, which also says what
              it now stands for: ``ops.cache_write``;
* ``read``    the cache back in 16 bits: ``ops.cache_read``;
* ``attn``    attention of single tokens, short runs and prompts over such a cache: ``ops.attn_cache``;
* ``sample``  the next token under temperature, top-k, top-p and min-p, from given random numbers: ``ops.sample``.

A cache row (one token, one key head) is ``hd / 2`` bytes and, for each group of ``group`` dims, a scale and a zero: a code c stands for
zero + scale c.  Within a row the dims lie as the tensor cores want them (``_order``).  ``run`` computes the plain form, or makes the package's
calls where ``own`` is set.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _named(name, **c):
    return dict(c, name=name) if name else c


def _write(name, B, T, heads, kv, hd, group, pos, spread, max_seq, rope=True, dtype="fp16", ragged=False):
    """``T`` new tokens for each of ``B`` sequences, the first of them at position ``pos`` (shortest text) to ``pos + spread``; with ``rope`` keys
    and queries are rotated on the way."""
    return _named(name, op="write", B=B, T=T, heads=heads, kv=kv, hd=hd, group=group, pos=pos, spread=spread, max_seq=max_seq, rope=rope,
                  dtype=dtype, ragged=ragged)


def _read(name, B, kv, hd, group, pos, spread, max_seq, dtype="fp16"):
    """The first ``pos`` to ``pos + spread`` rows of ``B`` sequences."""
    return _named(name, op="read", B=B, T=0, kv=kv, hd=hd, group=group, pos=pos, spread=spread, max_seq=max_seq, dtype=dtype, ragged=False)


def _attn(name, B, T, heads, kv, hd, group, pos, spread, max_seq, window=0, sinks=0, dtype="fp16", ragged=False):
    """As ``_write``, for the queries; ``window`` 0: all of the text before a token, else its last ``window`` positions and the first ``sinks``."""
    return _named(name, op="attn", B=B, T=T, heads=heads, kv=kv, hd=hd, group=group, pos=pos, spread=spread, max_seq=max_seq, window=window,
                  sinks=sinks, dtype=dtype, ragged=ragged)


def _sample(name, B, V, top_k, top_p, min_p, dtype="fp16", masked=False):
    """``B`` rows over a vocabulary of ``V``; ``top_k`` is the largest of the rows' (0: none has one)."""
    return _named(name, op="sample", B=B, V=V, top_k=top_k, top_p=top_p, min_p=min_p, dtype=dtype, masked=masked)


def listed():
    return [
        # One token of one sequence of the Llama-7B architecture: launch and latency.
        _write("write_b1_t1_h32", 1, 1, 32, 32, 128, 32, 700, 0, 768),
        # Three short prompts of unlike lengths, padded to the longest; narrow heads, positions learned elsewhere.
        _write("write_b3_t333_hd64", 3, 333, 12, 12, 64, 32, 0, 0, 400, False, "bf16", True),
        # A long prompt at once.
        _write("write_b1_t8192_h32kv8", 1, 8192, 32, 8, 128, 32, 0, 0, 8192),
        # One sequence of the Llama-7B architecture in the middle of its cache.
        _read("read_b1_kv32", 1, 32, 128, 32, 700, 0, 768),
        # Sixteen long texts with shared key heads, in larger groups.
        _read("read_b16_kv8_16384", 16, 8, 128, 64, 900, 15000, 16384),
        # A decode step of one sequence: latency.
        _attn("attn_decode_b1_h32", 1, 1, 32, 32, 128, 32, 700, 0, 768),
        # A decode step of sixteen long texts with shared key heads.
        _attn("attn_decode_b16_h32kv8", 16, 1, 32, 8, 128, 32, 900, 15000, 16384),
        # Short runs of tokens of unlike lengths; narrow heads, an odd window, larger groups.
        _attn("attn_run_b5_t5_hd64_w1000", 5, 5, 12, 4, 64, 64, 3, 2900, 3001, 1000, 5, "bf16", True),
        # The next 512 tokens of two long prompts, with the heads of an OPT-66B layer.
        _attn("attn_chunk_b2_t512_h72", 2, 512, 72, 72, 128, 32, 3500, 77, 4224),
        # One answer.
        _sample("sample_b1_v32000", 1, 32000, 50, 0.95, 0.0),
        # A batch with a request's own numbers for each row, some of them greedy, behind a grammar's mask; the vocabulary of OPT-66B.
        _sample("sample_b64_v50272", 64, 50272, 1000, 0.9, 0.02, "fp16", True),
        # A large batch over a vocabulary of odd size, logits in 32 bits, cut by top-p alone.
        _sample("sample_b128_v100003_fp32", 128, 100003, 0, 0.95, 0.0, "fp32"),
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
    dtype, hd, group = rng.choice(["fp16", "fp16", "bf16"]), rng.choice([64, 128, 128]), rng.choice([32, 32, 64])
    heads, kv = _draw_heads(rng)
    if kind < 0.2:
        T = _between(rng, 1, 4096)
        B = min(_between(rng, 1, 64), max(1, 12000000 // (T * (heads + 2 * kv) * hd)))
        pos = rng.choice([0, rng.randint(0, 500)])
        return _write(None, B, T, heads, kv, hd, group, pos, rng.choice([0, 31]), pos + T + 31 + rng.randint(0, 200), rng.random() < 0.7, dtype,
                      rng.random() < 0.4)
    if kind < 0.35:
        max_seq = _between(rng, 16, 16384)
        B = min(_between(rng, 1, 32), max(1, 120000000 // (kv * max_seq * hd)))
        pos = rng.randint(0, max_seq)
        return _read(None, B, kv, hd, group, pos, rng.randint(0, max_seq - pos), max_seq, dtype)
    window, sinks = rng.choice([(0, 0), (0, 0), (_between(rng, 1, 5000), rng.choice([0, 1, 4, 16, 130]))])
    if kind < 0.6:                             # a decode step
        max_seq = _between(rng, 64, 16384)
        B = min(_between(rng, 1, 48), max(1, 120000000 // (kv * max_seq * hd)))
        T = rng.choice([1, 1, 1, 1, 2, 5])
        pos = rng.randint(0, max_seq - T)
        return _attn(None, B, T, heads, kv, hd, group, pos, rng.randint(0, max_seq - T - pos), max_seq, window, sinks, dtype)
    if kind < 0.75:                            # a prompt or a chunk of one
        T, before = _between(rng, 6, 2000), rng.choice([0, 0, rng.randint(1, 2000)])
        B = min(rng.randint(1, 6), max(1, 20000000 // (heads * T * (T + before))))
        heads, kv = (heads, kv) if B * heads * T * (T + before) < 200000000 else (kv, kv) if B * kv * T * (T + before) < 200000000 else (1, 1)
        return _attn(None, B, T, heads, kv, hd, group, before, rng.choice([0, 0, 31]), before + T + 31 + rng.randint(0, 200), window, sinks, dtype,
                     rng.random() < 0.5)
    V = _between(rng, 1000, 100000)
    B = min(_between(rng, 1, 128), max(1, 10000000 // V))
    return _sample(None, B, V, rng.choice([0, 1, 40, _between(rng, 2, 5000)]), rng.choice([1.0, 0.95, 0.5]), rng.choice([0.0, 0.0, 0.05]),
                   rng.choice(["fp16", "bf16", "fp32"]), rng.random() < 0.5)


# ---- sizes that follow from a case alone -----------------------------------------------------------------------------------
def _positions(c):
    return [c["pos"] + c["spread"] * b // max(1, c["B"] - 1) for b in range(c["B"])]


def _counts(c):
    return [c["T"] - (b * 7919 % (c["T"] // 2 + 1) if c["ragged"] else 0) for b in range(c["B"])]


def _row_bytes(c):
    return c["hd"] // 2 + c["hd"] // c["group"] * 4


def work(case):
    c = case
    if c["op"] == "sample":
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": c["B"] * (c["V"] * size + 32), "flops": 2 * c["B"] * c["V"]}
    row = c["hd"] * 2
    if c["op"] == "read":
        rows = sum(_positions(c)) * c["kv"] * 2
        return {"bytes": rows * (_row_bytes(c) + row), "flops": 2 * rows * c["hd"]}
    tokens = sum(_counts(c))
    if c["op"] == "write":                     # keys and values in, their codes and what these stand for out; queries in and out; angles
        rows = tokens * c["kv"] * 2
        turned = (2 * tokens * c["heads"] * row + c["T"] * row) if c["rope"] else 0
        return {"bytes": rows * (2 * row + _row_bytes(c)) + turned, "flops": rows * c["hd"] * 6 + (tokens * c["heads"] * c["hd"] * 3 if c["rope"] else 0)}
    pairs = keys = 0
    for p, n in zip(_positions(c), _counts(c)):
        W, S = c["window"] or p + n, c["sinks"]
        first = max(0, p - W + 1)
        pairs += sum(min(W, i + 1) + min(S, max(0, i + 1 - W)) for i in range(p, p + n))
        keys += p + n - first + min(S, first)
    return {"bytes": 2 * tokens * c["heads"] * row + 2 * keys * c["kv"] * _row_bytes(c), "flops": 4 * c["hd"] * c["heads"] * pairs}


# ---- the format ------------------------------------------------------------------------------------------------------------
def _order(hd):
    """The dim of each code of a row, in the order of the row's bytes, the lower four bits of a byte first."""
    W, dims = hd // 64, []
    for word in range(hd // 8):
        a = 64 * (word % W) + 4 * (word // W)
        dims += [a, a + 2, a + 32, a + 34, a + 1, a + 3, a + 33, a + 35]
    return dims


def _quantise(x, group):
    """(codes uint8, constants [..., groups, 2]) of rows ``x`` [..., hd] in a 16-bit type."""
    g = x.float().reshape(*x.shape[:-1], -1, group)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).to(x.dtype).float()
    codes = torch.where(scale > 0, ((g - lo) / scale).round_().clamp_(0, 15), 0.0).to(torch.uint8)
    return codes.reshape(x.shape), torch.cat([scale, lo], -1).to(x.dtype)


def _packed(codes):
    c = codes[..., _order(codes.shape[-1])]
    return c[..., 0::2] | c[..., 1::2] << 4


def _values(packed, constants):
    """What a cache stands for, in 32 bits."""
    hd = packed.shape[-1] * 2
    codes = torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], hd)
    back = [0] * hd
    for place, dim in enumerate(_order(hd)):
        back[dim] = place
    g = codes[..., back].float().reshape(*constants.shape[:-1], -1)
    return (g * constants[..., :1].float() + constants[..., 1:].float()).reshape(*packed.shape[:-1], hd)


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[c["dtype"]]
    if c["op"] == "sample":
        return _prepare_sample(c, g, t, dev)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=t)

    B, T, kv, hd, S = c["B"], c["T"], c["kv"], c["hd"], c["max_seq"]
    s = {"op": c["op"], "group": c["group"]}
    if c["op"] == "write":
        cache = (torch.zeros(B, kv, S, hd // 2, dtype=torch.uint8, device=dev), torch.zeros(B, kv, S, hd // c["group"], 2, dtype=t, device=dev))
        cache += tuple(torch.zeros_like(x) for x in cache)
        # q|k|v as one linear leaves them; some dims of the keys are larger than the others
        heads = c["heads"]
        x = rand(B, T, heads + 2 * kv, hd)
        x[:, :, heads:heads + kv] *= 1 + 4 * (torch.rand(hd, generator=g, device=dev) > 0.95)
        s["q"], s["k"], s["v"] = x[:, :, :heads], x[:, :, heads:heads + kv], x[:, :, heads + kv:]
        s["k_out"], s["v_out"] = torch.zeros(B, kv, T, hd, dtype=t, device=dev), torch.zeros(B, kv, T, hd, dtype=t, device=dev)
        s["q_out"] = s["cos"] = s["sin"] = None
        if c["rope"]:
            angle = torch.arange(S, device=dev)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, device=dev).double() / hd)
            s["cos"], s["sin"] = angle.cos().to(t), angle.sin().to(t)
            s["q_out"] = torch.zeros(B, T, heads, hd, dtype=t, device=dev)
        else:
            s["q"] = None
    else:
        # the first keys lie along the queries' common direction: these collect a large share of the softmax
        k, v = rand(B, kv, S, hd), rand(B, kv, S, hd)
        if c["op"] == "attn":
            s["q"] = rand(B, T, c["heads"], hd) * 1.5 + 0.5
            k[:, :, :4] += 12.0 / hd ** 0.5
            s["window"], s["sinks"], s["keys"] = c["window"], c["sinks"], max(_positions(c)) + T
            s["out"] = torch.zeros_like(s["q"]) if c["ragged"] else None
        else:
            s["k_out"], s["v_out"] = torch.zeros_like(k), torch.zeros_like(v)
        cache = ()
        for x in (k, v):
            codes, constants = _quantise(x, c["group"])
            cache += (_packed(codes), constants)
    s["cache"] = cache                         # codes and constants of the keys, codes and constants of the values
    s["pos"] = torch.tensor(_positions(c), device=dev)
    s["counts"] = torch.tensor(_counts(c), device=dev) if c["ragged"] else None
    if own:
        from autogptq.tvm_b200 import ops
        s["handle"] = ops.QuantCache(cache[0], cache[2], cache[1], cache[3])
    return s


def _prepare_sample(c, g, t, dev):
    B, V = c["B"], c["V"]
    x = 3 * torch.randn(B, V, generator=g, device=dev)
    if c["masked"]:
        x.masked_fill_(torch.rand(B, V, generator=g, device=dev) < 0.5, -math.inf)
        x[:, 0] = 0
    s = {"op": "sample", "logits": x.to(t), "uniform": torch.rand(B, generator=g, device=dev)}
    row = torch.arange(B, device=dev)
    s["temperature"] = 0.6 + 0.6 * torch.rand(B, generator=g, device=dev)
    if B > 1:
        s["temperature"][row % 5 == 3] = 0      # greedy
    s["top_k"] = torch.where(row % 3 == 2, 0, (c["top_k"] - row * c["top_k"] // (2 * B)).clamp(min=1)) if c["top_k"] else None
    s["top_p"] = torch.full((B,), c["top_p"], device=dev) - 0.1 * torch.rand(B, generator=g, device=dev) if c["top_p"] < 1 else None
    s["min_p"] = torch.full((B,), c["min_p"], device=dev) if c["min_p"] > 0 else None
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from autogptq.tvm_b200 import ops
        if s["op"] == "write":
            ops.cache_write(s["handle"], s["k"], s["v"], s["pos"], counts=s["counts"], cos=s["cos"], sin=s["sin"], q=s["q"], q_out=s["q_out"],
                            k_out=s["k_out"].transpose(1, 2), v_out=s["v_out"].transpose(1, 2))
            return [x for x in (s["k_out"], s["v_out"], s["q_out"]) if x is not None]
        if s["op"] == "read":
            return ops.cache_read(s["handle"], lengths=s["pos"], k_out=s["k_out"], v_out=s["v_out"])
        if s["op"] == "attn":
            return ops.attn_cache(s["q"], s["handle"], s["pos"], window=s["window"] or None, sinks=s["sinks"], counts=s["counts"], out=s["out"])
        return ops.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn, "sample": _plain_sample}[s["op"]](s)


def _plain_write(s):
    (B, T, kv, hd), max_seq = s["k"].shape, s["cache"][0].shape[2]
    at = s["pos"][:, None] + torch.arange(T, device=s["k"].device)             # [B, T]
    there = at < max_seq if s["counts"] is None else torch.arange(T, device=at.device) < s["counts"][:, None]
    b, t = there.nonzero(as_tuple=True)
    place = at[b, t]

    def turned(x):
        x = x[b, t].float()
        if s["cos"] is None:
            return x
        cos, sin = s["cos"][place].float()[:, None], s["sin"][place].float()[:, None]
        return torch.stack([x[..., 0::2] * cos - x[..., 1::2] * sin, x[..., 0::2] * sin + x[..., 1::2] * cos], -1).flatten(-2)

    for x, out, codes_of, constants_of in ((turned(s["k"]), s["k_out"], *s["cache"][:2]), (s["v"][b, t], s["v_out"], *s["cache"][2:])):
        codes, constants = _quantise(x.to(s["k"].dtype), s["group"])
        packed = _packed(codes)
        codes_of[b, :, place], constants_of[b, :, place] = packed, constants
        out[b, :, t] = _values(packed, constants).to(out.dtype)
    if s["q"] is None:
        return [s["k_out"], s["v_out"]]
    s["q_out"][b, t] = turned(s["q"]).to(s["q_out"].dtype)
    return [s["k_out"], s["v_out"], s["q_out"]]


def _plain_read(s):
    there = (torch.arange(s["k_out"].shape[2], device=s["pos"].device) < s["pos"][:, None])[:, None, :, None]
    for out, i in ((s["k_out"], 0), (s["v_out"], 2)):
        torch.where(there, _values(*s["cache"][i:i + 2]).to(out.dtype), out, out=out)
    return s["k_out"], s["v_out"]


def _plain_attn(s):
    q, B, T = s["q"].float(), s["q"].shape[0], s["q"].shape[1]
    N = s["keys"]
    k, v = (_values(s["cache"][i][:, :, :N], s["cache"][i + 1][:, :, :N]) for i in (0, 2))
    heads, hd, kv = q.shape[2], q.shape[3], k.shape[1]
    G = heads // kv
    q = q.reshape(B, T, kv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, G * T, hd) * hd ** -0.5
    at = (s["pos"][:, None] + torch.arange(T, device=q.device))[:, :, None]              # position of each query
    j = torch.arange(N, device=q.device)
    hidden = j > at
    if s["window"]:
        hidden = hidden | ((j <= at - s["window"]) & (j >= s["sinks"]))
    scores = (q @ k.transpose(2, 3)).reshape(B, kv, G, T, N).masked_fill_(hidden[:, None, None], -math.inf).reshape(B, kv, G * T, N)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = (scores @ v / scores.sum(-1, keepdim=True)).reshape(B, kv, G, T, hd).permute(0, 3, 1, 2, 4).reshape(B, T, heads, hd).to(s["q"].dtype)
    if s["counts"] is not None:
        out = torch.where((torch.arange(T, device=q.device) < s["counts"][:, None])[:, :, None, None], out, s["out"])
    return out


def _plain_sample(s):
    """In 64 bits: sums over the vocabulary decide which token comes next."""
    x = s["logits"].double()
    B, V = x.shape
    cold = s["temperature"] == 0
    w = ((x - x.amax(1, keepdim=True)) / torch.where(cold, 1.0, s["temperature"].double())[:, None]).exp_()
    w, token = torch.sort(torch.where(cold[:, None], (x == x.amax(1, keepdim=True)).double(), w), dim=1, descending=True, stable=True)
    rank = torch.arange(V, device=x.device)
    kept = rank < torch.where(cold, 1, V)[:, None]
    if s["top_k"] is not None:
        kept &= (rank < s["top_k"][:, None]) | (s["top_k"] <= 0)[:, None]
    if s["top_p"] is not None:
        mass = w * kept
        before = mass.cumsum(1) - mass
        kept &= (before < s["top_p"].double()[:, None] * mass.sum(1, keepdim=True)) | (rank == 0)
    if s["min_p"] is not None:
        kept &= (w >= s["min_p"].double()[:, None]) | (rank == 0)
    mass = torch.zeros_like(w).scatter_(1, token, w * kept).cumsum(1)          # in the vocabulary's order
    return (mass <= s["uniform"].double()[:, None] * mass[:, -1:]).sum(1)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attn": _exact_attn, "sample": _exact_sample}[c["op"]](c, s)


def _exact_rows(codes, constants, hd):
    """Rows [n, hd / 2] and their constants in 64 bits: the word, half and place of each dim."""
    d = torch.arange(hd, device=codes.device)
    word = (d % 32) // 4 * (hd // 64) + d // 64
    nibble = (d % 2) * 4 + (d % 4) // 2 + (d % 64) // 32 * 2
    byte = codes[:, word * 4 + nibble // 2].long()
    c = torch.where(nibble % 2 == 1, byte // 16, byte % 16).double()
    group = d // (hd // constants.shape[1])
    return constants[:, group, 1].double() + c * constants[:, group, 0].double()


def _exact_write(c, s):
    kv, hd, n_groups = c["kv"], c["hd"], c["hd"] // c["group"]
    outs = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (s["k_out"], s["v_out"])]
    q_out = torch.zeros(s["q_out"].shape, dtype=torch.float64, device="cuda") if c["rope"] else None
    for b, (p, n) in enumerate(zip(_positions(c), _counts(c))):
        def turned(x):
            x = x.double()
            if not c["rope"]:
                return x
            z = torch.view_as_complex(x.reshape(*x.shape[:-1], hd // 2, 2))
            z = z * torch.complex(s["cos"][p:p + n].double(), s["sin"][p:p + n].double())[:, None]
            return torch.view_as_real(z).reshape(x.shape)

        if c["rope"]:
            q_out[b, :n] = turned(s["q"][b, :n])
        for x, out in ((turned(s["k"][b, :n]).to(s["k"].dtype), outs[0]), (s["v"][b, :n], outs[1])):
            x = x.double()
            for i in range(n_groups):
                g = x[..., i * c["group"]:(i + 1) * c["group"]]
                lo = g.min(-1, keepdim=True).values
                step = ((g.max(-1, keepdim=True).values - lo) / 15).to(s["k"].dtype).double()
                code = torch.clamp(torch.round((g - lo) / step.masked_fill(step == 0, 1)), max=15)
                out[b, :, :n, i * c["group"]:(i + 1) * c["group"]] = (lo + step * code).transpose(0, 1)
    return outs + ([q_out] if c["rope"] else [])


def _exact_read(c, s):
    outs = [torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
    for i, out in enumerate(outs):
        for b, n in enumerate(_positions(c)):
            for h in range(c["kv"]):
                out[b, h, :n] = _exact_rows(s["cache"][2 * i][b, h, :n], s["cache"][2 * i + 1][b, h, :n], c["hd"])
    return tuple(outs)


def _exact_attn(c, s):
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    G = heads // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (p, n) in enumerate(zip(_positions(c), _counts(c))):
        query = torch.arange(p, p + n, device="cuda")[:, None]
        key = torch.arange(p + n, device="cuda")[None]
        sees = key <= query
        if c["window"]:
            sees = sees & ((query - key < c["window"]) | (key < c["sinks"]))
        for h in range(kv):
            K, W = (_exact_rows(s["cache"][i][b, h, :p + n], s["cache"][i + 1][b, h, :p + n], hd) for i in (0, 2))
            for i in range(h * G, h * G + G):
                a = torch.einsum("td,nd->tn", s["q"][b, :n, i].double(), K) / math.sqrt(hd)
                a = torch.softmax(a.where(sees, torch.tensor(-math.inf, dtype=torch.float64, device="cuda")), 1)
                out[b, :n, i] = a @ W
    return out


def _exact_sample(c, s):
    """Row by row: the number of tokens kept, then the first token at which the kept ones' sum passes the random number's share of it."""
    out = []
    numbers = {k: None if s[k] is None else s[k].tolist() for k in ("uniform", "temperature", "top_k", "top_p", "min_p")}
    for b in range(c["B"]):
        x = s["logits"][b].double()
        t = numbers["temperature"][b]
        if t == 0:
            out.append(int((x == x.max()).nonzero()[0]))
            continue
        w = torch.softmax(x / t, 0)
        order = torch.argsort(-x, stable=True)
        n = c["V"]
        if numbers["top_k"] and numbers["top_k"][b] > 0:
            n = min(n, numbers["top_k"][b])
        if numbers["top_p"]:
            sums = torch.cumsum(w[order[:n]], 0)
            n = min(n, 1 + int((sums < numbers["top_p"][b] * sums[-1]).sum()))
        if numbers["min_p"]:
            n = max(1, min(n, int((w[order[:n]] >= numbers["min_p"][b] * w.max()).sum())))
        chosen = torch.sort(order[:n]).values
        sums = torch.cumsum(w[chosen], 0)
        at = torch.searchsorted(sums, torch.tensor([numbers["uniform"][b]], dtype=torch.float64, device="cuda") * sums[-1], right=True)
        out.append(int(chosen[min(int(at), n - 1)]))
    return torch.tensor(out, device="cuda")
