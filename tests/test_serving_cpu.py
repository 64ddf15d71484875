"""Rules on logits as a request states them, without a GPU."""
import pytest
import torch

from autogptq.tvm_b200 import decoder


def test_rules_become_one_row_per_sequence():
    r = decoder.LogitRules(repetition=1.5, presence=[0.25, -1], bias=[{3: 1.0, 9: 2.0}, {}], mask=torch.ones(1, 4, dtype=torch.int32))
    a = r.arguments(2, 100, torch.device("cpu"))
    assert a["repetition"].tolist() == [1.5, 1.5] and a["presence"].tolist() == [0.25, -1] and "frequency" not in a
    assert a["bias_tokens"].tolist() == [[3, 9], [-1, -1]] and a["bias_values"].tolist() == [[1, 2], [0, 0]]
    assert a["mask"].shape == (1, 4)
    assert decoder.LogitRules(bias={}).arguments(1, 100, torch.device("cpu"))["bias_tokens"].tolist() == [[-1]]
    assert decoder.LogitRules().arguments(3, 100, torch.device("cpu")) == {}


@pytest.mark.parametrize("rules", [dict(repetition=0), dict(repetition=-1.0), dict(repetition=[1, 1, 1]), dict(frequency=float("inf")), dict(presence=[0.0, float("nan")]),
                                   dict(bias={100: 1.0}), dict(bias={-1: 1.0}), dict(bias=[{}]), dict(mask=torch.zeros(3, 4, dtype=torch.int32)),
                                   dict(mask=torch.zeros(2, 4))])
def test_refused_rules(rules):
    with pytest.raises(ValueError):
        decoder.LogitRules(**rules).arguments(2, 100, torch.device("cpu"))


@pytest.mark.parametrize("tokens", [torch.zeros(1, 3).long(), torch.zeros(3), torch.tensor([1, 100]), torch.tensor([-1, 5]), [1, 2]])
def test_refused_prefixes(tokens):
    with pytest.raises(ValueError):
        decoder.check_prefix(tokens, 100)


def test_prefixes():
    decoder.check_prefix(torch.tensor([0, 99, 5]), 100)
    decoder.check_prefix(torch.empty(0, dtype=torch.long), 100)


def bare(batch, **more):
    """A decoder without layers: what it checks before anything is computed."""
    cfg = decoder.DecoderConfig(layers=0, hidden=256, heads=4, inter=512, vocab=103, **{"max_seq": 96, **more})
    return decoder.GPTQDecoder(cfg, batch=batch, device="cpu")


@pytest.mark.parametrize("batch,shape", [(1, (2, 6)), (2, (1, 6)), (2, (3, 6)), (2, (6,)), (1, (1, 2, 3))])
def test_prompts_of_another_batch_are_refused(batch, shape):
    """The kernels write a row of the caches for each of the model's sequences."""
    with pytest.raises(ValueError, match="a prompt is"):
        bare(batch).prefill(torch.zeros(shape, dtype=torch.long))


@pytest.mark.parametrize("change", [dict(qkv=(6, 768)), dict(q=(1, 6, 4, 64)), dict(k=(2, 4, 10, 64), v=(1, 4, 10, 64)), dict(k=(2, 2, 10, 64), v=(2, 2, 10, 64)),
                                    dict(cos=(5, 32)), dict(sin=(5, 32))])
def test_rotary_embedding_of_a_prompt_takes_tensors_that_fit(change):
    from autogptq.tvm_b200 import ops
    t = {n: torch.zeros(s, dtype=torch.float16) for n, s in dict(dict(qkv=(12, 768), cos=(6, 32), sin=(6, 32), q=(2, 6, 4, 64), k=(2, 4, 10, 64),
                                                                      v=(2, 4, 10, 64)), **change).items()}
    with pytest.raises(ValueError, match="are not those of"):
        ops.rope_prompt(t["qkv"], t["cos"], t["sin"], t["q"], t["k"], t["v"], 6, 4, 64, True)


def test_a_prompt_too_long_behind_a_prefix_leaves_the_position():
    m = bare(1, max_seq=70000)
    m.prefix, m._pos_host = torch.zeros(3, dtype=torch.long), 5
    with pytest.raises(ValueError, match="65535"):
        m.prefill(torch.zeros(1, 65536, dtype=torch.long))
    assert m._pos_host == 5


@pytest.mark.parametrize("rules", [dict(repetition=1e-50), dict(repetition=1e50), dict(frequency=[0.0, -1e39]), dict(presence=1e300), dict(bias={3: float("nan")})])
def test_numbers_are_refused_as_32_bits_hold_them(rules):
    """A repetition of 1e-50 is above 0 and not infinite, but is divided by as 0."""
    with pytest.raises(ValueError):
        decoder.LogitRules(**rules).arguments(2, 100, torch.device("cpu"))


def test_biases_are_fp32_whatever_the_default_type():
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.float64)
        a = decoder.LogitRules(bias={1: 0.5, 2: float("-inf")}).arguments(1, 100, torch.device("cpu"))
    finally:
        torch.set_default_dtype(before)
    assert a["bias_values"].dtype == torch.float32 and a["bias_values"].tolist() == [[0.5, float("-inf")]]


def arguments(op):
    """(call, its tensors by name), of sizes that fit."""
    from autogptq.tvm_b200 import ops
    h = dict(dtype=torch.float16)
    if op == "logits":
        return ops.adjust_logits, dict(logits=torch.zeros(2, 40, **h), history=torch.zeros(2, 5).long(), lengths=torch.zeros(2).long(), repetition=torch.ones(2),
                                       frequency=torch.zeros(2), presence=torch.zeros(2), bias_tokens=torch.zeros(2, 3).long(), bias_values=torch.zeros(2, 3),
                                       out=torch.zeros(2, 40, **h))
    t = dict(q=torch.zeros(2, 1, 4, 64, **h), k_cache=torch.zeros(2, 2, 9, 64, **h), v_cache=torch.zeros(2, 2, 9, 64, **h), pos=torch.zeros(1).long(),
             out=torch.zeros(2, 1, 4, 64, **h))
    if op == "window":
        return lambda **kw: ops.attn_window(window=4, **kw), t
    return ops.attn_prefix, dict(t, k_prefix=torch.zeros(2, 7, 64, **h), v_prefix=torch.zeros(2, 7, 64, **h))


FLOATS = [(op, n) for op in ("logits", "window", "prefix") for n, t in arguments(op)[1].items() if t.is_floating_point()]


@pytest.mark.parametrize("op,name", FLOATS)
def test_a_gradient_is_never_dropped(op, name):
    """There is no backward pass: whichever tensor asks for one, penalties and biases too, is refused (before the device is looked at)."""
    call, t = arguments(op)
    t[name].requires_grad_()
    with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
        call(**t)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        call(**t)


@pytest.mark.parametrize("op,name", FLOATS)
def test_a_tangent_is_never_dropped(op, name):
    """A dual number of forward mode neither requires a gradient nor is a wrapper; no_grad does not switch its tangent off."""
    from torch.autograd import forward_ad
    call, t = arguments(op)
    plain = t[name]
    with forward_ad.dual_level():
        t[name] = forward_ad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
            call(**t)
        with torch.no_grad(), pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
            call(**t)
    t[name] = plain
    with pytest.raises(RuntimeError, match="CUDA"):
        call(**t)
