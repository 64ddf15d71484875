"""Sampling as a request states it, without a GPU."""
import math

import pytest
import torch

from autogptq.tvm_b200 import decoder


def test_numbers_become_one_row_per_sequence():
    a = decoder.Sampling(temperature=[0.0, 1.5], top_k=40, min_p=[0, 0.5]).arguments(2, torch.device("cpu"))
    assert a["temperature"].tolist() == [0.0, 1.5] and a["top_k"].tolist() == [40, 40] and a["min_p"].tolist() == [0, 0.5] and "top_p" not in a
    assert a["top_k"].dtype == torch.int64 and a["temperature"].dtype == a["min_p"].dtype == torch.float32
    assert list(decoder.Sampling().arguments(3, torch.device("cpu"))) == ["temperature"]


@pytest.mark.parametrize("numbers", [dict(temperature=-1), dict(temperature=math.nan), dict(temperature=math.inf), dict(temperature=1e39), dict(temperature=[1.0]),
                                     dict(top_k=-1), dict(top_k=1.5), dict(top_k=[1, 2, 3]), dict(top_p=1.1), dict(top_p=-0.1), dict(top_p=math.nan), dict(min_p=2.0),
                                     dict(min_p=[0.1, -0.1])])
def test_refused_numbers(numbers):
    with pytest.raises(ValueError):
        decoder.Sampling(**numbers).arguments(2, torch.device("cpu"))


def bare(**more):
    cfg = decoder.DecoderConfig(layers=0, hidden=256, inter=512, **{"heads": 4, "vocab": 103, "max_seq": 96, **more})
    return decoder.GPTQDecoder(cfg, batch=2, device="cpu")


def test_a_model_keeps_its_numbers():
    m = bare()
    m.set_sampling(decoder.Sampling(top_p=0.5, seed=4))
    assert m._uniform.shape == (96, 2) and m._sampling_arguments["top_p"].tolist() == [0.5, 0.5]
    first = m._uniform.clone()
    m.set_sampling(decoder.Sampling(seed=4))
    assert torch.equal(first, m._uniform)
    m.set_sampling(None)
    assert m._uniform is None and m._sampling_arguments == {}
    with pytest.raises(ValueError):
        bare(vocab=(1 << 18) + 1).set_sampling(decoder.Sampling())


@pytest.mark.parametrize("bad", [dict(cache_bits=8), dict(cache_bits=4, cache_group=16), dict(cache_bits=4, heads=8)])
def test_caches_are_refused(bad):
    with pytest.raises(ValueError):
        bare(**bad)


def test_a_prompt_too_long_for_caches_of_4_bits_leaves_the_position():
    m = bare(max_seq=70000, cache_bits=4)
    m._pos_host = 5
    with pytest.raises(ValueError, match="65535"):
        m.prefill(torch.zeros(2, 65536, dtype=torch.long))
    assert m._pos_host == 5
