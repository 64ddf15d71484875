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
