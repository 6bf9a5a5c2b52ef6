"""``apply_microscaled`` over a model, with stand-ins for the layers that need a GPU."""
import weakref

import pytest
import torch
from torch import nn

from trellis_b200 import quant


class _Standin(nn.Module):
    made = []

    def __init__(self, weight, bias, fmt, activations, rotate, seed):
        super().__init__()
        _Standin.made.append((seed, [w() is not None for w in _Standin.watched]))


@pytest.fixture
def standin(monkeypatch):
    monkeypatch.setattr(quant, "MicroscaledLinear", _Standin)
    _Standin.made = []
    return _Standin


def test_each_layer_goes_before_the_next_is_replaced(standin):
    """The 16-bit weights of a model and its 4-bit ones are never all there at once."""
    model = nn.Sequential(nn.Linear(8, 8), nn.Sequential(nn.Linear(8, 4), nn.ReLU()), nn.Linear(4, 4))
    standin.watched = [weakref.ref(m.weight) for m in (model[0], model[1][0], model[2])]
    assert quant.apply_microscaled(model) == 3
    assert [alive for _, alive in standin.made] == [[True, True, True], [False, True, True], [False, False, True]]
    assert [seed for seed, _ in standin.made] == [quant.seed_from_name(n) for n in ("0", "1.0", "2")]


def test_a_layer_with_several_names_is_replaced_once(standin):
    shared = nn.Linear(8, 8)
    model = nn.ModuleDict({"a": shared, "b": nn.ModuleDict({"c": shared}), "d": nn.Linear(8, 8), "e": nn.ModuleDict({"c": shared})})
    standin.watched = []
    assert quant.apply_microscaled(model, skip=lambda n: n == "e.c") == 2
    assert model["a"] is model["b"]["c"] and isinstance(model["a"], _Standin) and isinstance(model["d"], _Standin) and model["e"]["c"] is shared


def test_nothing_is_replaced_where_a_later_layer_is_refused(standin):
    standin.watched = []
    for last in (nn.Linear(48, 8), nn.Linear(64, 8).double()):
        model = nn.Sequential(nn.Linear(64, 48), last)
        with pytest.raises(ValueError):
            quant.apply_microscaled(model, activations=4, rotate=64)
        assert not standin.made and all(type(m) is nn.Linear for m in model)


def test_layers_without_values_are_refused_before_any_is_replaced(standin):
    standin.watched = []
    model = nn.Sequential(nn.Linear(64, 48), nn.Linear(48, 8, device="meta"))
    with pytest.raises(ValueError, match="^1: "):
        quant.apply_microscaled(model)
    assert not standin.made and type(model[0]) is nn.Linear
