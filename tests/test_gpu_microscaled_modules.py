"""Models whose layers are kept in 4 bits, beyond what their products give: what the replaced layers had, and what their owners do with them."""
import gc
import weakref

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def quant():
    from trellis_b200 import quant
    return quant


def test_replacements_keep_the_mode_of_their_layers(quant):
    model = nn.Sequential(nn.Linear(32, 48), nn.Sequential(nn.Linear(48, 16)), nn.Dropout()).cuda().eval()
    model[1].train()
    assert quant.apply_microscaled(model) == 2
    assert not model[0].training and model[1][0].training and not model[2].training
    model.train()
    assert model[0].training
