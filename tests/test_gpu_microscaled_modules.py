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


def test_forward_hooks_go_with_the_layer(quant):
    model = nn.Sequential(nn.Linear(32, 48), nn.Linear(48, 16)).cuda()
    seen = []
    handle = model[0].register_forward_hook(lambda mod, args, out: seen.append(out.shape))
    model[1].register_forward_pre_hook(lambda mod, args: (args[0] * 0,))
    model[1].register_forward_hook(lambda mod, args, kwargs, out: out + 1, with_kwargs=True)
    bias = model[1].bias.data.clone()
    assert quant.apply_microscaled(model) == 2
    with torch.no_grad():
        y = model(torch.randn(3, 32, device="cuda"))
    assert seen == [(3, 48)] and torch.equal(y, (bias + 1).expand(3, 16))
    handle.remove()
    with torch.no_grad():
        model(torch.randn(3, 32, device="cuda"))
    assert len(seen) == 1


@pytest.mark.parametrize("change", ("norm", "prune", "forward", "state"))
def test_layers_that_are_more_than_their_weight_are_refused(quant, change):
    from torch.nn.utils import prune, weight_norm
    model = nn.Sequential(nn.Linear(32, 48), nn.Linear(48, 16)).cuda()
    if change == "norm":
        weight_norm(model[1])
    elif change == "prune":
        prune.random_unstructured(model[1], "weight", 0.3)
    elif change == "forward":
        model[1].forward = lambda x: x
    else:
        model[1].register_state_dict_pre_hook(lambda *a: None)
    with pytest.raises(ValueError, match="^1: "):
        quant.apply_microscaled(model)
    assert type(model[0]) is nn.Linear and quant.apply_microscaled(model, skip=lambda name: name == "1") == 1


@pytest.mark.parametrize("batch_first", (True, False))
@pytest.mark.parametrize("mode", ("train", "eval", "no_grad", "padded"))
def test_transformer_layers_that_read_their_weights(quant, batch_first, mode):
    """In evaluation torch's encoder hands its layers' weights to one fused function, unless they are not plain tensors."""
    torch.manual_seed(0)
    layer = nn.TransformerEncoderLayer(64, 4, 128, dropout=0.0, batch_first=batch_first, device="cuda")
    model = nn.TransformerEncoder(layer, 2)
    assert quant.apply_microscaled(model) == 4
    for m in model.layers:
        assert isinstance(m.linear1, quant.MicroscaledLinear)
    model.requires_grad_(False).train(mode == "train")
    x = torch.randn(2, 5, 64, device="cuda")
    mask = torch.tensor([[False] * 5, [False] * 3 + [True] * 2], device="cuda") if mode == "padded" and batch_first else None
    with torch.set_grad_enabled(mode in ("train", "eval")):
        y = model(x, src_key_padding_mask=mask)
    # the same layers with the values of their 4-bit weights, on torch's plain path
    from trellis_b200 import microscale as ms
    plain = nn.TransformerEncoder(nn.TransformerEncoderLayer(64, 4, 128, dropout=0.0, batch_first=batch_first, device="cuda"), 2).double()
    state = {n: t.double() for n, t in model.state_dict().items() if "linear" not in n}
    for i, m in enumerate(model.layers):
        for name in ("linear1", "linear2"):
            state[f"layers.{i}.{name}.weight"] = ms.dequantize(getattr(m, name).weight).double()
            state[f"layers.{i}.{name}.bias"] = getattr(m, name).bias.double()
    plain.load_state_dict(state)
    want = plain.requires_grad_(False).train()(x.double(), src_key_padding_mask=mask)
    # two layers, each three sums of at most 128 products of fp32 numbers and a normalisation: 1e-3 is a hundred times what their roundings can add up to
    off = (y.double() - want).abs()
    assert (off if mask is None else off[~mask]).max() < 1e-3


def test_torch_functions_refuse_a_matrix_in_four_bits(quant):
    layer = quant.MicroscaledLinear(torch.randn(16, 32))
    with pytest.raises(TypeError):
        nn.functional.linear(torch.randn(3, 32, device="cuda"), layer.weight)


@pytest.mark.parametrize("activations", (4, 16))
def test_inputs_of_every_width_and_none(quant, activations):
    layer = quant.MicroscaledLinear(torch.randn(16, 32), torch.randn(16), activations=activations)
    with torch.no_grad():
        for shape in ((0, 32), (2, 0, 32), (32,), (1, 1, 1, 32)):
            assert layer(torch.randn(shape, device="cuda")).shape == (*shape[:-1], 16)
        for shape in ((0, 64), (4, 16), (2, 64), (), (16, 2)):
            with pytest.raises(ValueError, match="32"):
                layer(torch.randn(shape, device="cuda"))
        none = quant.MicroscaledLinear(torch.zeros(5, 0), torch.arange(5.0), activations=activations)
        assert torch.equal(none(torch.zeros(3, 0, device="cuda")).cpu(), torch.arange(5.0).expand(3, 5))
