"""Modules whose products have an epilogue, and mixtures of experts as modules."""
import moe_plain as plain
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


def rnd(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


def dense(m, x, logits, gate, up, down, act, fmt, gate_bias=None, up_bias=None, down_bias=None):
    """The layer in fp64 with the 4-bit values of the matrices, each token through its experts."""
    from trellis_b200 import microscale as ms
    v = lambda w: ms.dequantize(ms.quantize(w, fmt)).double()  # noqa: E731
    weights, chosen, *_ = plain.route(logits, m.top_k, m.score, m.normalize)
    out = torch.zeros(x.shape[0], down.shape[1], dtype=torch.float64, device="cuda")
    for i in range(x.shape[0]):
        for j in range(m.top_k):
            e = int(chosen[i, j])
            if e >= 0:
                h = x[i].double() @ v(up[e]).t() + (0 if up_bias is None else up_bias[e].double())
                if gate is None:
                    h = plain.activate(h, act)
                else:
                    h = plain.activate(x[i].double() @ v(gate[e]).t() + (0 if gate_bias is None else gate_bias[e].double()), plain.GATED[act]) * h
                out[i] += weights[i, j] * (h.to(x.dtype).double() @ v(down[e]).t() + (0 if down_bias is None else down_bias[e].double()))
    return out


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("act,biases", [("swiglu", True), ("geglu", False), ("gelu", True), ("relu", False)])
def test_experts(act, biases, fmt):
    """As near to 64 bits as the roundings of the inner and of the last result leave it: 2^-9 of their sizes each (bf16), taken fourfold."""
    from trellis_b200.quant import MicroscaledExperts
    r = rnd(1)
    gated = act in plain.GATED
    up, down, gate = r(6, 72, 128) * 0.1, r(6, 96, 72) * 0.1, r(6, 72, 128) * 0.1 if gated else None
    ub, gb, db = (r(6, 72), r(6, 72) if gated else None, r(6, 96)) if biases else (None, None, None)
    m = MicroscaledExperts(up, down, 2, gate, fmt, act, up_bias=ub, gate_bias=gb, down_bias=db, score="sigmoid")
    x, logits, res = r(3, 7, 128).bfloat16(), r(3, 7, 6), r(3, 7, 96).bfloat16()
    out = m(x, logits, res)
    want = dense(m, x.reshape(21, 128), logits.reshape(21, 6), gate, up, down, act, fmt, gb, ub, db) + res.reshape(21, 96).double()
    assert out.shape == (3, 7, 96) and out.dtype == torch.bfloat16
    assert float((out.reshape(21, 96).double() - want).norm() / want.norm()) < 4 * 2.0 ** -9
    assert torch.equal(m(x[0, 0], logits[0, 0], res[0, 0]), m(x[:1, :1], logits[:1, :1], res[:1, :1])[0, 0])
    assert m(x[:0], logits[:0]).shape == (0, 7, 96)


def test_router_types_and_state():
    from trellis_b200.quant import MicroscaledExperts
    r = rnd(2)
    up, down, gate = r(4, 40, 64), r(4, 64, 40), r(4, 40, 64)
    router = nn.Linear(64, 4, bias=False, device="cuda", dtype=torch.bfloat16)
    m = MicroscaledExperts(up, down, 2, gate, "nvfp4", router=router)
    x = r(5, 64).bfloat16()
    with torch.no_grad():
        want = m(x)
        assert torch.equal(want, MicroscaledExperts(up, down, 2, gate, "nvfp4")(x, router(x)))
    m = m.to(torch.bfloat16)
    assert m.up_row_scale.dtype == torch.float32 and m.down_row_scale.dtype == torch.float32 and m.up_codes.dtype == torch.uint8
    with torch.no_grad():
        assert torch.equal(m(x), want)
        other = MicroscaledExperts(up * 0, down * 0, 2, gate * 0, "nvfp4", router=nn.Linear(64, 4, bias=False, device="cuda", dtype=torch.bfloat16))
        other.load_state_dict(m.state_dict())
        assert torch.equal(other(x), want)
    with pytest.raises(ValueError):
        m(x, router(x).detach())
    with pytest.raises(ValueError):
        MicroscaledExperts(up, down, 2, gate)(x)
    with pytest.raises(ValueError):
        m(r(5, 63).bfloat16())


@pytest.mark.parametrize("change", [dict(top_k=5), dict(top_k=0), dict(gate=None), dict(activation="gelu"), dict(activation="tanh"), dict(score="x"), dict(down="wrong"), dict(gate="wrong"),
                                    dict(gate_bias="bias"), dict(up_bias="bias"), dict(fmt="int4")])
def test_refusals(change):
    from trellis_b200.quant import MicroscaledExperts
    up = torch.randn(4, 40, 64, device="cuda")
    args = dict(up=up, down=torch.randn(4, 64, 40, device="cuda"), top_k=2, gate=up, fmt="nvfp4", activation="swiglu", score="softmax")
    args.update({k: {"wrong": up[:, :7], "bias": up[:, :, 0]}.get(v, v) if isinstance(v, str) else v for k, v in change.items()})
    with pytest.raises(ValueError):
        MicroscaledExperts(**args)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_linear_with_an_activation(dtype):
    from trellis_b200 import microscale as ms
    from trellis_b200.quant import MicroscaledLinear
    r = rnd(3)
    w, b, x = r(96, 64), r(96), r(2, 5, 64).to(dtype)
    for act in ("gelu", "swiglu"):
        m = MicroscaledLinear(w, b, activation=act)
        res = r(2, 5, 48 if act == "swiglu" else 96).to(dtype)
        assert torch.equal(m(x), ms.linear(x, ms.quantize(w, "nvfp4"), b, act)) and torch.equal(m(x, res), ms.linear(x, ms.quantize(w, "nvfp4"), b, act, res))
        assert act in repr(m)
    plain_one = MicroscaledLinear(w, b)
    assert torch.equal(plain_one(x), ms.linear(x, ms.quantize(w, "nvfp4")) + b.to(dtype))      # a bias alone: as it was
    assert torch.equal(plain_one(x, x.new_ones(2, 5, 96)), ms.linear(x, ms.quantize(w, "nvfp4"), b, residual=x.new_ones(2, 5, 96)))
    for bad in (lambda: MicroscaledLinear(w, b, activations=4, activation="gelu"), lambda: MicroscaledLinear(w[:95], None, activation="swiglu"), lambda: MicroscaledLinear(w, activation="tanh"),
                lambda: MicroscaledLinear(w, b, activations=4)(x, x.new_ones(2, 5, 96))):
        with pytest.raises(ValueError):
            bad()


def test_a_linear_layer_saved_without_an_activation():
    """A module's state as it was before there were activations."""
    import copy

    from trellis_b200 import quant
    layer = quant.MicroscaledLinear(rnd(0)(96, 64), rnd(1)(96))
    old = copy.deepcopy(layer)
    del old.__dict__["activation"]
    x = rnd(2)(5, 64).bfloat16()
    assert torch.equal(old(x), layer(x)) and torch.equal(old(x, x.new_zeros(5, 96)), layer(x, x.new_zeros(5, 96))) and repr(old) == repr(layer)
