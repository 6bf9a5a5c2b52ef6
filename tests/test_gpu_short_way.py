"""The extension that takes the small calls gives what the calls through ctypes give, and leaves to them what it does not take."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def both(monkeypatch):
    """Runs a call the short way and the other way; the two results, or the two refusals."""
    from trellis_b200 import _lib
    short = _lib.short()
    assert short, "tcq_torch.so is not built"

    def run(call):
        got = []
        for way in (short, False):
            monkeypatch.setattr(_lib, "_short", way)
            try:
                got.append(call())
            except ValueError as e:
                got.append(str(e))
        monkeypatch.setattr(_lib, "_short", short)
        return got
    return run


def same(a, b):
    if isinstance(a, tuple):
        assert type(a) is type(b) and all(same(x, y) for x, y in zip(a, b))
        return True
    assert isinstance(a, torch.Tensor) and a.dtype == b.dtype and a.shape == b.shape and a.is_contiguous() and a.device == b.device
    assert torch.equal(a.nan_to_num(-7), b.nan_to_num(-7))
    return True


def setup(fmt="nvfp4"):
    from trellis_b200 import experts, microscale as ms
    g = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return rnd, ms.quantize(rnd(96, 160), fmt), experts.quantize_experts(rnd(5, 96, 160), fmt)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
def test_results(both, fmt, dtype):
    from trellis_b200 import experts, microscale as ms
    rnd, w, e = setup(fmt)
    for shape in ((1, 160), (7, 160), (2, 3, 160), (160,), (0, 160), (300, 160)):
        x = rnd(*shape).to(dtype)
        for act in (None, "relu", "gelu", "gelu_tanh", "silu", "geglu", "swiglu"):
            r = rnd(*shape[:-1], 48 if act in ms.GATED else 96).to(dtype)
            for bias in (None, rnd(96), rnd(96).half()):
                same(*both(lambda: ms.linear(x, w, bias, act, r)))
    wide = rnd(9, 200).to(dtype)
    same(*both(lambda: ms.linear(wide[:, 3:163], w, None, "silu", wide[:, :96])))
    same(*both(lambda: ms.linear(wide.t()[:160].t(), w, wide[0, :192:2].contiguous(), None, wide[:, :96].t().contiguous().t())))
    logits = rnd(50, 5).to(dtype)
    for top in (1, 3, 5):
        for score in ("softmax", "sigmoid"):
            for norm in (True, False):
                same(*both(lambda: experts.route(logits, top, score, norm)))
    same(*both(lambda: experts.route(wide[:, 2:7], 2)))
    same(*both(lambda: experts.route(logits[:0], 2)))
    r = experts.route(logits, 2)
    y = rnd(100, 33).to(dtype)
    for residual in (None, rnd(50, 33), rnd(50, 33).half()):
        same(*both(lambda: experts.combine(y, r, residual)))
    same(*both(lambda: experts.combine(y, r, dtype=torch.float16)))
    if dtype != torch.float32:
        x = rnd(50, 160).to(dtype)
        for tokens in (None, r.tokens):
            for act in (None, "swiglu"):
                for out in (None, torch.float32, dtype):
                    offsets = r.offsets if tokens is not None else torch.tensor([0, 3, 3, 20, 49, 50], device=DEV).int()
                    same(*both(lambda: experts.grouped_linear(x, e, offsets, tokens, rnd(5, 96) * 0 + 1, act, out)))


def test_refusals(both):
    """What is refused is refused in the same words."""
    from trellis_b200 import experts, microscale as ms
    rnd, w, e = setup()
    x, r = rnd(4, 160).bfloat16(), experts.route(rnd(4, 5), 2)
    off, grad = r.offsets, rnd(4, 160).bfloat16().requires_grad_()
    calls = [lambda: ms.linear(x[:, :100], w, activation="relu"), lambda: ms.linear(x, w, activation="tanh"), lambda: ms.linear(x, w, residual=rnd(4, 96)), lambda: ms.linear(x, w, residual=x),
             lambda: ms.linear(x, w, bias=rnd(95)), lambda: ms.linear(x, w, bias=rnd(96).double()), lambda: ms.linear(x, w, bias=torch.zeros(96)), lambda: ms.linear(x.cpu(), w, activation="relu"),
             lambda: ms.linear(grad, w, activation="relu"), lambda: ms.linear(x, w, bias=rnd(96).requires_grad_()), lambda: ms.linear(x, w, residual=rnd(4, 96).bfloat16().requires_grad_()),
             lambda: ms.linear(x.double(), w, activation="relu"), lambda: ms.linear(x, w._replace(codes=w.codes[:5]), activation="relu"), lambda: ms.linear(x, e, activation="relu"),
             lambda: ms.linear(x, w._replace(row_scale=None), activation="relu"),
             lambda: experts.grouped_linear(x.float(), e, off, r.tokens), lambda: experts.grouped_linear(x, e, off[:-1], r.tokens), lambda: experts.grouped_linear(x, e, off.long(), r.tokens),
             lambda: experts.grouped_linear(x, e, off, r.tokens.long()), lambda: experts.grouped_linear(x, e, off.cpu(), r.tokens), lambda: experts.grouped_linear(grad, e, off, r.tokens),
             lambda: experts.grouped_linear(x, e, off, r.tokens, activation="x"), lambda: experts.grouped_linear(x, e, off, r.tokens, bias=rnd(96)), lambda: experts.grouped_linear(x, w, off),
             lambda: experts.grouped_linear(x, e, off, r.tokens, dtype=torch.int32), lambda: experts.grouped_linear(x[None], e, off, r.tokens),
             lambda: experts.route(rnd(4, 5), 6), lambda: experts.route(rnd(4), 1), lambda: experts.route(rnd(4, 5).requires_grad_(), 1), lambda: experts.route(rnd(4, 5), 2, "x"),
             lambda: experts.route(rnd(4, 5).int(), 2), lambda: experts.combine(x, r, rnd(3, 160)), lambda: experts.combine(x, r, rnd(4, 160), torch.float16), lambda: experts.combine(grad, r),
             lambda: experts.combine(x, r._replace(weights=r.weights.double())), lambda: experts.combine(x, r._replace(places=r.places.long())), lambda: experts.combine(x.int(), r)]
    for i, call in enumerate(calls):
        a, b = both(call)
        assert isinstance(a, str) and a == b, i
    with torch.no_grad():
        same(*both(lambda: ms.linear(grad, w, activation="relu")))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ms.linear(dual, w, activation="relu"), lambda: experts.grouped_linear(dual, e, off, r.tokens), lambda: experts.combine(dual, r)):
            a, b = both(call)
            assert isinstance(a, str) and a == b


def test_results_have_no_history():
    from trellis_b200 import experts, microscale as ms
    rnd, w, e = setup()
    x = rnd(4, 160).bfloat16()
    for t in (ms.linear(x, w, activation="relu"), *experts.route(rnd(4, 5), 2), experts.grouped_linear(x, e, torch.tensor([0, 1, 2, 3, 4, 4], device=DEV).int())):
        assert not t.requires_grad and t.grad_fn is None
