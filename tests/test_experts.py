"""What mixtures of experts and products with an epilogue refuse, without a GPU: through Python and through the C ABI."""
import ctypes

import pytest
import torch

from trellis_b200 import _lib, experts, microscale as ms


def matrix(n=8, k=32, fmt="nvfp4"):
    codes, scales = ms._storage(n, k, fmt)
    return ms.Microscaled(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), torch.ones(n) if fmt == "nvfp4" else None, (n, k), fmt)


def stack(e=3, n=8, k=32, fmt="nvfp4"):
    codes, scales = ms._storage(n, k, fmt)
    return experts.ExpertMatrices(torch.zeros((e, *codes), dtype=torch.uint8), torch.zeros((e, *scales), dtype=torch.uint8), torch.ones(e, n) if fmt == "nvfp4" else None,
                                  (e, n, k), fmt)


def test_activations_by_name():
    assert ms._check_act(None, 7) == (0, 7) and ms._check_act("swiglu", 8) == (6, 4)
    for act, n in (("tanh", 8), ("swiglu", 7), ("geglu", 1), ("", 4)):
        with pytest.raises(ValueError):
            ms._check_act(act, n)


def test_bias():
    dev = torch.device("cpu")
    assert ms._check_bias(None, (4,), dev) is None
    b = torch.zeros(4, 2)[:, 0]
    assert ms._check_bias(b, (4,), dev).is_contiguous()
    for bad in (torch.zeros(3), torch.zeros(1, 4), torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int32), torch.zeros(4, device="meta"), torch.zeros(4, requires_grad=True)):
        with pytest.raises(ValueError):
            ms._check_bias(bad, (4,), dev)


def test_interleave():
    g, u = torch.arange(6.0).reshape(2, 3), -torch.arange(6.0).reshape(2, 3)
    w = ms.interleave(g, u)
    assert torch.equal(w[0::2], g) and torch.equal(w[1::2], u)
    assert ms.interleave(g[None], u[None]).shape == (1, 4, 3)
    for a, b in ((g, u[:1]), (g[0], u[0])):
        with pytest.raises(ValueError):
            ms.interleave(a, b)


def test_cpu_tensors_are_refused():
    x, r = torch.zeros(2, 32, dtype=torch.bfloat16), experts.Routing(torch.ones(2, 1), *[torch.zeros(2, 1, dtype=torch.int32)] * 4)
    for call in (lambda: ms.linear(x, matrix(), activation="relu"), lambda: ms.linear(x, matrix(fmt="mxfp4"), bias=torch.zeros(8)),
                 lambda: experts.grouped_linear(x, stack(), torch.zeros(4, dtype=torch.int32)), lambda: experts.route(torch.zeros(2, 4), 2),
                 lambda: experts.combine(x, r), lambda: experts.quantize_experts(torch.zeros(2, 4, 32)), lambda: experts.stack_experts([matrix()])):
        with pytest.raises((ValueError, RuntimeError)):
            call()


@pytest.mark.parametrize("change", [dict(codes=torch.zeros(3, 8, 32, dtype=torch.uint8)), dict(codes=torch.zeros(3, 8, 16)), dict(row_scale=None), dict(row_scale=torch.ones(8)),
                                    dict(scales=torch.zeros(3, 1, 2, 32, 4, 4, dtype=torch.uint8)), dict(fmt="int4"), dict(fmt="mxfp4"), dict(shape=(3, 9, 32)), dict(shape=(2, 8, 32)),
                                    dict(row_scale=torch.ones(3, 8, requires_grad=True))])
def test_malformed_matrices(change):
    with pytest.raises(ValueError):
        experts._check_e(stack()._replace(**change), "w")


def test_arguments():
    with pytest.raises(ValueError):
        experts._check_e(matrix(), "w")
    for top in (0, 5, True, 2.0, 33):
        with pytest.raises(ValueError):
            experts.route(torch.zeros(2, 4), top)
    for bad in (torch.zeros(4), torch.zeros(2, 4, 1), torch.zeros(2, 2000), torch.zeros(2, 4, dtype=torch.float64)):
        with pytest.raises((ValueError, RuntimeError)):
            experts.route(bad, 2)
    with pytest.raises(ValueError):
        experts.route(torch.zeros(2, 4), 2, score="linear")
    with pytest.raises(ValueError):
        experts.route(torch.zeros(2, 4, requires_grad=True), 2)
    for w in (torch.zeros(4, 32), torch.zeros(2, 4, 32, dtype=torch.float64)):
        with pytest.raises(ValueError):
            experts.quantize_experts(w)
    with pytest.raises(ValueError):
        experts.stack_experts([])
    with pytest.raises(TypeError):
        torch.zeros(3) + stack()


def test_the_short_way_leaves_what_it_does_not_take():
    """On the CPU it takes nothing: the Python functions say what is wrong, with it as without it."""
    short = _lib.short()
    assert short, "tcq_torch.so is not built"
    x, w, e = torch.zeros(2, 32, dtype=torch.bfloat16), matrix(), stack()
    r = experts.Routing(torch.ones(2, 1), *[torch.zeros(2, 1, dtype=torch.int32)] * 4)
    for got in (short.linear(x, w, None, "relu", None), short.linear(None, w, None, "relu", None), short.linear(x, (1, 2), None, None, x), short.linear(x, w, None, "tanh", None),
                short.linear(x, w), short.grouped_linear(x, e, torch.zeros(4, dtype=torch.int32), None, None, None, None), short.grouped_linear(x, w, None, None, None, None, None),
                short.grouped_linear(), short.route(torch.zeros(2, 4), 2, "softmax", True), short.route(torch.zeros(2, 4), 1 << 70, "softmax", True), short.route(3, 2, "softmax", True),
                short.combine(x, r, None, None), short.combine(x, None, None, None), short.combine(x, r, None, 7),
                short.linear(x, w._replace(shape=(1 << 80, 32)), None, "relu", None), short.linear(x, w._replace(shape=("a", 32)), None, "relu", None)):
        assert got is None
    with pytest.raises(TypeError):
        short.bind(1, 2)


# ------------------------------------------------------------------------------------------------ the C ABI
BAD_COUNT, NULL, MISALIGNED, WORKSPACE, BAD, FORMAT = -3, -4, -5, -6, -8, -12


def at(address=4096):
    return ctypes.c_void_p(address)


GROUPED = dict(x=at(), dtype=2, x_rows=10, ldx=64, tokens=None, offsets=at(), groups=3, rows=10, codes=at(), scales=at(), row_scale=at(), n=8, k=64, format=1, bias=at(), bias_dtype=0,
               activation=6, residual=at(), ldr=8, y=at(), y_dtype=2, ldy=8, ws=at(), ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("code,change", [
    (FORMAT, dict(dtype=0)), (FORMAT, dict(dtype=3)), (FORMAT, dict(format=2)), (FORMAT, dict(y_dtype=7)), (FORMAT, dict(bias_dtype=-1)), (BAD_COUNT, dict(rows=-1)), (BAD_COUNT, dict(n=-1)),
    (BAD_COUNT, dict(k=-2)), (BAD_COUNT, dict(groups=-1)), (BAD_COUNT, dict(x_rows=-1)), (BAD, dict(groups=0)), (BAD, dict(groups=1025)), (BAD, dict(rows=(1 << 30) + 1)),
    (BAD, dict(groups=1024, n=1 << 21)), (BAD, dict(rows=1 << 30, n=300, x_rows=1 << 30)), (BAD, dict(k=(1 << 24) + 1, ldx=1 << 25)), (BAD, dict(k=0)), (BAD, dict(ldx=63)), (BAD, dict(x_rows=9)),
    (BAD, dict(activation=7)), (BAD, dict(activation=-1)), (BAD, dict(n=7)), (BAD, dict(ldy=3)), (BAD, dict(ldr=3)), (NULL, dict(offsets=None)), (NULL, dict(x=None)), (NULL, dict(codes=None)),
    (NULL, dict(scales=None)), (NULL, dict(row_scale=None)), (NULL, dict(format=0)), (NULL, dict(y=None)), (NULL, dict(ws=None)), (MISALIGNED, dict(x=at(4097))), (MISALIGNED, dict(codes=at(4104))),
    (MISALIGNED, dict(scales=at(4104))), (MISALIGNED, dict(row_scale=at(4098))), (MISALIGNED, dict(bias=at(4098))), (MISALIGNED, dict(residual=at(4097))), (MISALIGNED, dict(y=at(4097))),
    (MISALIGNED, dict(tokens=at(4098))), (MISALIGNED, dict(offsets=at(4098))), (MISALIGNED, dict(ws=at(4224))), (WORKSPACE, dict(ws_bytes=100))])
def test_grouped_refusals(code, change):
    assert _lib.lib().tcq_ms_grouped_linear(*{**GROUPED, **change}.values()) == code
    assert _lib.lib().tcq_selftest_ms_grouped_waits(1, *{**GROUPED, **change}.values()) == code


def test_grouped_calls_of_nothing():
    L = _lib.lib()
    assert L.tcq_ms_grouped_linear(*{**GROUPED, "rows": 0}.values()) == 0 and L.tcq_ms_grouped_linear(*{**GROUPED, "n": 0}.values()) == 0
    assert L.tcq_selftest_ms_grouped_waits(-1, *GROUPED.values()) == BAD_COUNT
    assert L.tcq_ms_grouped_linear_workspace_bytes(0, 3, 8, 64, 2, 1, 1) == 0 and L.tcq_ms_grouped_linear_workspace_bytes(10, 3, 8, 64, 0, 1, 1) == 0
    assert L.tcq_ms_grouped_linear_workspace_bytes(10, 3, 8, 64, 2, 1, 1) > 0


EPILOGUE = dict(h=at(), rows=4, n=8, bias=at(), bias_dtype=0, activation=5, residual=at(), ldr=4, y=at(), y_dtype=0, ldy=4, stream=None)


@pytest.mark.parametrize("code,change", [(BAD_COUNT, dict(rows=-1)), (BAD_COUNT, dict(n=-1)), (BAD, dict(activation=9)), (BAD, dict(n=7)), (BAD, dict(ldy=3)), (BAD, dict(ldr=3)), (NULL, dict(h=None)),
                                         (NULL, dict(y=None)), (MISALIGNED, dict(h=at(4098))), (FORMAT, dict(y_dtype=3)), (0, dict(rows=0)), (0, dict(n=0))])
def test_epilogue_refusals(code, change):
    assert _lib.lib().tcq_ms_epilogue(*{**EPILOGUE, **change}.values()) == code


ROUTE = dict(logits=at(), dtype=0, tokens=1000, ld=16, experts=16, top=2, score=0, normalize=1, weights=at(), chosen=at(), places=at(), order=at(), offsets=at(), ws=at(), ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("code,change", [(FORMAT, dict(dtype=3)), (BAD_COUNT, dict(tokens=-1)), (BAD, dict(experts=0)), (BAD, dict(experts=1025, ld=2000)), (BAD, dict(top=0)), (BAD, dict(top=17)),
                                         (BAD, dict(top=33, experts=64, ld=64)), (BAD, dict(tokens=1 << 30)), (BAD, dict(ld=15)), (BAD, dict(score=2)), (BAD, dict(normalize=2)), (NULL, dict(logits=None)),
                                         (NULL, dict(weights=None)), (NULL, dict(chosen=None)), (NULL, dict(places=None)), (NULL, dict(order=None)), (NULL, dict(offsets=None)), (NULL, dict(ws=None)),
                                         (MISALIGNED, dict(logits=at(4097))), (MISALIGNED, dict(weights=at(4098))), (WORKSPACE, dict(ws_bytes=16))])
def test_route_refusals(code, change):
    assert _lib.lib().tcq_route(*{**ROUTE, **change}.values()) == code


COMBINE = dict(y=at(), dtype=2, rows=20, ldy=8, n=8, weights=at(), places=at(), tokens=10, top=2, residual=at(), ldr=8, out=at(), out_dtype=2, ldo=8, stream=None)


@pytest.mark.parametrize("code,change", [(FORMAT, dict(dtype=-1)), (FORMAT, dict(out_dtype=3)), (BAD_COUNT, dict(rows=-1)), (BAD_COUNT, dict(n=-1)), (BAD_COUNT, dict(tokens=-1)), (BAD, dict(top=0)),
                                         (BAD, dict(top=33)), (BAD, dict(ldy=7)), (BAD, dict(ldr=7)), (BAD, dict(ldo=7)), (BAD, dict(rows=1 << 31)), (NULL, dict(y=None)), (NULL, dict(weights=None)),
                                         (NULL, dict(places=None)), (NULL, dict(out=None)), (MISALIGNED, dict(y=at(4097))), (MISALIGNED, dict(out=at(4097))), (MISALIGNED, dict(residual=at(4097))),
                                         (MISALIGNED, dict(places=at(4098))), (0, dict(tokens=0)), (0, dict(n=0))])
def test_combine_refusals(code, change):
    assert _lib.lib().tcq_combine(*{**COMBINE, **change}.values()) == code
