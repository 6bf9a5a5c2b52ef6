"""Calls of the operators around experts at which something could go wrong that sizes between do not show."""
import ms_cases
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k", [(1, 64), (2, 64), (1, 700), (2, 512)])
def test_many_items_of_the_same_rows(m, k, fmt):
    """One or two rows through a matrix of more than three times 128 rows for every SM: a CTA's items share what x was cut into.  Whole numbers, bit for bit, call after call."""
    from trellis_b200 import microscale as ms
    n = 128 * 148 * 4 - 77
    w, wv = ms_cases.whole_matrix(n, k, fmt, 1)
    x = ms_cases.whole_tokens(m, k, torch.bfloat16, 2)
    want = (x.double() @ wv.t()).to(torch.bfloat16)
    b = torch.zeros(n, device=DEV)
    got = [ms.linear(x, w, bias=b) for _ in range(20)]
    assert all(torch.equal(y, want) for y in got)


def digits_bound(x, w, fmt):
    """Of fp32 sums of x's 4-bit parts times w (fp64 [m, k], [n, k]).  A number of x is rounded to 21 binary places of the power of two of its block's largest, 2^-22 of that off, or of 2^-17 of the
    row's largest (nvfp4), 2^-39 of it off.  Its digits' magnitudes are less than three times its own, or than that step; sums of 64 columns each are cut off by 2^-22 of theirs at most."""
    import moe_plain as plain
    b, k = plain.BLOCK[fmt], x.shape[1]
    amax = torch.nn.functional.pad(x.abs(), (0, -k % b)).reshape(x.shape[0], -1, b).amax(2).repeat_interleave(b, 1)[:, :k]
    step = torch.maximum(amax * 2.0 ** -22, x.abs().amax(1, keepdim=True) * (2.0 ** -39 if fmt == "nvfp4" else 0))
    return (step + (3 * x.abs() + 2 * step) * (k / 64 + 8) * 2.0 ** -22) @ w.abs().t()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m", [1, 2, 3, 7, 15, 30, 130, 700])
def test_a_channel_far_above_the_others(m, dtype, fmt):
    """A channel 60000 times the others, in whose column some results have no weight: these are as near to 64 bits as bf16 is (2^-9), the steps of the channel's block, 2^-7, notwithstanding (2^-7 sqrt(32 / 777) at most of the size of all)."""
    import moe_plain as plain
    from trellis_b200 import experts, microscale as ms
    g = torch.Generator(device=DEV).manual_seed(m)
    for n, k in ((256, 4096), (300, 777)):
        w = torch.randn(1, n, k, generator=g, device=DEV) * 0.02
        w[:, ::2, 100] = 0
        q = experts.quantize_experts(w, fmt)
        wv = ms.dequantize(experts.expert(q, 0)).double()
        x = torch.randn(m, k, generator=g, device=DEV)
        x[:, 100] = 60000.0
        x = x.to(dtype)
        y = experts.grouped_linear(x, q, torch.tensor([0, m], device=DEV).int(), dtype=torch.float32)
        want, bound = plain.epilogue(x.double() @ wv.t(), digits_bound(x.double(), wv, fmt), None, None, None, torch.float32)
        assert bool(((y.double() - want).abs() <= bound).all())
        rest = y[:, ::2].double() - want[:, ::2]
        assert float(rest.norm() / want[:, ::2].norm()) < 2.0 ** -9
        z = ms.linear(x, experts.expert(q, 0), bias=torch.zeros(n, device=DEV))
        assert torch.equal(z, y.to(dtype))


@pytest.mark.parametrize("dtype,apart", [(torch.bfloat16, 14), (torch.float16, 11)], ids=str)
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [1, 2, 3, 20, 200])
def test_every_bit_as_far_down_as_the_digits_reach(m, fmt, dtype, apart):
    """A block's numbers down to 2^-14 (fp16: 2^-11) of its largest count with every bit.  Each result is one number of x times one weight: exact, or (a block's largest may have been rounded up
    to 2, so that the least are further below it) of the number rounded to 21 places of its block's power of two."""
    import moe_plain as plain
    from trellis_b200 import experts, microscale as ms
    g = torch.Generator(device=DEV).manual_seed(m)
    k = 256
    w = torch.eye(k, device=DEV)[None]
    q = experts.quantize_experts(w, fmt)
    x = torch.ldexp(torch.rand(m, k, generator=g, device=DEV) + 1, -torch.randint(0, apart + 1, (m, k), generator=g, device=DEV)) * torch.randn(m, k, generator=g, device=DEV).sign()
    x[:, ::16] = 1.5
    x = x.to(dtype)
    y = experts.grouped_linear(x, q, torch.tensor([0, m], device=DEV).int(), dtype=torch.float32)
    wv, xd, b = ms.dequantize(experts.expert(q, 0)).double().diagonal(), x.double(), plain.BLOCK[fmt]
    step = torch.exp2(xd.abs().reshape(m, -1, b).amax(2).log2().floor() - 21).repeat_interleave(b, 1)
    rounded = (xd / step).round() * step
    assert bool((rounded == xd).float().mean() > 0.99)
    assert bool(((y.double() == xd * wv) | (y.double() == rounded * wv)).all())


@pytest.mark.parametrize("act", ["silu", "swiglu", "gelu_tanh", "gelu", "geglu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m", [1, 40, 400])
def test_tails_of_activations(m, dtype, act):
    """Sums that are exact, from far below zero to far above: results to a few ulp of their own size, not of one.  fp32: the function's 8 ulp (an exponential and a quotient 2 each, or erfc 4, and
    products and sums of 1 / 2), and what the rounding of its argument makes of it: the exponent of the tanh form is off by 4 roundings of itself, |2 z| <= 1.6 |h| + 0.08 |h|^3, erfc's argument
    by 2, of h^2 / 2 in its exponent and so of h^2 + 1 in the result.  And half a step of the type; below the normal numbers, steps of the least number: the exponential's, times |h|, and
    the result's."""
    import moe_plain as plain
    from trellis_b200 import microscale as ms
    reach = {"silu": 100, "swiglu": 100, "gelu_tanh": 11, "gelu": 13, "geglu": 13}[act]
    h = torch.linspace(-reach, 30, m * 16, dtype=torch.float64, device=DEV).to(torch.bfloat16 if dtype != torch.float16 else dtype).reshape(m, 16)
    x = torch.zeros(m, 64, device=DEV)
    x[:, 0:32:2], x[:, 33::2] = h.float(), 1.0
    w = torch.zeros(32 if act in plain.GATED else 16, 64, device=DEV)
    for j in range(16):
        if act in plain.GATED:
            w[2 * j, 2 * j], w[2 * j + 1, 2 * j + 33] = 1.0, 1.0
        else:
            w[j, 2 * j] = 1.0
    q = ms.quantize(w, "mxfp4")
    assert torch.equal(ms.dequantize(q), w)
    y = ms.linear(x.to(dtype), q, activation=act).double()
    hd = h.double()
    want = plain.activate(hd, plain.GATED.get(act, act))
    a = hd.abs()
    grows = {"silu": 0 * a, "gelu_tanh": 4 * (1.6 * a + 0.08 * a ** 3), "gelu": 2 * (a * a + 1)}[plain.GATED.get(act, act)]
    info = torch.finfo(dtype)
    bound = want.abs() * (8 * 2.0 ** -23 + grows * 2.0 ** -24 + info.eps / 2) + (a + 2) * 2.0 ** -149 + info.smallest_normal * info.eps / 2
    off = (y - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), float(hd.flatten()[(off / bound).argmax()]))


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 1031])
def test_combining_rows_of_almost_31_bits_of_columns(n):
    """The last turn of a row's columns ends behind 2^31; what lies before and behind the result stays as it is."""
    from trellis_b200 import _lib
    y = torch.arange(n, dtype=torch.int64, device=DEV).bitwise_and_(255).to(torch.bfloat16)[None]
    room = torch.full((n + 8192,), -1.0, dtype=torch.bfloat16, device=DEV)
    out = room[4096:4096 + n][None]
    weights, places = torch.full((1, 1), 2.0, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    rc = _lib.lib().tcq_combine(y.data_ptr(), 2, 1, n, n, weights.data_ptr(), places.data_ptr(), 1, 1, None, 0, out.data_ptr(), 2, n, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(out, y * 2) and bool((room[:4096] == -1).all()) and bool((room[4096 + n:] == -1).all())


def test_routing_as_many_tokens_as_are_taken():
    """2^31 - 2 tokens of one expert: the last chunk ends where an int does."""
    from trellis_b200 import experts
    t = 2 ** 31 - 2
    r = experts.route(torch.zeros(t, 1, dtype=torch.bfloat16, device=DEV), 1)
    assert r.offsets.tolist() == [0, t]
    for at in (0, 1 << 30, t - (1 << 26)):
        want = torch.arange(at, at + (1 << 26), dtype=torch.int32, device=DEV)
        part = slice(at, at + (1 << 26))
        assert torch.equal(r.places[part, 0], want) and torch.equal(r.tokens[part], want)
        assert bool((r.weights[part] == 1).all()) and bool((r.experts[part] == 0).all())
    del r
    torch.cuda.empty_cache()


def test_a_routing_as_a_plain_tuple(monkeypatch):
    """Its parts count, not its type, with the extension and without."""
    from trellis_b200 import _lib, experts
    g = torch.Generator(device=DEV).manual_seed(0)
    r, y = experts.route(torch.randn(6, 5, generator=g, device=DEV), 2), torch.randn(12, 40, generator=g, device=DEV)
    want = experts.combine(y, r)
    for way in (_lib.short(), False):
        monkeypatch.setattr(_lib, "_short", way)
        assert torch.equal(experts.combine(y, tuple(r)), want) and torch.equal(experts.combine(y, r), want)
        for bad in (tuple(r)[:4], list(r), r.weights):
            with pytest.raises(ValueError):
                experts.combine(y, bad)


@pytest.mark.parametrize("t", [13, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("score,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_weights_of_special_logits(score, normalize, dtype, t):
    """Weight by weight: a row that is not finite excuses no other.  An exponential of a rounded difference of up to 103 (beyond, it is nothing), 2^-17.3, twice, its own 2 ulp, and a sum of five: 2^-16;
    below the normal numbers, their steps (2^-126 is more).  Without an expert a weight is 0."""
    import moe_plain as plain
    from trellis_b200 import experts
    inf, nan = float("inf"), float("nan")
    rows = [[0.0, -0.0, 0.0, -0.0, 1e-45], [-inf] * 5, [-inf, 2.0, -inf, -inf, -inf], [nan, 1.0, 2.0, 3.0, 4.0], [-3e38, 3e38, -inf, -3e38, 3e38], [-200.0, -201.0, -200.0, -inf, -300.0],
            [-1e-40, -2e-40, 1e-40, 0.0, -inf], [1.0, -inf, -inf, -inf, 1.0], [-29.0, -95.0, -60.0, -88.5, -110.0], [-31.0, -29.5, -94.0, -101.0, -115.0], [0.5, -70.0, -85.0, -87.0, -20.0],
            [60.0, 20.0, -20.0, -26.0, -16.0], [88.0, 90.0, 87.0, 3.0, -3.0]]
    logits = torch.tensor(rows, device=DEV).repeat(-(-t // len(rows)), 1)[:t].to(dtype).contiguous()
    for top in (1, 2, 5):
        r, want = experts.route(logits, top, score, normalize), plain.route(logits, top, score, normalize)
        got, weights = r.weights.cpu().double(), want[0]
        assert torch.equal(r.experts.cpu().long(), want[1])
        assert torch.equal(got.isnan(), weights.isnan()) and int(weights.isnan().sum()) == (-(-(t - 3) // len(rows)) * (1 if score == "sigmoid" and not normalize else top))
        assert bool((got[want[1] < 0] == 0).all())
        off = (got - weights).abs()
        assert bool(((off <= weights * 2.0 ** -16 + 2.0 ** -126) | weights.isnan()).all())


@pytest.mark.parametrize("fmt,dtype", [("mxfp4", torch.bfloat16), ("nvfp4", torch.bfloat16), ("nvfp4", torch.float16)], ids=str)
@pytest.mark.parametrize("n,gather", [(1500, False), (20000, True)])
def test_waits_of_many_rows_that_run_out(n, gather, fmt, dtype):
    """Loads of weights that never come, in the form that takes hundreds of rows a group (it has no workspace but for rows that it puts in order): the kernel ends, what needed them is NaN, what did
    not is right, and so is the next call."""
    from trellis_b200 import _lib, experts
    g = torch.Generator(device=DEV).manual_seed(0)
    e, rows, k = 2, 600, 512                                      # two loads an item; one item a CTA, or four and more
    w = experts.quantize_experts(torch.randn(e, n, k, generator=g, device=DEV) * k ** -0.5, fmt)
    x = torch.randn(rows, k, generator=g, device=DEV).to(dtype)
    tokens = torch.randperm(rows, generator=g, device=DEV).int() if gather else None
    offsets = torch.tensor([0, 290, rows], device=DEV).int()
    want = experts.grouped_linear(x, w, offsets, tokens)
    L, f, d = _lib.lib(), 0 if fmt == "mxfp4" else 1, 2 if dtype == torch.bfloat16 else 1
    assert L.tcq_ms_grouped_linear_workspace_bytes(rows, e, n, k, d, f, 1) == 0 and L.tcq_ms_grouped_linear_workspace_bytes(rows, e, n, k, d, f, 0) == rows * k * 2
    ws = torch.empty(rows * k * 2, dtype=torch.uint8, device=DEV)
    for loads in (0, 1, 2, 3, 5, 1000):
        y = torch.zeros(rows, n, dtype=dtype, device=DEV)
        rc = L.tcq_selftest_ms_grouped_waits(loads, x.data_ptr(), d, rows, k, None if tokens is None else tokens.data_ptr(), offsets.data_ptr(), e, rows, w.codes.data_ptr(), w.scales.data_ptr(),
                                             None if w.row_scale is None else w.row_scale.data_ptr(), n, k, f, None, 0, 0, None, 0, y.data_ptr(), d, n, ws.data_ptr(), rows * k * 2,
                                             torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        right = y == want
        assert bool((y.isnan() | right).all())
        if loads < 2:
            assert bool(y.isnan().all())
        elif n == 1500 or loads == 1000:
            assert bool(right.all())
        else:
            assert bool(y.isnan().any()) and bool(right.any())
    assert torch.equal(experts.grouped_linear(x, w, offsets, tokens), want)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("t", [3, 60])
def test_a_layer_whose_inner_results_leave_fp16(t, fmt):
    """fp16 tokens whose gated results are beyond 65504, and whose outputs are not: with a bf16 inner type they are right.  Off by the rounding of the inner results, 2^-9, and of the last
    ones, 2^-12, of each one's size: in norm no more than their sum, taken twice."""
    import moe_plain as plain
    from trellis_b200 import experts, microscale as ms
    from trellis_b200.quant import MicroscaledExperts
    g = torch.Generator(device=DEV).manual_seed(t)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    e, n, k, out = 3, 64, 96, 40
    up, gate, down = rnd(e, n, k), rnd(e, n, k), rnd(e, out, n) * 1e-3
    x, logits = (rnd(t, k) * 60).half(), rnd(t, e)
    m = MicroscaledExperts(up, down, 2, gate, fmt, inner=torch.bfloat16)
    y = m(x, logits)
    weights, chosen, *_ = plain.route(logits, 2, "softmax", True)
    uv, dv = ([ms.dequantize(experts.expert(q, i)).double() for i in range(e)] for q in (m.up, m.down))
    want, most = torch.zeros(t, out, dtype=torch.float64, device=DEV), 0.0
    for i in range(t):
        for j in range(2):
            h = x[i].double() @ uv[chosen[i, j]].t()
            h = plain.activate(h[0::2], "silu") * h[1::2]
            most = max(most, float(h.abs().max()))
            want[i] += weights[i, j] * (h @ dv[chosen[i, j]].t())
    assert most > 70000 and float(want.abs().max()) < 60000 and y.dtype == torch.float16
    assert bool(y.isfinite().all()) and float((y.double() - want).norm() / want.norm()) < 2 * (2.0 ** -9 + 2.0 ** -12)
    assert not bool(MicroscaledExperts(up, down, 2, gate, fmt)(x, logits).isfinite().all())
    old = MicroscaledExperts(up, down, 2, gate, fmt)
    del old.__dict__["inner"]
    assert torch.equal(old(x.bfloat16(), logits), MicroscaledExperts(up, down, 2, gate, fmt)(x.bfloat16(), logits))
    with pytest.raises(ValueError):
        MicroscaledExperts(up, down, 2, gate, fmt, inner=torch.float32)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [1, 2, 3, 20, 60, 300])
def test_the_largest_and_the_least_numbers(m, fmt):
    """bf16 numbers up to the largest, and down to the least normal ones, times weights of 1: themselves, and nothing infinite on the way."""
    from trellis_b200 import experts, microscale as ms
    g = torch.Generator(device=DEV).manual_seed(m)
    k = 64
    w = torch.eye(k, device=DEV)[None]
    q = experts.quantize_experts(w, fmt)
    wv = ms.dequantize(experts.expert(q, 0)).double().diagonal()
    q = q._replace(row_scale=q.row_scale / wv.float()) if fmt == "nvfp4" else q          # exactly one, or as near as fp32 comes
    wv = ms.dequantize(experts.expert(q, 0)).double().diagonal()
    for low, high in ((1.0, 1.99), (1.40, 1.46), (1.5, 1.75)):
        for power in (127, 126, 0, -100):
            x = (torch.rand(m, k, generator=g, device=DEV) * (high - low) + low).bfloat16().double().clamp(max=1.9921875) * 2.0 ** power * torch.randn(m, k, generator=g, device=DEV).sign()
            x = x.to(torch.bfloat16)
            y = experts.grouped_linear(x, q, torch.tensor([0, m], device=DEV).int(), dtype=torch.float32)
            want = x.double() * wv
            assert bool(x.isfinite().all()) and bool(((y.double() - want).abs() <= want.abs() * 2.0 ** -22).all()), (low, power)
