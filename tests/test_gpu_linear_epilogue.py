"""``microscale.linear`` with bias, activation and residual against the definition in 64 bits."""
import moe_plain as plain
import ms_cases
import pytest
import torch

pytestmark = pytest.mark.gpu
ACTS = (None, "relu", "gelu", "gelu_tanh", "silu", "geglu", "swiglu")
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def case(m, n, k, fmt, dtype, act, bias, residual, seed=0):
    from trellis_b200 import microscale as ms
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = ms.quantize(rnd(n, k) * k ** -0.5, fmt)
    x = (rnd(m, k) * torch.exp(rnd(k))).to(dtype)
    b = None if bias is None else rnd(n).to(bias)
    r = rnd(m, n // 2 if act in plain.GATED else n).to(dtype) if residual else None
    return x, w, b, r


def check(y, x, w, b, act, r):
    from trellis_b200 import microscale as ms
    wv, xd = ms.dequantize(w).double(), x.double()
    bound = plain.fp32_bound(xd, wv) if x.dtype == torch.float32 else plain.sums_bound(xd, wv, w.fmt)
    want, bound = plain.epilogue(xd @ wv.t(), bound, b, act, r, x.dtype)
    assert y.dtype == x.dtype and y.shape == want.shape
    off = (y.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.3g} of what it may"


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m", [1, 5, 21, 22, 150])
def test_activations(m, dtype, act, fmt):
    from trellis_b200 import microscale as ms
    x, w, b, r = case(m, 260, 520, fmt, dtype, act, torch.float32, True)
    check(ms.linear(x, w, b, act, r), x, w, b, act, r)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 2, 16), (2, 127, 31), (3, 128, 32), (1, 129, 33), (2, 4096, 4096), (1, 4096, 12288), (10, 1000, 1111), (20, 256, 2048), (21, 130, 257),
                                   (42, 24, 256), (64, 1024, 1024), (100, 20000, 264), (333, 384, 1000), (1030, 640, 512)])
def test_sizes(m, n, k, dtype, fmt):
    from trellis_b200 import microscale as ms
    x, w, b, r = case(m, n, k, fmt, dtype, None, dtype, True)
    check(ms.linear(x, w, bias=b, residual=r), x, w, b, None, r)
    if n % 2 == 0:
        check(ms.linear(x, w, activation="swiglu"), x, w, None, "swiglu", None)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 700), (2, 5000, 2048), (9, 128, 4096), (21, 1111, 1000), (64, 512, 512), (200, 2048, 768), (700, 300, 300)])
def test_whole_numbers_are_exact(m, n, k, fmt):
    """Sums of whole numbers that fp32 holds: the results are theirs, bit for bit, and so are those of any other way to add them."""
    from trellis_b200 import microscale as ms
    w, wv = ms_cases.whole_matrix(n, k, fmt, 1)
    x = ms_cases.whole_tokens(m, k, torch.bfloat16, 2)
    b = torch.randint(-50, 50, (n,), device="cuda").float()
    want = x.double() @ wv.t() + b.double()
    assert torch.equal(ms.linear(x, w, bias=b), want.to(torch.bfloat16))
    assert torch.equal(ms.linear(x.half(), w, bias=b, activation="relu"), want.clamp(min=0).half())


@pytest.mark.parametrize("m", [1, 4, 30, 300])
def test_strides_and_addresses(m):
    """Rows at any distance and address, results for more axes; what lies between rows is not read."""
    from trellis_b200 import microscale as ms
    x, w, b, r = case(m, 130, 333, "nvfp4", torch.bfloat16, None, torch.float32, True)
    want = ms.linear(x, w, b, "silu", r)
    for off in (1, 8):
        pad = torch.full((m, 333 + 11), float("nan"), dtype=x.dtype, device="cuda")
        pad[:, off:off + 333] = x
        rp = torch.full((m, 130 + 5), float("nan"), dtype=x.dtype, device="cuda")
        rp[:, 3:133] = r
        assert torch.equal(ms.linear(pad[:, off:off + 333], w, b, "silu", rp[:, 3:133]), want)
    assert torch.equal(ms.linear(x.t().contiguous().t(), w, b, "silu", r.t().contiguous().t()), want)
    assert torch.equal(ms.linear(x.reshape(1, m, 1, 333), w, b.double().float().expand(2, 130)[0], "silu", r.reshape(1, m, 1, 130)), want.reshape(1, m, 1, 130))
    assert torch.equal(ms.linear(x[0], w, b, "silu", r[0]).reshape(1, -1), ms.linear(x[:1], w, b, "silu", r[:1]))


def test_no_tokens_no_rows_no_columns():
    from trellis_b200 import microscale as ms
    x, w, b, r = case(3, 64, 32, "mxfp4", torch.bfloat16, None, torch.float32, True)
    assert ms.linear(x[:0], w, b, "relu").shape == (0, 64)
    empty = ms.quantize(torch.zeros(0, 32, device="cuda"), "mxfp4")
    assert ms.linear(x, empty, activation="swiglu").shape == (3, 0)
    none = ms.quantize(torch.zeros(64, 0, device="cuda"), "nvfp4")
    for dtype in DTYPES:
        got = ms.linear(torch.zeros(3, 0, dtype=dtype, device="cuda"), none, b, "relu", r.to(dtype))
        assert torch.equal(got, (b.clamp(min=0) + r.float()).to(dtype))
        assert got.dtype == dtype


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [3, 25])
def test_not_finite_rows(m, fmt):
    """A token with a NaN or an infinity gives NaN, the others what they give without it."""
    from trellis_b200 import microscale as ms
    x, w, b, r = case(m, 200, 300, fmt, torch.bfloat16, None, torch.float32, True)
    want = ms.linear(x, w, b, "gelu", r)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[1, 37] = bad
        got = ms.linear(y, w, b, "gelu", r)
        assert bool(got[1].isnan().all())
        keep = [i for i in range(m) if i != 1]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_not_finite_rows_of_many(fmt):
    """The same among many tokens, where an infinity may also give what its sums have."""
    from trellis_b200 import microscale as ms
    x, w, b, _ = case(300, 200, 300, fmt, torch.bfloat16, None, torch.float32, False)
    want = ms.linear(x, w, b)
    y = x.clone()
    y[1, 37], y[40, 299], y[299, 0] = float("nan"), float("inf"), -float("inf")
    got = ms.linear(y, w, b)
    exact = y[[40, 299]].double() @ ms.dequantize(w).double().t() + b.double()
    assert bool(got[1].isnan().all()) and bool((got[[40, 299]].isnan() | (got[[40, 299]] == exact)).all())
    keep = [i for i in range(300) if i not in (1, 40, 299)]
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("power", [-100, -30, 30, 100])
def test_size_of_activations(power, fmt):
    """A power of two in x is one in the results, exactly."""
    from trellis_b200 import microscale as ms
    x, w, _, _ = case(5, 200, 300, fmt, torch.bfloat16, None, None, False)
    want = ms.linear(x, w, activation="relu")
    assert torch.equal(ms.linear((x.float() * 2.0 ** power).bfloat16(), w, activation="relu"), (want.float() * 2.0 ** power).bfloat16())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_outliers_leave_the_others(fmt):
    """One channel a thousand times the others, whose weights are zero: what is left of the others is within the bound, and near bf16's own."""
    from trellis_b200 import microscale as ms
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(128, 512, generator=g, device="cuda")
    w[:, 100] = 0
    q = ms.quantize(w, fmt)
    x = torch.randn(4, 512, generator=g, device="cuda")
    x[:, 100] = 1000
    x = x.bfloat16()
    y = ms.linear(x, q, bias=torch.zeros(128, device="cuda"))
    check(y, x, q, None, None, None)
    want = x.double() @ ms.dequantize(q).double().t()
    assert float((y.double() - want).norm() / want.norm()) < 2.0 ** -8


def test_fp32_is_the_product_with_the_epilogue_behind():
    from trellis_b200 import microscale as ms
    x, w, b, r = case(12, 64, 96, "nvfp4", torch.float32, None, torch.float16, True)
    assert torch.equal(ms.linear(x, w, b, "relu", r), torch.relu(ms.linear(x, w) + b.float()) + r)


def test_captured_on_another_stream():
    from trellis_b200 import microscale as ms
    x, w, b, r = case(6, 512, 2048, "mxfp4", torch.float16, "swiglu", torch.float16, True)
    want = ms.linear(x, w, b, "swiglu", r)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(ms.linear(x, w, b, "swiglu", r), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        y = ms.linear(static, w, b, "swiglu", r)
    for seed in (1, 2):
        x2, _, _, _ = case(6, 512, 2048, "mxfp4", torch.float16, "swiglu", None, False, seed)
        static.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ms.linear(x2, w, b, "swiglu", r))
