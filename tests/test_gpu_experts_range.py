"""Grouped products at the ends of what they take: offsets and row numbers that point anywhere, sizes of weights and activations, matrices that are not finite, many groups, long rows."""
import moe_plain as plain
import ms_cases
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(e, rows, n, k, fmt, seed=0, dtype=torch.bfloat16):
    from trellis_b200 import experts
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = experts.quantize_experts(torch.randn(e, n, k, generator=g, device=DEV) * k ** -0.5, fmt)
    return w, torch.randn(rows, k, generator=g, device=DEV).to(dtype)


def into(x, w, offsets, tokens=None, act=0):
    """The product into a result that holds sevens."""
    from trellis_b200 import microscale as ms
    e, n, k = w.shape
    rows = x.shape[0] if tokens is None else tokens.shape[0]
    y = torch.full((rows, n), 7.0, dtype=x.dtype, device=DEV)
    ms._grouped(0, x, tokens, torch.tensor(offsets, dtype=torch.int32, device=DEV), e, rows, w.codes, w.scales, w.row_scale, n, k, w.fmt, None, act, None, y)
    return y


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows", [3, 12, 50, 2000])
def test_offsets_that_point_anywhere(rows, fmt):
    """In every form: rows of no group stay as they are, falling offsets and offsets outside the rows reach no further than they may."""
    from trellis_b200 import experts
    w, x = case(4, rows, 136, 264, fmt)
    a, b, c = rows // 3, rows // 2, rows - 1
    full = experts.grouped_linear(x, w, torch.tensor([0, a, b, c, rows], device=DEV).int())
    assert torch.equal(into(x, w, [-5, a, b, c, 1 << 30]), full) and torch.equal(into(x, w, [-(1 << 31), a, b, c, (1 << 31) - 1]), full)
    y = into(x, w, [a, a, b, c, c])
    assert torch.equal(y[a:c], full[a:c]) and bool((y[:a] == 7).all()) and bool((y[c:] == 7).all())
    y = into(x, w, [0, a, b, a, 0])                                       # as [0, a, b, b, b]
    assert torch.equal(y[:b], full[:b]) and bool((y[b:] == 7).all())
    for nothing in ([rows] * 5, [0] * 5, [rows + 1, -3, 5, 2, 0], [1 << 30, 0, 1, 2, 3]):
        assert bool((into(x, w, nothing) == 7).all())
    one = into(x, w, [0, 0, 0, 0, rows])                                  # all to the last
    assert torch.equal(one, experts.grouped_linear(x, w, torch.tensor([0, 0, 0, 0, rows], device=DEV).int()))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows", [3, 12, 50, 2000])
def test_tokens_that_point_anywhere(rows, fmt):
    w, x = case(2, 7, 136, 264, fmt)
    g = torch.Generator(device=DEV).manual_seed(rows)
    tokens = torch.randint(0, 7, (rows,), generator=g, device=DEV).int()
    offsets = [0, rows // 3, rows]
    want = into(x, w, offsets, tokens)
    bad = tokens.clone()
    at = [0, rows // 2, rows - 1]
    bad[at] = torch.tensor([-1, 7, (1 << 31) - 1], device=DEV).int()
    y = into(x, w, offsets, bad)
    keep = [i for i in range(rows) if i not in at]
    assert bool(y[at].isnan().all()) and torch.equal(y[keep], want[keep])
    assert bool(into(x[:0], w, offsets, tokens).isnan().all())             # an x without rows


@pytest.mark.parametrize("rows", [2, 20, 300])
@pytest.mark.parametrize("power", [-90, -30, 30, 90])
def test_sizes_of_weights(power, rows):
    """Powers of two in the row scales (nvfp4) or block scales (mxfp4) are powers of two in the results, exactly, against activations that make up for them."""
    from trellis_b200 import experts
    for fmt in ("mxfp4", "nvfp4"):
        w, x = case(3, rows, 136, 264, fmt)
        offsets = torch.tensor([0, 1, rows // 2, rows], device=DEV).int()
        want = experts.grouped_linear(x, w, offsets, dtype=torch.float32)
        if fmt == "nvfp4":
            v = w._replace(row_scale=w.row_scale * 2.0 ** power)
        else:
            v = w._replace(scales=torch.where(w.scales > 0, w.scales.int() + power, 0).to(torch.uint8))
        assert torch.equal(experts.grouped_linear(x, v, offsets, dtype=torch.float32), want * 2.0 ** power)
        small = (x.float() * 2.0 ** -power).bfloat16()
        assert torch.equal(experts.grouped_linear(small, v, offsets, dtype=torch.float32), want)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows", [2, 20, 300])
def test_weights_that_are_not_finite(rows, fmt):
    """A NaN in a row of one matrix is that result's of that group's rows, and nobody else's."""
    from trellis_b200 import experts, microscale as ms
    g = torch.Generator(device=DEV).manual_seed(0)
    m = torch.randn(2, 200, 256, generator=g, device=DEV)
    x = torch.randn(rows, 256, generator=g, device=DEV).bfloat16()
    offsets = torch.tensor([0, rows // 2, rows], device=DEV).int()
    want = experts.grouped_linear(x, experts.quantize_experts(m, fmt), offsets)
    m[1, 130, 77] = float("nan")
    got = experts.grouped_linear(x, experts.quantize_experts(m, fmt), offsets)
    assert bool(got[rows // 2:, 130].isnan().all())
    got[rows // 2:, 130] = want[rows // 2:, 130]
    assert torch.equal(got, want)
    assert not bool(ms.linear(x, ms.quantize(m[0], fmt), activation="relu").isnan().any())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_small_blocks_beside_large_ones(fmt):
    """Blocks of a token up to 2^40 apart: each within the bound, and exact as far as its digits reach."""
    from trellis_b200 import microscale as ms
    g = torch.Generator(device=DEV).manual_seed(0)
    q, wv = ms_cases.whole_matrix(130, 512, fmt, 3)
    for m in (1, 5):
        x = torch.randint(-8, 9, (m, 512), generator=g, device=DEV).double() * torch.exp2(-(torch.arange(512, device=DEV) // 32 * 2.6).floor())
        x = x.bfloat16()
        y = ms.linear(x, q, bias=torch.zeros(130, device=DEV))
        want, bound = plain.epilogue(x.double() @ wv.t(), plain.sums_bound(x.double(), wv, fmt), None, None, None, torch.bfloat16)
        assert bool(((y.double() - want).abs() <= bound).all())


def test_many_groups():
    """1024 groups, most of them without rows."""
    from trellis_b200 import experts
    w, x = case(1024, 70, 32, 64, "mxfp4")
    g = torch.Generator(device=DEV).manual_seed(5)
    r = experts.route(torch.randn(70, 1024, generator=g, device=DEV), 1)
    y = experts.grouped_linear(x, w, r.offsets, r.tokens, dtype=torch.float32)
    e = r.experts[:, 0].long()
    from trellis_b200 import microscale as ms
    for i in range(70):
        one = ms.dequantize(experts.expert(w, int(e[i]))).double()
        xd = x[i:i + 1].double()
        want, bound = plain.epilogue(xd @ one.t(), plain.sums_bound(xd, one, "mxfp4"), None, None, None, torch.float32)
        assert bool(((y[int(r.places[i, 0])].double() - want[0]).abs() <= bound[0]).all())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k", [(1, 10752), (1, 11000), (2, 8192), (2, 8200), (2, 20000), (3, 40000), (40, 30000)])
def test_long_rows(m, k, fmt):
    """Rows that a CTA holds and rows that it does not, whole numbers: bit for bit."""
    from trellis_b200 import microscale as ms
    w, wv = ms_cases.whole_matrix(140, k, fmt, 1)
    x = ms_cases.whole_tokens(m, k, torch.bfloat16, 2)
    want = x.double() @ wv.t()
    assert float(want.abs().max()) < 2 ** 22 and torch.equal(ms.linear(x, w, bias=torch.zeros(140, device=DEV)), want.to(torch.bfloat16))


def test_calls_in_turn_on_one_stream():
    """Kernels begin while the one before ends: what one writes, the next one reads, call after call, captured or not."""
    from trellis_b200 import experts, microscale as ms
    g = torch.Generator(device=DEV).manual_seed(0)
    a, av = ms_cases.whole_matrix(256, 256, "mxfp4", 1)
    up, down = (experts.quantize_experts(torch.randn(8, *s, generator=g, device=DEV) * 0.1, "nvfp4") for s in ((256, 256), (256, 128)))
    xs = [torch.randn(4, 256, generator=g, device=DEV).bfloat16() for _ in range(3)]

    def chain(x, wait):
        for _ in range(6):
            x = ms.linear(x, a, activation="relu") * 2.0 ** -10
            wait()
            r = experts.route(x[:, :8], 2)
            wait()
            h = experts.grouped_linear(x, up, r.offsets, r.tokens, activation="swiglu")
            wait()
            y = experts.grouped_linear(h, down, r.offsets, dtype=torch.float32)
            wait()
            x = experts.combine(y, r, x)
            wait()
        return x
    want = [chain(x, torch.cuda.synchronize) for x in xs]
    for _ in range(5):
        assert all(torch.equal(chain(x, lambda: None), y) for x, y in zip(xs, want))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(static, lambda: None)
    for x, y in zip(xs, want):
        static.copy_(x)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("n", [3850, 3970, 4096])
@pytest.mark.parametrize("rows,counts", [(100, [25, 25, 25, 25]), (100, [0, 1, 60, 39]), (100, [100, 0, 0, 0]), (100, [18, 21, 22, 39])])
def test_matrices_of_many_rows(rows, counts, n, fmt, dtype):
    """More items than SMs, in halves of 128 rows of a matrix, its last one alone or not whole, with rows of x gathered and not."""
    from trellis_b200 import experts
    w, x = case(4, rows, n, 296, fmt, dtype=dtype)
    offsets = torch.tensor([0, *counts], device=DEV).cumsum(0).int()
    y, back = experts.grouped_linear(x, w, offsets, dtype=torch.float32), torch.arange(rows - 1, -1, -1, device=DEV).int()
    assert torch.equal(experts.grouped_linear(x[back.long()], w, offsets, back, dtype=torch.float32), y)
    bias, gated = torch.randn(4, n, device=DEV), experts.grouped_linear(x, w, offsets, activation="swiglu")
    with_bias = experts.grouped_linear(x, w, offsets, bias=bias)
    at = offsets.tolist()
    for e in range(4):
        i, j = at[e], at[e + 1]
        from trellis_b200 import microscale as ms
        one, xd = ms.dequantize(experts.expert(w, e)).double(), x[i:j].double()
        if i == j:
            continue
        h, b = xd @ one.t(), plain.sums_bound(xd, one, fmt)
        for got, bi, act, dt in ((y, None, None, torch.float32), (gated, None, "swiglu", dtype), (with_bias, bias[e], None, dtype)):
            want, bound = plain.epilogue(h, b, bi, act, None, dt)
            assert bool(((got[i:j].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_many_items_for_each_sm(fmt):
    """Every group's result is that of its rows alone: sums of 64 columns, so that no form adds them in another order."""
    from trellis_b200 import experts
    e, rows, n = 96, 1500, 1182
    w, x = case(e, rows, n, 64, fmt)
    g = torch.Generator(device=DEV).manual_seed(3)
    offsets = torch.cat([torch.zeros(1, device=DEV), torch.randint(0, e, (rows,), generator=g, device=DEV).bincount(minlength=e).cumsum(0)]).int()
    y, at = experts.grouped_linear(x, w, offsets, dtype=torch.float32), offsets.tolist()
    for i in range(e):
        if at[i] < at[i + 1]:
            mine = w._replace(codes=w.codes[i:i + 1], scales=w.scales[i:i + 1], row_scale=None if w.row_scale is None else w.row_scale[i:i + 1], shape=(1, n, 64))
            assert torch.equal(experts.grouped_linear(x[at[i]:at[i + 1]], mine, torch.tensor([0, at[i + 1] - at[i]], device=DEV).int(), dtype=torch.float32), y[at[i]:at[i + 1]])


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_waits_for_matrices_of_many_rows_that_run_out(fmt):
    """Loads that never come where a CTA has several items: the kernel ends, and what needed them is NaN; the next call is right."""
    from trellis_b200 import _lib, experts
    e, rows, n, k = 8, 200, 4000, 512
    w, x = case(e, rows, n, k, fmt)
    offsets = torch.arange(0, rows + 1, rows // e, device=DEV).int()
    want = experts.grouped_linear(x, w, offsets)
    L, f = _lib.lib(), 0 if fmt == "mxfp4" else 1
    size = L.tcq_ms_grouped_linear_workspace_bytes(rows, e, n, k, 2, f, 1)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    for loads in (0, 1, 2, 3):                                    # two a first item
        y = torch.zeros(rows, n, dtype=torch.bfloat16, device=DEV)
        rc = L.tcq_selftest_ms_grouped_waits(loads, x.data_ptr(), 2, rows, k, None, offsets.data_ptr(), e, rows, w.codes.data_ptr(), w.scales.data_ptr(),
                                             None if w.row_scale is None else w.row_scale.data_ptr(), n, k, f, None, 0, 0, None, 0, y.data_ptr(), 2, n, ws.data_ptr(), size,
                                             torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert bool((y.isnan() | (y == want)).all()) and bool(y.isnan().any()) and (loads < 2 or bool((y == want).any()))
    assert torch.equal(experts.grouped_linear(x, w, offsets), want)


@pytest.mark.parametrize("rows,n,k,dtype", [(66000, 33000, 64, torch.bfloat16), (1050000, 40, 2056, torch.float16), (1050000, 130, 2049, torch.bfloat16)])
def test_more_bytes_than_31_bits_count(rows, n, k, dtype):
    """Results, or rows of x (where they lie, and put in order), of more than 2^31 bytes: the first and last rows and one between, which are other forms' than a small call's."""
    from trellis_b200 import experts, microscale as ms
    fmt = "nvfp4"
    g = torch.Generator(device=DEV).manual_seed(0)
    w = experts.quantize_experts(torch.randn(2, n, k, generator=g, device=DEV) * k ** -0.5, fmt)
    x = torch.empty(rows, k, dtype=dtype, device=DEV)
    ends = torch.randn(600, k, generator=g, device=DEV).to(dtype)
    x[:300], x[300:-300], x[-300:] = ends[:300], 1, ends[300:]
    y = experts.grouped_linear(x, w, torch.tensor([0, 300, rows], device=DEV).int(), activation="swiglu")
    assert rows * max(n // 2, k) > 2 ** 30
    for e, at in ((0, slice(0, 300)), (1, slice(rows // 2, rows // 2 + 1)), (1, slice(rows - 300, rows))):
        one, xd = ms.dequantize(experts.expert(w, e)).double(), x[at].double()
        want, bound = plain.epilogue(xd @ one.t(), plain.sums_bound(xd, one, fmt), None, "swiglu", None, dtype)
        assert bool(((y[at].double() - want).abs() <= bound).all())


def test_combining_more_numbers_than_31_bits_count():
    from trellis_b200 import experts
    for n in (2048, 2051):
        tokens, g = 1060000, torch.Generator(device=DEV).manual_seed(0)
        y = torch.randn(64, n, generator=g, device=DEV).bfloat16()
        places = torch.randint(0, 64, (tokens, 2), generator=g, device=DEV).int()
        weights = torch.rand(tokens, 2, generator=g, device=DEV)
        out = experts.combine(y, experts.Routing(weights, places, places, places.flatten(), places.flatten()))
        assert out.numel() > 2 ** 31
        for at in (slice(0, 40), slice(tokens // 2, tokens // 2 + 40), slice(tokens - 40, tokens)):
            p, v = places[at].contiguous(), weights[at].contiguous()
            assert torch.equal(out[at], experts.combine(y, experts.Routing(v, p, p, p.flatten(), p.flatten())))
