"""Mixtures of experts: grouped products, routing, combining and a whole layer against their definitions in 64 bits."""
import moe_plain as plain
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rnd(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def values(w):
    from trellis_b200 import experts, microscale as ms
    return torch.stack([ms.dequantize(experts.expert(w, e)) for e in range(w.shape[0])]).double()


def matrices(g, e, n, k, fmt):
    from trellis_b200 import experts
    return experts.quantize_experts(rnd(g, e, n, k) * k ** -0.5, fmt)


def offsets_of(counts):
    return torch.tensor([0] + counts, device=DEV).cumsum(0).int()


def check_grouped(y, x, w, offsets, tokens, bias, act, dtype):
    wv, rows = values(w), x if tokens is None else x[tokens.long()]
    bounds = offsets.tolist()
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if a < b:
            xd = rows[a:b].double()
            want, bound = plain.epilogue(xd @ wv[e].t(), plain.sums_bound(xd, wv[e], w.fmt), None if bias is None else bias[e], act, None, dtype)
            off = (y[a:b].double() - want).abs()
            assert bool((off <= bound).all()), f"expert {e}: off by {float((off / bound).max()):.3g} of what it may"


COUNTS = {"one each": [1] * 8, "one of many": [0] * 60 + [1] + [0] * 3, "ragged": [0, 5, 1, 0, 40, 22, 21, 0, 3, 64, 0], "all to the last": [0, 0, 0, 200], "many": [300, 0, 129, 1, 450],
          "even": [6] * 33, "single": [37], "two hundred": [1] * 100 + [2] * 50 + [0] * 50}


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("n,k,act", [(264, 520, "swiglu"), (130, 257, None), (1024, 256, "gelu")])
def test_grouped(name, n, k, act, fmt):
    from trellis_b200 import experts
    counts = COUNTS[name]
    g = torch.Generator(device=DEV).manual_seed(len(name))
    w = matrices(g, len(counts), n, k, fmt)
    for dtype in (torch.bfloat16, torch.float16):
        x = rnd(g, sum(counts), k).to(dtype)
        bias = rnd(g, len(counts), n).to(dtype)
        offsets = offsets_of(counts)
        y = experts.grouped_linear(x, w, offsets, bias=bias, activation=act)
        assert y.dtype == dtype
        check_grouped(y, x, w, offsets, None, bias, act, dtype)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("t,rows", [(1, 8), (7, 40), (50, 700), (600, 2000)])
def test_gathered_rows(t, rows, fmt):
    """Rows of x by number, the same ones several times, in fp32 results too; equal to the rows put in order first."""
    from trellis_b200 import experts
    g = torch.Generator(device=DEV).manual_seed(t)
    w = matrices(g, 8, 256, 384, fmt)
    x = rnd(g, t, 384).bfloat16()
    tokens = torch.randint(0, t, (rows,), generator=g, device=DEV).int()
    cuts = torch.sort(torch.randint(0, rows + 1, (7,), generator=g, device=DEV))[0].int()
    offsets = torch.cat((cuts.new_zeros(1), cuts, cuts.new_full((1,), rows)))
    y = experts.grouped_linear(x, w, offsets, tokens=tokens, dtype=torch.float32)
    assert y.dtype == torch.float32
    check_grouped(y, x, w, offsets, tokens, None, None, torch.float32)
    assert torch.equal(y, experts.grouped_linear(x[tokens.long()], w, offsets, dtype=torch.float32))


def test_each_group_is_a_linear_layer():
    """Whole numbers: grouped products equal those of each matrix by itself, bit for bit, at every size of group."""
    import ms_cases
    from trellis_b200 import experts, microscale as ms
    for fmt in ("mxfp4", "nvfp4"):
        parts = [ms_cases.whole_matrix(300, 500, fmt, s) for s in range(6)]
        w = experts.stack_experts([q for q, _ in parts])
        counts = [1, 0, 17, 90, 260, 3]
        offsets = offsets_of(counts)
        x = ms_cases.whole_tokens(sum(counts), 500, torch.bfloat16, 9)
        y = experts.grouped_linear(x, w, offsets, activation="relu", dtype=torch.float32)
        b = offsets.tolist()
        for e, (q, v) in enumerate(parts):
            assert torch.equal(y[b[e]:b[e + 1]].double(), (x[b[e]:b[e + 1]].double() @ v.t()).clamp(min=0))
            if counts[e]:
                assert torch.equal(ms.linear(x[b[e]:b[e + 1]], q, activation="relu"), y[b[e]:b[e + 1]].bfloat16())


def test_rows_of_no_group_are_left():
    """Rows before the first and behind the last offset are not written, offsets that fall or leave the rows reach no further, and tokens outside x give NaN."""
    from trellis_b200 import experts, microscale as ms
    g = torch.Generator(device=DEV).manual_seed(3)
    w = matrices(g, 4, 128, 256, "nvfp4")
    x = rnd(g, 50, 256).bfloat16()
    full = experts.grouped_linear(x, w, offsets_of([10, 20, 5, 15]))

    def into(offsets):
        y = torch.full((50, 128), 7.0, dtype=torch.bfloat16, device=DEV)
        ms._grouped(0, x, None, torch.tensor(offsets, dtype=torch.int32, device=DEV), 4, 50, w.codes, w.scales, w.row_scale, 128, 256, "nvfp4", None, 0, None, y)
        return y
    y = into([10, 10, 30, 35, 40])
    assert torch.equal(y[10:35], full[10:35]) and bool((y[:10] == 7).all()) and bool((y[40:] == 7).all())
    assert torch.equal(into([-5, 10, 30, 35, 1 << 30]), full)                                 # as far as there are rows
    assert torch.equal(into([0, 10, 30, 20, 10])[:30], full[:30]) and bool((into([0, 10, 30, 20, 10])[30:] == 7).all())
    assert bool((into([60, 70, 80, 90, 100]) == 7).all()) and bool((into([0, 0, 0, 0, 0]) == 7).all())
    tokens = torch.arange(50, device=DEV).int()
    tokens[[3, 20, 49]] = torch.tensor([-1, 50, 1 << 30], device=DEV).int()
    y = experts.grouped_linear(x, w, offsets_of([10, 20, 5, 15]), tokens=tokens)
    good = [i for i in range(50) if i not in (3, 20, 49)]
    assert torch.equal(y[good], full[good]) and bool(y[[3, 20, 49]].isnan().all())


def same_routing(r, want, top):
    weights, chosen, places, tokens, offsets = want
    assert torch.equal(r.experts.cpu().long(), chosen) and torch.equal(r.places.cpu().long(), places)
    assert torch.equal(r.tokens.cpu().long(), tokens) and torch.equal(r.offsets.cpu().long(), offsets)
    # exp of a difference that is rounded (2^-24 of up to about 90), and a sum of up to 1024
    off = (r.weights.cpu().double() - weights).abs()
    assert bool((off <= weights * 2.0 ** -16 + 2.0 ** -126).all() | weights.isnan().any()) and torch.equal(r.weights.cpu().isnan(), weights.isnan())


@pytest.mark.parametrize("score,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("t,e,top", [(0, 4, 2), (1, 1, 1), (1, 128, 8), (3, 2, 2), (5, 33, 5), (63, 61, 2), (64, 64, 6), (65, 65, 7), (200, 129, 8), (300, 16, 1), (70, 256, 32), (40, 300, 32),
                                     (100, 1024, 8), (1500, 7, 3)])
def test_route(t, e, top, score, normalize):
    from trellis_b200 import experts
    g = torch.Generator(device=DEV).manual_seed(t + e)
    for dtype in (torch.float32, torch.bfloat16):
        logits = (rnd(g, t, e) * 3).to(dtype)                     # (bf16: ties)
        same_routing(experts.route(logits, top, score, normalize), plain.route(logits, top, score, normalize), top)


@pytest.mark.parametrize("t", [9, 100])
def test_route_of_special_logits(t):
    from trellis_b200 import experts
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([[0.0, -0.0, 0.0, -0.0, 1e-45], [-inf] * 5, [-inf, 2.0, -inf, -inf, -inf], [nan, 1.0, 2.0, 3.0, 4.0], [-3e38, 3e38, -inf, -3e38, 3e38], [5.0] * 5, [-200.0, -201.0, -200.0, -inf, -300.0],
                         [-1e-40, -2e-40, 1e-40, 0.0, -inf], [1.0, -inf, -inf, -inf, 1.0]], device=DEV)
    logits = rows.repeat(-(-t // 9), 1)[:t].contiguous()
    for score in ("softmax", "sigmoid"):
        for normalize in (True, False):
            for top in (1, 3, 5):
                same_routing(experts.route(logits, top, score, normalize), plain.route(logits, top, score, normalize), top)
    wide = torch.full((t, 9), nan, device=DEV)
    wide[:, 2:7] = logits
    r, s = experts.route(wide[:, 2:7], 3), experts.route(logits, 3)
    assert all(torch.equal(a.nan_to_num(-9.0), b.nan_to_num(-9.0)) for a, b in zip(r, s))


@pytest.mark.parametrize("n", [1, 7, 8, 264, 2035])
@pytest.mark.parametrize("t,top", [(1, 8), (33, 1), (100, 5), (5, 32)])
def test_combine(t, top, n):
    from trellis_b200 import experts
    g = torch.Generator(device=DEV).manual_seed(n)
    rows = t * top
    for y_type, out_type in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16), (torch.float16, torch.float32)):
        y = rnd(g, rows, n).to(y_type)
        weights = rnd(g, t, top).abs()
        places = torch.randperm(rows, generator=g, device=DEV).reshape(t, top).int()
        places[0, top // 2] = -1
        y[rows - 1] = float("nan")                                # nobody's
        places[places == rows - 1] = -1
        r = experts.Routing(weights, places, places, places.flatten(), places.flatten())
        res = rnd(g, t, n).to(out_type)
        for residual in (None, res):
            got = experts.combine(y, r, residual, out_type)
            keep = (places >= 0)[..., None]
            parts = torch.where(keep, y.double()[places.clamp(min=0).long()], 0.0) * weights.double()[..., None]
            want = parts.sum(1) + (0 if residual is None else residual.double())
            info = torch.finfo(out_type)
            bound = (parts.abs().sum(1) + want.abs()) * (top + 2) * 2.0 ** -24
            bound = bound + (want.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps / 2
            assert got.dtype == out_type and bool(((got.double() - want).abs() <= bound).all())
        wide = torch.full((rows, n + 3), float("nan"), dtype=y_type, device=DEV)
        wide[:, 1:n + 1] = y
        assert torch.equal(experts.combine(wide[:, 1:n + 1], r, res), experts.combine(y, r, res))


def layer(x, logits, up, down, top, residual, act="swiglu"):
    from trellis_b200 import experts
    r = experts.route(logits, top)
    h = experts.grouped_linear(x, up, r.offsets, tokens=r.tokens, activation=act)
    return experts.combine(experts.grouped_linear(h, down, r.offsets, dtype=torch.float32), r, residual)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("t,e,top,n,k", [(1, 16, 4, 96, 320), (13, 8, 2, 130, 256), (300, 5, 3, 100, 200)])
def test_layer(t, e, top, n, k, fmt):
    """A whole layer, with padded tokens that go nowhere, against 64 bits: as far off as the rounding of what lies between is."""
    from trellis_b200 import experts
    g = torch.Generator(device=DEV).manual_seed(t)
    up, down = matrices(g, e, 2 * n, k, fmt), matrices(g, e, k, n, fmt)
    x, logits, res = rnd(g, t, k).bfloat16(), rnd(g, t, e) * 2, rnd(g, t, k).bfloat16()
    if t > 1:
        logits[t // 2] = -float("inf")
    out = layer(x, logits, up, down, top, res)
    weights, chosen, *_ = plain.route(logits, top, "softmax", True)
    uv, dv = values(up), values(down)
    want, bound = torch.zeros(t, k, dtype=torch.float64, device=DEV), torch.zeros(t, k, dtype=torch.float64, device=DEV)
    for i in range(t):
        for j in range(top):
            if chosen[i, j] >= 0:
                w, d = uv[chosen[i, j]], dv[chosen[i, j]]
                xd = x[i:i + 1].double()
                h, hb = plain.epilogue(xd @ w.t(), plain.sums_bound(xd, w, fmt), None, "swiglu", None, torch.bfloat16)
                y, yb = plain.epilogue(h @ d.t(), plain.sums_bound(h.abs() + hb, d, fmt) + hb @ d.abs().t(), None, None, None, torch.float32)
                want[i] += weights[i, j] * y[0]
                bound[i] += weights[i, j] * (yb[0] + y[0].abs() * 2.0 ** -15)
    want = want + res.double()
    bound = bound + want.abs() * (2.0 ** -8 + 2.0 ** -20)
    assert bool(((out.double() - want).abs() <= bound).all())
    if t > 1:
        assert torch.equal(out[t // 2], res[t // 2])


def test_captured_layer_follows_its_inputs():
    """One captured graph, replayed with other logits: the counts of rows are the GPU's business.  Two such graphs beside each other share nothing."""
    g = torch.Generator(device=DEV).manual_seed(0)
    up, down = matrices(g, 12, 256, 320, "nvfp4"), matrices(g, 12, 320, 128, "nvfp4")
    runs = []
    for t in (4, 90):
        x, logits, res = rnd(g, t, 320).half(), rnd(g, t, 12), rnd(g, t, 320).half()
        layer(x, logits, up, down, 3, res)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, logits, up, down, 3, res)
        runs.append((graph, x, logits, res, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        for graph, x, logits, res, out in runs:
            x.copy_(rnd(g, *x.shape))
            logits.copy_(rnd(g, *logits.shape))
        torch.cuda.synchronize()
        for stream, run in zip(streams, runs):
            with torch.cuda.stream(stream):
                run[0].replay()
        torch.cuda.synchronize()
        for graph, x, logits, res, out in runs:
            assert torch.equal(out, layer(x, logits, up, down, 3, res))


def test_calls_are_repeatable_beside_one_another():
    from trellis_b200 import experts
    g = torch.Generator(device=DEV).manual_seed(0)
    w = matrices(g, 16, 512, 1024, "mxfp4")
    x = rnd(g, 64, 1024).bfloat16()
    r = experts.route(rnd(g, 64, 16), 4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(experts.grouped_linear(x, w, r.offsets, tokens=r.tokens, activation="silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(y, got[0]) for y in got)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows,counts", [(3, [1, 2]), (40, [40]), (300, [100, 200])])
def test_waits_that_run_out(rows, counts, fmt):
    """Loads that never come: the kernel ends, and what needed them is NaN; the next call is right."""
    from trellis_b200 import _lib, experts
    g = torch.Generator(device=DEV).manual_seed(0)
    n, k = 200, 2048
    w = matrices(g, len(counts), n, k, fmt)
    x, offsets = rnd(g, rows, k).bfloat16(), offsets_of(counts)
    want = experts.grouped_linear(x, w, offsets)
    L = _lib.lib()
    f = 0 if fmt == "mxfp4" else 1
    size = L.tcq_ms_grouped_linear_workspace_bytes(rows, len(counts), n, k, 2, f, 1)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device=DEV)
    for loads in (0, 1, 3):                                       # of eight stages, which four CTAs share at most: one load is too few for any of them
        y = torch.zeros(rows, n, dtype=torch.bfloat16, device=DEV)
        rc = L.tcq_selftest_ms_grouped_waits(loads, x.data_ptr(), 2, rows, k, None, offsets.data_ptr(), len(counts), rows, w.codes.data_ptr(), w.scales.data_ptr(),
                                             None if w.row_scale is None else w.row_scale.data_ptr(), n, k, f, None, 0, 0, None, 0, y.data_ptr(), 2, n, ws.data_ptr(), size,
                                             torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert bool((y.isnan() | (y == want)).all()) and (loads > 1 or bool(y.isnan().any()))
    assert torch.equal(experts.grouped_linear(x, w, offsets), want)
