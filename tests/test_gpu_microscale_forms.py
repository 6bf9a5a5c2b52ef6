"""Every form of the microscaled products at sizes that the launch rules send to it, ragged on all sides, several tiles a CTA where the form has them.

Whole numbers throughout: sums are exact in fp32 in any order, so a result is the real one, rounded once.  The tables name the form (the kernel's template
arguments) that each size takes on 148 SMs, and one test holds them against the kernels that run.
"""
import re

import pytest
import torch

from ms_cases import BLOCK, whole_matrix, whole_tokens

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MX, NV = 0, 1                                                    # the kernels' numbers of the formats
NAMES = ("mxfp4", "nvfp4")
TYPES = {F32: "float", F16: "__half", BF16: "__nv_bfloat16"}

# Few tokens: (type, format, m, n, k) -> parts of x, stages of W.  Whole groups of 128 rows in turns; beside two stages x is held whole.
FEW = [((t, f, m, n, k), (p, s)) for f in (MX, NV) for t, m, n, k, p, s in (
    (BF16, 3, 76001, 515, 1, 3), (BF16, 8, 40001, 4000, 1, 2), (F16, 5, 76001, 300, 1, 3), (F16, 7, 40001, 4111, 1, 2), (F32, 3, 76001, 515, 3, 3), (F32, 8, 40001, 1111, 3, 2))]

# More tokens: -> rows of x in a tile, parts, fp16 products.  128 rows of x only where all tiles run at once.
MANY = ([((t, f, m, n, k), (nt, 1, t is F16)) for t, f in ((BF16, MX), (BF16, NV), (F16, NV)) for m, n, k, nt in (
    (13, 76001, 330, 16), (27, 76001, 330, 32), (50, 76001, 515, 64), (100, 9001, 200, 128), (90, 3001, 1111, 128), (300, 20001, 330, 256), (777, 12001, 300, 256))]
        + [((F16, MX, m, n, k), (nt, 2, False)) for m, n, k, nt in ((15, 76001, 330, 32), (30, 76001, 330, 64), (60, 9001, 515, 128), (120, 20001, 330, 256))]
        + [((F16, MX, m, n, k), (nt, 1, True)) for m, n, k, nt in ((140, 6001, 330, 128), (300, 20001, 515, 256), (1000, 12289, 320, 256))]
        + [((F32, f, m, n, k), (nt, 3, False)) for f in (MX, NV) for m, n, k, nt in ((10, 40001, 515, 32), (21, 40001, 330, 64), (50, 20001, 1111, 64))])

# Both sides in 4 bits: (format, m, n, k) -> tokens of a tile on one SM, or rows of W on a pair.
ONE = [((f, m, n, k), nt) for f in (MX, NV) for m, n, k, nt in ((3, 76001, 515, 8), (12, 76001, 330, 16), (30, 40001, 515, 32), (60, 40001, 300, 64), (100, 20001, 515, 128), (128, 9001, 8001, 128))]
PAIR = [((f, m, n, k), nt) for f in (MX, NV) for m, n, k, nt in ((300, 9701, 515, 128), (100, 4001, 1111, 128), (2100, 12201, 300, 256), (600, 24001, 4111, 256))]


def _of(case, form):
    """The kernel of a case, by name and template arguments."""
    if form[0] in ("few", "many"):
        t, f, *_ = case
        args = (TYPES[t], f, *form[1]) if form[0] == "few" else (TYPES[t], f, *form[1][:2], str(form[1][2]).lower())
        return f"tcq_ms_linear_{form[0]}_kernel<{', '.join(map(str, args))}>"
    return f"tcq_ms_{'matmul' if form[0] == 'one' else 'pair'}_kernel<{case[0]}, {form[1]}>"


LINEAR = [(c, ("few", f)) for c, f in FEW] + [(c, ("many", f)) for c, f in MANY]
MATMUL = [(c, ("one", f)) for c, f in ONE] + [(c, ("pair", f)) for c, f in PAIR]


@pytest.fixture(scope="module")
def ms():
    from trellis_b200 import microscale
    return microscale


def _exact(want, dtype):
    return want.to(dtype)                                        # (sums are whole multiples of 2^-6 below 2^24: fp64 and fp32 have them)


@pytest.mark.parametrize("case,form", LINEAR, ids=[_of(c, f) + "-" + "-".join(map(str, c[2:])) for c, f in LINEAR])
def test_linear_of_every_form(ms, case, form):
    dtype, f, m, n, k = case
    w, wv = whole_matrix(n, k, NAMES[f], n + k)
    x = whole_tokens(m, k, dtype, m)
    want = _exact(x.double() @ wv.t(), dtype)
    assert torch.equal(ms.linear(x, w), want)
    wide = torch.full((m, k + 9), float("nan"), dtype=dtype, device="cuda")       # rows at another address, among NaN
    wide[:, 3:3 + k] = x
    assert torch.equal(ms.linear(wide[:, 3:3 + k], w), want)


@pytest.mark.parametrize("case,form", MATMUL, ids=[_of(c, f) + "-" + "-".join(map(str, c[1:])) for c, f in MATMUL])
def test_matmul_of_every_form(ms, case, form):
    f, m, n, k = case
    (w, wv), (x, xv) = whole_matrix(n, k, NAMES[f], n + k), whole_matrix(m, k, NAMES[f], m)
    want = xv @ wv.t()
    for dtype in (F32, F16, BF16):
        assert torch.equal(ms.matmul(x, w, dtype), _exact(want, dtype)), dtype


@pytest.mark.parametrize("m,n,k", ((300, 20001, 515), (140, 6001, 330)))
def test_prompts_through_scales_too_far_apart_for_fp16(ms, m, n, k):
    """fp16 tokens, mxfp4 rows whose scales fp16 weights do not hold: the form of two bf16 parts, several tiles a CTA."""
    w, wv = whole_matrix(n, k, "mxfp4", n)
    scales = ms.block_scales(w).clone()
    scales[5::7, 3] = 127 - 40
    codes = w.codes[:, :-(-k // 2)]
    far = ms.from_blocks(codes, scales, None, k, "mxfp4")
    wv = wv.clone()
    old = ms.block_scales(w)[5::7, 3].double() - 127
    wv[5::7, 96:128] *= torch.exp2(-40 - old)[:, None]
    x = whole_tokens(m, k, F16, m)
    x[:, 96:128] = 0                                             # so that sums stay whole ...
    x[1::2] = 0
    x[1::2, 96:128] = whole_tokens(m, 32, F16, 1)[1::2] * 2.0 ** 12       # ... or are multiples of 2^-29 below 2^-15
    assert torch.equal(ms.linear(x, far), _exact(x.double() @ wv.t(), F16))


@pytest.mark.parametrize("m", (300, 777))
def test_prompts_repeat_and_do_not_mix(ms, m):
    """Several tiles a CTA, from three streams at once: equal bits every time, and rows that do not depend on the others."""
    n, k = 20001, 515
    calls = []
    for fmt in NAMES:
        w, _ = whole_matrix(n, k, fmt, 1)
        for t in (F16, BF16):
            x = torch.randn(m, k, generator=torch.Generator(device="cuda").manual_seed(m), device="cuda").to(t)
            calls.append(lambda x=x, w=w: ms.linear(x, w))
            other = x.clone()
            other[1:] *= 100
            assert torch.equal(ms.linear(other, w)[0], ms.linear(x, w)[0])
        q = ms.quantize(x, fmt)
        calls.append(lambda q=q, w=w: ms.matmul(q, w))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], {}
    for turn in range(3):
        for i, c in enumerate(calls):
            with torch.cuda.stream(streams[(i + turn) % 3]):
                got[turn, i] = c()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for (_, i), y in got.items())


def test_the_tables_name_the_kernels_that_run(ms):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the tables are for 148 SMs")
    from torch.profiler import ProfilerActivity, profile
    ran = {}
    with profile(activities=[ProfilerActivity.CUDA]):            # (the first session loses its kernels now and then)
        torch.zeros(1, device="cuda")
    for case, form in LINEAR + MATMUL:
        if form[0] in ("few", "many"):
            dtype, f, m, n, k = case
            call = lambda: ms.linear(x, w)
            x = torch.zeros(m, k, dtype=dtype, device="cuda")
        else:
            f, m, n, k = case
            x = _zeros(ms, m, k, f)
            call = lambda: ms.matmul(x, w)
        w = _zeros(ms, n, k, f)
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            call()
            torch.cuda.synchronize()
        ran[case, form] = {m[0] for e in prof.events() for m in [re.search(r"tcq_ms_\w+<[^>]*>", e.name)] if m}
    if not any(ran.values()):
        pytest.skip("no kernels recorded")
    for (case, form), names in ran.items():
        assert _of(case, form) in names, (case, names)


def _zeros(ms, rows, k, f):
    q = torch.zeros(rows, -(-k // 2), dtype=torch.uint8, device="cuda")
    return ms.from_blocks(q, torch.zeros(rows, -(-k // BLOCK[NAMES[f]]), dtype=torch.uint8, device="cuda"), None if f == MX else 1.0, k, NAMES[f])


@pytest.mark.parametrize("f", (MX, NV))
@pytest.mark.parametrize("op,m,n,k", (("matmul", 300, 9728, 515), ("matmul", 2100, 12288, 300), ("matmul", 100, 20000, 515), ("matmul", 5, 76000, 300), ("matmul", 20, 1024, 2304),
                                      ("linear", 300, 20000, 515), ("linear", 140, 6016, 330), ("linear", 50, 76000, 300), ("linear", 7, 76000, 300), ("linear", 40, 1024, 2304)))
def test_rows_of_results_with_room_behind_them(ms, f, op, m, n, k):
    """Results by the C entries, rows of any length and start: what lies behind column n and row m stays."""
    from trellis_b200 import _lib
    lib, stream, code = _lib.lib(), torch.cuda.current_stream().cuda_stream, {F32: 0, F16: 1, BF16: 2}
    w, wv = whole_matrix(n, k, NAMES[f], n)
    ptr = lambda t: None if t is None else t.data_ptr()
    weights = (w.codes.data_ptr(), w.scales.data_ptr(), ptr(w.row_scale))
    if op == "matmul":
        x, xv = whole_matrix(m, k, NAMES[f], m)
        want = xv @ wv.t()
    for dtype in (F32, F16, BF16):
        if op == "linear":
            x = whole_tokens(m, k, dtype, m)
            want = x.double() @ wv.t()
            ws = torch.empty(lib.tcq_ms_linear_workspace_bytes(m, n, k, code[dtype], f), dtype=torch.uint8, device="cuda")
        for ldy, start in ((n, 0), (n + 3, 1), (n + 8, 8), (n + 32, 0)):
            flat = torch.full((start + (m + 2) * ldy,), 77.0, dtype=dtype, device="cuda")
            y = flat[start:].view(m + 2, ldy)
            if op == "matmul":
                rc = lib.tcq_ms_matmul(x.codes.data_ptr(), x.scales.data_ptr(), ptr(x.row_scale), m, *weights, n, k, f, y.data_ptr(), code[dtype], ldy, stream)
            else:
                rc = lib.tcq_ms_linear(x.data_ptr(), code[dtype], m, k, *weights, n, k, f, y.data_ptr(), ldy, ws.data_ptr(), ws.numel(), stream)
            assert rc == 0 and torch.equal(y[:m, :n], _exact(want, dtype)), (dtype, ldy, start)
            y[:m, :n] = 77.0
            assert (flat == 77).all()
