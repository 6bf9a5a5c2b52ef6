"""4-bit microscaled quantisation and products on the GPU, against their definition in 64 bits (``ms_plain``).

Tolerances.  Codes, scales and values are exact.  For a product over k columns in fp32, every order of summation, with rounding or
truncation of each of at most k + 8 sums and one rounding of each operand's scaling, is within (k + 16) * 2^-23 * sum |x w| of the
real sum; the result's rounding adds half a step, eps / 2 of it.  Where all sums are whole numbers below 2^24 times one power of two,
every order gives the same, and the only error is the result's rounding.
"""
import ctypes

import pytest
import torch

import ms_plain as P

pytestmark = pytest.mark.gpu
FMTS = ("mxfp4", "nvfp4")
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


@pytest.fixture(scope="module")
def ms():
    from trellis_b200 import microscale
    return microscale


def _same(q, x, fmt):
    codes, byte, row = P.quantize(x.cpu().double(), fmt)
    got = P.unpack(q)
    assert torch.equal(got[1], byte), "scales"
    assert torch.equal(got[0], codes), "codes"
    if fmt == "nvfp4":
        assert torch.equal(got[2], row), "row scales"
    else:
        assert q.row_scale is None
    return P.values(codes, byte, row, fmt)


def _matrix(rows, k, dtype, seed):
    """Values over many binades, with blocks and rows of zeros, ties, numbers of few bits and far outliers."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.ldexp(torch.ones(rows, 1), torch.randint(-6, 6, (rows, 1), generator=g))
    pick = torch.rand(rows, k, generator=g)
    x = torch.where(pick < 0.02, x * 30, x)
    x = torch.where((pick > 0.3) & (pick < 0.6), torch.randint(-24, 25, (rows, k), generator=g) / 4.0, x)
    x[torch.rand(rows, generator=g) < 0.1] = 0.0
    x[:, (k // 3):(k // 3 + 40)] *= (torch.rand(rows, 1, generator=g) < 0.7)
    return x.to(dtype).cuda()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", ((1, 1), (1, 16), (3, 17), (2, 31), (5, 32), (7, 33), (130, 257), (129, 256), (40, 700), (3, 4144), (2, 12293), (1, 40000)))
def test_quantize_and_back(ms, fmt, dtype, rows, k):
    x = _matrix(rows, k, dtype, rows * 1000 + k)
    q = ms.quantize(x, fmt)
    want = _same(q, x, fmt)
    for out in DTYPES:
        assert torch.equal(ms.dequantize(q, out).cpu(), want.to(out)), out


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_special_values(ms, fmt):
    inf, nan, big, tiny = float("inf"), float("nan"), 3.4028234663852886e38, 1e-45
    x = torch.zeros(12, 96)
    x[0, :7] = torch.tensor([0.0, -0.0, 1.0, -1.0, 0.25, -0.25, 6.0])
    x[1, 5], x[2, 40], x[3, 95] = inf, nan, -inf
    x[1, 40:60] = 0.3
    x[2, 0:8] = 5.0
    x[4] = big
    x[5] = tiny
    x[6, ::2] = 1e-38
    x[7, 3], x[7, 50] = big, 1.0
    x[8, 0], x[8, 64:] = 1e-30, 1e-40
    x[9] = nan
    x[10, :32] = torch.arange(32) / 4.0
    x[11, :], x[11, 7] = 1.17549435e-38, 2.0 ** -78
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype).cuda()
        q = ms.quantize(xd, fmt)
        want = _same(q, xd, fmt)
        back = ms.dequantize(q).cpu()
        assert torch.equal(torch.isnan(back), torch.isnan(want)) and torch.equal(back.nan_to_num(), want.float().nan_to_num())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lo,hi", ((0, 16), (16, 32)))
def test_quotients_next_to_borders(ms, fmt, lo, hi):
    """Every e4m3 mantissa times every border, and the fp32 numbers on both sides of the product."""
    rows = []
    for m in range(8):
        for border in P.BORDERS:
            t = torch.tensor((8 + m) / 8.0 * border)
            rows += [torch.nextafter(t, torch.tensor(0.0)), t, torch.nextafter(t, torch.tensor(100.0))]
    near = torch.stack(rows)
    x = torch.zeros(8, 32 * near.numel())
    for m in range(8):
        x[m, lo::32] = near
        x[m, lo + 1::32] = 6.0 * (8 + m) / 8.0                   # this block's scale is (8 + m) / 8 in nvfp4 ...
        x[m, 0 if lo else 16::32] = 2688.0                       # ... as the row's largest value makes its scale 1
    x = x.cuda()
    _same(ms.quantize(x, fmt), x, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_row_strides_and_offsets(ms, fmt, dtype):
    whole = _matrix(9, 400, dtype, 5)
    for view in (whole[:, 3:300], whole[1:8:2, 16:336], whole[:, :1], whole.t()[5:9], whole[2:3].expand(4, 400)):
        _same(ms.quantize(view, fmt), view, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", ((1, 1023), (5, 257), (3, 4097), (37, 511), (9, 130), (2, 20001), (6, 8199)))
def test_rows_at_any_address(ms, fmt, dtype, rows, k):
    """Rows of both sides that start anywhere, and what lies around them: read as it must not count, left as it was."""
    from trellis_b200 import _lib
    stream, code = torch.cuda.current_stream().cuda_stream, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    x = _matrix(rows, k, dtype, rows * 1000 + k)
    want = _same(ms.quantize(x, fmt), x, fmt).to(dtype)
    for pad, lo in ((0, 0), (1, 1), (3, 2), (16, 7), (11, 9)):
        flat = torch.full((rows * (k + pad) + 32,), float("nan"), dtype=dtype, device="cuda")
        view = flat[lo:lo + rows * (k + pad)].view(rows, k + pad)[:, :k]
        view.copy_(x)
        q = ms.quantize(view, fmt)
        assert torch.equal(q.codes, ms.quantize(x, fmt).codes) and torch.equal(ms.dequantize(q, dtype).cpu(), want)
        flat.fill_(77.0)
        assert _lib.lib().tcq_ms_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), None if fmt == "mxfp4" else q.row_scale.data_ptr(), rows, k, FMTS.index(fmt),
                                            view.data_ptr(), code, k + pad, stream) == 0
        assert torch.equal(view.cpu(), want)
        view.fill_(77.0)
        assert (flat == 77).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rotate,rows,k", ((16, 3, 48), (32, 5, 32), (32, 2, 4128), (64, 130, 192), (128, 7, 128), (128, 3, 12288)))
def test_quantize_rotated(ms, fmt, dtype, rotate, rows, k):
    """Scales and codes are those of values within the transform's rounding: log2(b) + 1 fp32 operations on sums of at most sum |x|."""
    g = torch.Generator().manual_seed(k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(dtype).cuda()
    signs = (torch.randint(0, 2, (k,), generator=g) * 2.0 - 1).cuda()
    codes, byte, row = P.unpack(ms.quantize(x, fmt, rotate=rotate, signs=signs))
    y = P.hadamard_blocks(x.cpu(), signs.cpu(), rotate)
    err = x.cpu().double().abs().reshape(rows, -1, rotate).sum(2).repeat_interleave(rotate, 1) * rotate ** -0.5 * (rotate.bit_length() + 2) * 2.0 ** -24
    lo, hi = P.quantize((y.abs() - err).clamp(min=0), fmt), P.quantize(y.abs() + err, fmt)
    if fmt == "nvfp4":
        assert ((row >= lo[2]) & (row <= hi[2])).all()
    sv = P.scale_values(byte, fmt) * (1 if row is None else row[:, None])
    slo = P.scale_values(lo[1], fmt) * (1 if row is None else lo[2][:, None])
    shi = P.scale_values(hi[1], fmt) * (1 if row is None else hi[2][:, None])
    assert ((sv >= slo) & (sv <= shi)).all()
    d = sv.repeat_interleave(P.BLOCK[fmt], 1)[:, :k]
    v = torch.tensor(P.VALUES, dtype=torch.float64)[codes & 7]
    up = torch.tensor(P.BORDERS + (float("inf"),), dtype=torch.float64)[codes & 7]
    down = torch.tensor((0.0,) + P.BORDERS, dtype=torch.float64)[codes & 7]
    assert ((y.abs() <= up * d + err) & (y.abs() >= down * d - err))[d > 0].all() and not v[d == 0].any()
    assert (((codes >= 8) == (y < 0)) | (y.abs() <= err)).all()


# ------------------------------------------------------------------------------------------------ products
SHAPES = ((1, 1, 1), (1, 16, 16), (2, 100, 31), (3, 128, 32), (5, 129, 96), (8, 300, 256), (9, 64, 257), (16, 257, 513), (17, 130, 1000),
          (33, 1, 64), (64, 128, 512), (65, 48, 300), (100, 256, 640), (129, 129, 129), (257, 300, 272), (300, 520, 768))


def _whole_number_case(rows, k, fmt, seed):
    """A matrix whose values are whole numbers of at most 12 units of 1/2."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (rows, k), generator=g)
    nb = -(-k // P.BLOCK[fmt])
    one = 127 if fmt == "mxfp4" else 0x38
    step = 1 if fmt == "mxfp4" else 8
    return codes, one + step * torch.randint(0, 2, (rows, nb), generator=g), (None if fmt == "mxfp4" else torch.ldexp(torch.ones(rows), torch.randint(-2, 3, (rows,), generator=g)))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_of_whole_numbers_is_exact(ms, fmt, dtype, m, n, k):
    w = _whole_number_case(n, k, fmt, n + k)
    x = torch.randint(-8, 9, (m, k), generator=torch.Generator().manual_seed(m)).to(dtype)
    got = ms.linear(x.cuda(), P.pack(*w, fmt, "cuda")).cpu()
    assert got.dtype == dtype and torch.equal(got, (x.double() @ P.values(*w, fmt).t()).to(dtype))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_of_whole_numbers_is_exact(ms, fmt, dtype, m, n, k):
    w, x = _whole_number_case(n, k, fmt, n + k), _whole_number_case(m, k, fmt, m)
    got = ms.matmul(P.pack(*x, fmt, "cuda"), P.pack(*w, fmt, "cuda"), dtype).cpu()
    assert got.dtype == dtype and torch.equal(got, (P.values(*x, fmt) @ P.values(*w, fmt).t()).to(dtype))


def _close(got, x, w, k, dtype):
    ref, bound = x @ w.t(), x.abs() @ w.abs().t()
    tol = (k + 16) * 2.0 ** -23 * bound + torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -10) + torch.finfo(dtype).smallest_normal
    got = got.cpu().double()
    # a real result of at least the largest number and half a step rounds to infinity; within the tolerance of that, to either
    most = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
    over = torch.isinf(got) & (torch.sign(got) == torch.sign(ref)) & (ref.abs() + tol >= most)
    off = torch.where(over, torch.zeros_like(ref), (got - ref).abs())
    assert (off <= tol).all(), f"{(off / tol).max():.3g} of the tolerance"


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", ((1, 300, 512), (4, 1024, 4096), (7, 129, 999), (20, 256, 272), (130, 200, 640), (513, 384, 1024)))
def test_linear_within_rounding(ms, fmt, dtype, m, n, k):
    w = P.random_matrix(n, k, fmt, torch.Generator().manual_seed(n * k))
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype)
    _close(ms.linear(x.cuda(), P.pack(*w, fmt, "cuda")), x.double(), P.values(*w, fmt), k, dtype)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", ((1, 300, 512), (4, 1024, 4096), (7, 129, 999), (20, 256, 272), (130, 200, 640), (513, 384, 1024)))
def test_matmul_within_rounding(ms, fmt, dtype, m, n, k):
    w, x = P.random_matrix(n, k, fmt, torch.Generator().manual_seed(n * k)), P.random_matrix(m, k, fmt, torch.Generator().manual_seed(m))
    _close(ms.matmul(P.pack(*x, fmt, "cuda"), P.pack(*w, fmt, "cuda"), dtype), P.values(*x, fmt), P.values(*w, fmt), k, dtype)


def test_linear_keeps_24_bits_of_fp32(ms):
    """One nonzero product a result: nothing but the product's own rounding is lost."""
    g = torch.Generator().manual_seed(1)
    k = 64
    codes, byte = torch.zeros(k, k, dtype=torch.int64), torch.full((k, k // 16), 0x38)
    codes[torch.arange(k), torch.arange(k)] = 3                  # 1.5 on the diagonal
    w = P.pack(codes, byte, torch.ones(k), "nvfp4", "cuda")
    for m in (1, 6, 40):
        x = torch.randn(m, k, generator=g) * torch.ldexp(torch.ones(m, k), torch.randint(-90, 90, (m, k), generator=g))
        x[0, 0], x[0, 1] = 3.4e38 / 2, -1.5e-38
        assert torch.equal(ms.linear(x.cuda(), w).cpu(), x * 1.5)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("m", (1, 3, 8, 9, 70))
def test_activations_of_any_range(ms, fmt, dtype, m):
    """Numbers over a type's whole range next to each other, one nonzero product a result: each is the product, rounded once."""
    k = 512
    g = torch.Generator().manual_seed(m)
    codes, byte = torch.zeros(k, k, dtype=torch.int64), torch.full((k, k // P.BLOCK[fmt]), 127 if fmt == "mxfp4" else 0x38)
    codes[torch.arange(k), torch.arange(k)] = 3                  # 1.5 on the diagonal
    w = P.pack(codes, byte, None if fmt == "mxfp4" else torch.ones(k), fmt, "cuda")
    lo, hi = (-24, 15) if dtype == torch.float16 else (-133, 126)
    x = (torch.rand(m, k, generator=g) * torch.ldexp(torch.ones(m, k), torch.randint(lo, hi, (m, k), generator=g))).to(dtype)
    x[0, :4] = torch.tensor([torch.finfo(dtype).tiny, -torch.finfo(dtype).tiny / 2, torch.finfo(dtype).max / 2, 0.0])
    assert torch.equal(ms.linear(x.cuda(), w).cpu(), (x.double() * 1.5).to(dtype))


@pytest.mark.parametrize("m", (9, 70, 300))
@pytest.mark.parametrize("apart", (36, 37, 100))
def test_fp16_times_scales_far_apart(ms, m, apart):
    """mxfp4 rows whose scales fp16 weights just hold, and just not; blocks of zeros with the smallest scale among them count for nothing."""
    n, k = 200, 320
    g = torch.Generator().manual_seed(apart)
    codes = torch.randint(0, 16, (n, k), generator=g)
    byte = torch.full((n, k // 32), 127)
    byte[::3, 2:4], byte[::3, 4] = 127 - apart, 127 + 3
    byte[::3, 2:4] += 3
    for column, zero in ((1, 0), (7, 8)):
        byte[:, column] = 0
        codes[:, 32 * column:32 * column + 32] = torch.where(codes[:, 32 * column:32 * column + 32] > 7, zero, 0)
    x = torch.zeros(m, k, dtype=torch.float16)
    hot = torch.randint(0, k // 32, (m,), generator=g)                # whole numbers in one block of columns a token: exact sums
    for i in range(m):
        x[i, 32 * hot[i]:32 * hot[i] + 32] = torch.randint(-8, 9, (32,), generator=g) * (2.0 ** (10 if hot[i] in (2, 3) else 0))
    want = x.double() @ P.values(codes, byte, None, "mxfp4").t()
    assert torch.equal(ms.linear(x.cuda(), P.pack(codes, byte, None, "mxfp4", "cuda")).cpu(), want.half())


@pytest.mark.parametrize("m,n", ((2000, 300), (200, 2500)))
@pytest.mark.parametrize("apart", (36, 37, 100))
def test_many_fp16_tokens_times_scales_far_apart(ms, m, n, apart):
    """The same where there are enough tiles for fp16 weights: rows that these hold, and rows that they do not, with NaN blocks and rows at any address."""
    k = 328
    g = torch.Generator().manual_seed(apart)
    codes = torch.randint(0, 16, (n, k), generator=g)
    byte = torch.full((n, 11), 127)
    byte[::3, 2:4], byte[::3, 4] = 127 - apart + 3, 127 + 3
    byte[:, 1], codes[:, 32:64] = 0, 0
    x = torch.zeros(m, k, dtype=torch.float16)
    hot = torch.randint(0, 11, (m,), generator=g)                     # whole numbers in one block of columns a token: exact sums
    for i in range(m):
        part = x[i, 32 * hot[i]:32 * hot[i] + 32]
        part.copy_(torch.randint(-8, 9, (len(part),), generator=g) * (2.0 ** (10 if hot[i] in (2, 3) else 0)))
    want = (x.double() @ P.values(codes, byte, None, "mxfp4").t()).half()
    w = P.pack(codes, byte, None, "mxfp4", "cuda")
    wide = torch.full((m, k + 3), float("nan"), dtype=torch.float16, device="cuda")
    for lo in (0, 1, 3):
        wide.fill_(float("nan"))
        wide[:, lo:lo + k] = x.cuda()
        assert torch.equal(ms.linear(wide[:, lo:lo + k], w).cpu(), want)
    held = x.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ms.linear(held, w)
    for sign in (-1, 1):
        held.copy_(x * sign)
        graph.replay()
        assert torch.equal(out.cpu(), want * sign)
    byte[5, 6] = 255
    got = ms.linear(x.cuda(), P.pack(codes, byte, None, "mxfp4", "cuda")).cpu()
    assert torch.isnan(got[:, 5]).all()
    got[:, 5], want[:, 5] = 0, 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("m,n,k", ((1300, 520, 768), (200, 2433, 257), (4800, 1, 64), (2401, 129, 31)))
def test_many_fp16_tokens_times_whole_numbers(ms, m, n, k):
    w = _whole_number_case(n, k, "mxfp4", n + k)
    x = torch.randint(-8, 9, (m, k), generator=torch.Generator().manual_seed(m)).half()
    assert torch.equal(ms.linear(x.cuda(), P.pack(*w, "mxfp4", "cuda")).cpu(), (x.double() @ P.values(*w, "mxfp4").t()).half())


@pytest.mark.parametrize("fmt", FMTS)
def test_scales_at_the_ends_of_their_range(ms, fmt):
    """The smallest and the largest scales of a format, in the weights and (products of both) in the activations."""
    k, n, m = 64, 24, 3
    g = torch.Generator().manual_seed(2)
    codes = torch.randint(0, 16, (n, k), generator=g)
    ends = torch.tensor((0, 1, 2, 30, 126, 127, 128, 180) if fmt == "mxfp4" else (0, 1, 7, 8, 0x38, 0x7D, 0x7E, 9))
    byte = ends[torch.arange(n) % 8][:, None].expand(n, k // P.BLOCK[fmt]).contiguous()
    row = None if fmt == "mxfp4" else torch.ldexp(torch.ones(n), torch.arange(n) % 40 - 20)
    wv = P.values(codes, byte, row, fmt)
    w = P.pack(codes, byte, row, fmt, "cuda")
    assert torch.equal(ms.dequantize(w).cpu().double(), wv)
    for dtype in (torch.float32, torch.bfloat16):
        for rows in (m, 150):
            x = torch.randint(-4, 5, (rows, k), generator=g).to(dtype)
            want = x.double() @ wv.t()
            assert torch.equal(ms.linear(x.cuda(), w).cpu(), want.to(dtype))
    xc, xb, xr = _whole_number_case(m, k, fmt, 9)
    want = P.values(xc, xb, xr, fmt) @ wv.t()
    assert torch.equal(ms.matmul(P.pack(xc, xb, xr, fmt, "cuda"), w, torch.float32).cpu().double(), want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", (1, 20, 140))
def test_nan_and_infinity_stay_in_their_rows(ms, fmt, m):
    n, k = 140, 320
    w = P.random_matrix(n, k, fmt, torch.Generator().manual_seed(0))
    x = torch.randint(-3, 4, (m, k), generator=torch.Generator().manual_seed(1)).double()
    wb = w[1].clone()
    wb[5, 2] = 255 if fmt == "mxfp4" else 0x7F                   # a NaN block of row 5
    wq, wv = P.pack(w[0], wb, w[2], fmt, "cuda"), P.values(w[0], wb, w[2], fmt)
    xs = x.clone()
    xs[0, 7] = float("inf")
    for dtype in (torch.float32, torch.bfloat16):
        got = ms.linear(xs.to(dtype).cuda(), wq).cpu().double()
        want = xs @ wv.t()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        assert torch.equal(torch.sign(got[torch.isinf(got)]), torch.sign(want[torch.isinf(want)]))
    xq = ms.quantize(xs.float().cuda(), fmt)
    got = ms.matmul(xq, wq, torch.float32).cpu()
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[0], bad[:, 5] = True, True
    assert torch.equal(torch.isnan(got), bad) and torch.isfinite(got[~bad]).all()


def test_linear_row_strides_and_leading_dimensions(ms):
    w = _whole_number_case(70, 96, "nvfp4", 3)
    wq, wv = P.pack(*w, "nvfp4", "cuda"), P.values(*w, "nvfp4")
    base = torch.randint(-8, 9, (40, 203), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    for m in (1, 5, 40):
        for lo in (0, 1, 8, 107):
            x = base[:m, lo:lo + 96]
            assert torch.equal(ms.linear(x.cuda() if lo == 0 else base.cuda()[:m, lo:lo + 96], wq).cpu(), (x.double() @ wv.t()).to(x.dtype))
    x = base[:24, :96].reshape(2, 3, 4, 96).cuda()
    assert torch.equal(ms.linear(x, wq).cpu(), (x.cpu().double() @ wv.t()).to(x.dtype))
    assert torch.equal(ms.linear(x[0, 0, 0], wq).cpu(), (x[0, 0, 0].cpu().double() @ wv.t()).to(x.dtype))
    assert ms.linear(x[:0], wq).shape == (0, 3, 4, 70)


def test_empty_matrices(ms):
    for fmt in FMTS:
        q = ms.quantize(torch.zeros(0, 40, device="cuda"), fmt)
        assert ms.dequantize(q).shape == (0, 40) and ms.matmul(q, q).shape == (0, 0)
        q0 = ms.quantize(torch.zeros(3, 0, device="cuda"), fmt)
        assert ms.dequantize(q0).shape == (3, 0)
        assert torch.equal(ms.matmul(q0, q0, torch.float32).cpu(), torch.zeros(3, 3))
        assert torch.equal(ms.linear(torch.zeros(2, 0, device="cuda"), q0).cpu(), torch.zeros(2, 3))


def test_results_leave_the_rest_of_their_buffer_alone(ms):
    from trellis_b200 import _lib
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for n, k in ((70, 96), (128, 256), (200, 300)):
        wc = _whole_number_case(n, k, "nvfp4", 3)
        w, wv = P.pack(*wc, "nvfp4", "cuda"), P.values(*wc, "nvfp4")
        for m in (1, 7, 40, 130):
            x = torch.randint(-4, 5, (m, k)).to(torch.bfloat16)
            xc = _whole_number_case(m, k, "nvfp4", 8)
            xq = P.pack(*xc, "nvfp4", "cuda")
            for ldy in (n + 3, n + 8):
                y = torch.full((m + 2, ldy), 77.0, dtype=torch.bfloat16, device="cuda")
                xd = x.cuda()
                ws = torch.empty(lib.tcq_ms_linear_workspace_bytes(m, n, k, 2, 1), dtype=torch.uint8, device="cuda")
                assert lib.tcq_ms_linear(xd.data_ptr(), 2, m, k, w.codes.data_ptr(), w.scales.data_ptr(), w.row_scale.data_ptr(), n, k, 1, y.data_ptr(), ldy, ws.data_ptr(), ws.numel(), stream) == 0
                assert torch.equal(y[:m, :n].cpu(), (x.double() @ wv.t()).to(torch.bfloat16))
                assert (y[m:] == 77).all() and (y[:, n:] == 77).all()
                y.fill_(77.0)
                assert lib.tcq_ms_matmul(xq.codes.data_ptr(), xq.scales.data_ptr(), xq.row_scale.data_ptr(), m, w.codes.data_ptr(), w.scales.data_ptr(),
                                         w.row_scale.data_ptr(), n, k, 1, y.data_ptr(), 2, ldy, stream) == 0
                assert torch.equal(y[:m, :n].cpu(), (P.values(*xc, "nvfp4") @ wv.t()).to(torch.bfloat16))
                assert (y[m:] == 77).all() and (y[:, n:] == 77).all()


@pytest.mark.parametrize("m", (1, 8, 50, 300))
def test_calls_repeat_on_streams_and_in_graphs(ms, m):
    """Equal bits from call to call, from two streams at once, and from a captured graph that is fed new inputs."""
    n, k = 520, 1536
    w = P.pack(*P.random_matrix(n, k, "nvfp4", torch.Generator().manual_seed(0)), "nvfp4", "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16) for _ in range(3)]
    step = lambda x: (ms.linear(x, w), ms.matmul(ms.quantize(x, "nvfp4"), w))
    want = [step(x) for x in xs]
    for x, t in zip(xs, want):
        assert all(torch.equal(a, b) for a, b in zip(step(x), t))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(step(x))
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(t, want[i % 3]))
    held = xs[0].clone()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    with torch.cuda.graph(other):
        out2 = step(held)
    for i in (1, 2, 0):
        held.copy_(xs[i])
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])) and all(torch.equal(a, b) for a, b in zip(out2, want[i]))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", ((1, 4600, 2304), (9, 2100, 2304), (30, 5000, 600), (42, 700, 4096), (60, 130, 8200), (100, 300, 4096), (128, 1000, 2111), (200, 130, 2048)))
def test_shared_columns_within_rounding(ms, fmt, dtype, m, n, k):
    """Sizes at which clusters of two, four and eight CTAs share the columns, in tiles of 8 to 128 rows of x, and two CTAs an SM."""
    w = P.random_matrix(n, k, fmt, torch.Generator().manual_seed(n * k))
    wq, wv = P.pack(*w, fmt, "cuda"), P.values(*w, fmt)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype)
    _close(ms.linear(x.cuda(), wq), x.double(), wv, k, dtype)
    if m <= 128:
        t = P.random_matrix(m, k, fmt, torch.Generator().manual_seed(m))
        _close(ms.matmul(P.pack(*t, fmt, "cuda"), wq, dtype), P.values(*t, fmt), wv, k, dtype)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype,m,n,k", ((torch.float16, 7, 300, 32000), (torch.bfloat16, 8, 130, 32700), (torch.float32, 2, 260, 32000), (torch.float32, 8, 40000, 1000)))
def test_few_tokens_beside_two_stages(ms, fmt, dtype, m, n, k):
    """All of a CTA's columns of x are held where one stage less of the weights makes room for them."""
    w = P.random_matrix(n, k, fmt, torch.Generator().manual_seed(n))
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype)
    _close(ms.linear(x.cuda(), P.pack(*w, fmt, "cuda")), x.double(), P.values(*w, fmt), k, dtype)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype,m,n,k", ((torch.bfloat16, 1, 40900, 1100), (torch.float16, 5, 77000, 600), (torch.float32, 3, 38000, 513), (torch.bfloat16, 8, 37900, 1300), (torch.float16, 2, 151936, 257)))
def test_few_tokens_through_many_rows(ms, fmt, dtype, m, n, k):
    """More groups of rows than CTAs: whole ones in turns, then the last ones shared."""
    w = _whole_number_case(n, k, fmt, n + k)
    x = torch.randint(-8, 9, (m, k), generator=torch.Generator().manual_seed(m)).to(dtype)
    wq = P.pack(*w, fmt, "cuda")
    got = ms.linear(x.cuda(), wq)
    assert torch.equal(got.cpu(), (x.double() @ P.values(*w, fmt).t()).to(dtype))
    again = [ms.linear(x.cuda(), wq) for _ in range(3)]
    assert all(torch.equal(y, got) for y in again)


def test_products_of_every_size_at_once(ms):
    """Kernels that take a whole SM, half of one and no tensor memory, in clusters of several sizes, from six streams at once."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n, k = 1300, 4096
    calls = []
    for fmt in FMTS:
        w = P.pack(*P.random_matrix(n, k, fmt, torch.Generator().manual_seed(0)), fmt, "cuda")
        for m in (1, 16, 60, 100, 300):
            x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
            xq = ms.quantize(x, fmt)
            calls += [lambda x=x, w=w: ms.linear(x, w), lambda x=xq, w=w: ms.matmul(x, w), lambda x=x.half(), w=w: ms.linear(x, w), lambda x=x[:40].float(), w=w: ms.linear(x, w)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(6)]
    got = {}
    for turn in range(6):
        for i in range(len(calls)):
            with torch.cuda.stream(streams[(i + turn) % 6]):
                got[turn, i] = calls[i]()
    torch.cuda.synchronize()
    for (turn, i), y in got.items():
        assert torch.equal(y, want[i]), (turn, i)


@pytest.mark.parametrize("m", (3, 130))
def test_rows_do_not_depend_on_each_other(ms, m):
    w = P.pack(*P.random_matrix(200, 640, "nvfp4", torch.Generator().manual_seed(0)), "nvfp4", "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, 640, generator=g, device="cuda").to(torch.bfloat16)
    other = x.clone()
    other[1:] = torch.randn(m - 1, 640, generator=g, device="cuda") * 1e4
    other[2] = float("nan")
    assert torch.equal(ms.linear(x, w)[0], ms.linear(other, w)[0])
    assert torch.equal(ms.matmul(ms.quantize(x), w)[0], ms.matmul(ms.quantize(other), w)[0])


def test_refusals_on_the_device(ms):
    w = P.pack(*P.random_matrix(20, 64, "nvfp4", torch.Generator().manual_seed(0)), "nvfp4", "cuda")
    x = torch.zeros(2, 64, device="cuda")
    for bad in (lambda: ms.linear(x[:, :48], w), lambda: ms.linear(x.cpu(), w), lambda: ms.linear(x.double(), w), lambda: ms.linear(x.clone().requires_grad_(), w),
                lambda: ms.matmul(ms.quantize(x, "mxfp4"), w), lambda: ms.matmul(ms.quantize(x[:, :48]), w), lambda: ms.matmul(ms.quantize(x), w, torch.float64),
                lambda: ms.quantize(x, rotate=16, signs=torch.ones(64)), lambda: ms.quantize(x, rotate=16, signs=torch.ones(32, device="cuda")),
                lambda: ms.dequantize(w, torch.int8), lambda: ms.dequantize(w._replace(scales=w.scales.cpu()))):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        assert ms.linear(x.clone().requires_grad_(), w).shape == (2, 20)


# ------------------------------------------------------------------------------------------------ as they are used together
@pytest.mark.parametrize("fmt", FMTS)
def test_fake_quantised_model(ms, fmt):
    from trellis_b200 import quant
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(96, 200), torch.nn.ReLU(), torch.nn.Linear(200, 33)).cuda()
    before = [m.weight.data.clone() for m in (model[0], model[2])]
    assert quant.apply_fake_quant(model, quant.MicroscaleQuantizer(fmt)) == 2
    for m, w in zip((model[0], model[2]), before):
        assert torch.equal(m.weight.data.cpu(), P.values(*P.quantize(w.cpu(), fmt), fmt).float())
    w = torch.randn(64, 256)
    w[:, 3] *= 50
    plain = quant.MicroscaleQuantizer(fmt).quantize_weight(w)
    turned = quant.MicroscaleQuantizer(fmt, rotate=128, seed=5).quantize_weight(w)
    assert plain.device.type == "cpu" and turned.shape == w.shape
    assert ((turned - w).norm() / w.norm()) < 0.2


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("activations,rotate", ((16, 0), (4, 0), (4, 32)))
def test_model_in_four_bits(ms, fmt, activations, rotate):
    """A model's layers replaced: each gives the product of its own 4-bit values, at one token and at many, eager and captured."""
    from trellis_b200 import quant
    torch.manual_seed(1)
    model = torch.nn.Sequential(torch.nn.Linear(128, 256), torch.nn.ReLU(), torch.nn.Linear(256, 96, bias=False)).cuda().to(torch.bfloat16)
    bias = model[0].bias.data.clone()
    assert quant.apply_microscaled(model, fmt, activations, rotate) == 2
    layer = model[0]
    assert set(dict(layer.named_buffers())) >= {"codes", "scales"}
    wv = P.values(*P.unpack(layer.weight), fmt)
    for lead in ((1,), (2, 5), (150,)):
        x = torch.randn(*lead, 128, device="cuda").to(torch.bfloat16)
        got = layer(x)
        flat = x.reshape(-1, 128)
        if activations == 16:
            xv = flat.cpu().double()
        else:
            xv = P.values(*P.unpack(ms.quantize(flat, fmt, rotate, layer.signs)), fmt)
        y = xv @ wv.t()
        tol = 2.0 ** -8 * (y.abs() + (y + bias.cpu().double()).abs()) + (128 + 16) * 2.0 ** -23 * (xv.abs() @ wv.abs().t()) + 1e-30
        assert ((got.reshape(-1, 256).cpu().double() - (y + bias.cpu().double())).abs() <= tol * (1 + 2.0 ** -7)).all()
    x = torch.randn(3, 128, device="cuda").to(torch.bfloat16)
    want = model(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    again = quant.apply_microscaled(torch.nn.Sequential(torch.nn.Linear(128, 8)).cuda(), fmt)
    assert again == 1


@pytest.mark.parametrize("activations,rotate", ((16, 0), (4, 64)))
def test_module_given_another_type_keeps_its_scales(ms, activations, rotate):
    from trellis_b200 import quant
    torch.manual_seed(2)
    model = torch.nn.Sequential(torch.nn.Linear(128, 40)).cuda()
    assert quant.apply_microscaled(model, "nvfp4", activations, rotate) == 1
    before = {k: v.clone() for k, v in model.state_dict().items()}
    x = torch.randn(4, 128, device="cuda").half()
    want = model(x)
    model.half()
    assert model[0].row_scale.dtype == torch.float32 and torch.equal(model(x), want)
    other = torch.nn.Sequential(quant.MicroscaledLinear(torch.zeros(40, 128), torch.zeros(40), "nvfp4", activations, rotate))
    other.load_state_dict(before)
    assert torch.equal(other(x), want)
    for name, t in other.to("cpu").state_dict().items():
        assert t.device.type == "cpu" and torch.equal(t, before[name].cpu())


def test_rotated_product_is_the_product(ms):
    """Both sides rotated: the product of the values is that of the unrotated ones, up to what 4 bits leave."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(300, 512, generator=g, device="cuda")
    x = torch.randn(40, 512, generator=g, device="cuda")
    x[:, 17] *= 100                                              # an outlier channel
    signs = torch.randint(0, 2, (512,), generator=g, device="cuda").float() * 2 - 1
    want = x.double() @ w.double().t()
    err = {}
    for r in (0, 128):
        a = dict(rotate=r, signs=signs) if r else {}
        y = ms.matmul(ms.quantize(x, **a), ms.quantize(w, **a), torch.float32).double()
        err[r] = float((y - want).norm() / want.norm())
    assert err[128] < 0.25


def test_layers_with_several_names_and_subclasses(ms):
    from trellis_b200 import quant
    torch.manual_seed(2)
    shared = torch.nn.Linear(64, 64)
    model = torch.nn.ModuleDict({"a": shared, "b": torch.nn.ModuleDict({"c": shared}), "attn": torch.nn.MultiheadAttention(64, 4), "d": torch.nn.Linear(64, 32)}).cuda()
    assert quant.apply_microscaled(model) == 2
    assert model["a"] is model["b"]["c"] and isinstance(model["a"], quant.MicroscaledLinear) and isinstance(model["d"], quant.MicroscaledLinear)
    x = torch.randn(5, 2, 64, device="cuda")
    y, _ = model["attn"](x, x, x)
    assert torch.equal(ms.linear(x, model["d"].weight) + model["d"].bias, model["d"](x)) and y.shape == x.shape


def test_a_model_is_replaced_whole_or_not_at_all(ms):
    from trellis_b200 import quant
    model = torch.nn.Sequential(torch.nn.Linear(64, 48), torch.nn.Linear(48, 8)).cuda()
    with pytest.raises(ValueError):
        quant.apply_microscaled(model, activations=4, rotate=64)
    assert all(type(m) is torch.nn.Linear for m in model)


@pytest.mark.parametrize("activations", (4, 16))
def test_module_refuses_inputs_that_need_a_gradient(ms, activations):
    from trellis_b200 import quant
    layer = quant.MicroscaledLinear(torch.randn(16, 32), activations=activations)
    x = torch.randn(3, 32, device="cuda", requires_grad=True)
    with pytest.raises(ValueError):
        layer(x)
    with torch.no_grad():
        assert layer(x).shape == (3, 16)
