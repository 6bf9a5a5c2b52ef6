"""Products and values at the ends of the types' ranges, where each factor is far from 1 and their product is not.

Weights are e2m1 x block scale x row scale, and any of the three may be large where another is small.  A result is finite where the sum of the
products' magnitudes is, whatever the parts of a product are by themselves.

Tolerances.  One product a result (six bits of a weight, up to 24 of x; row scales powers of two): fp32 parts are added with roundings of at most 2^-8 of
half a step, then the result's rounding, half a step; results below the smallest normal number are rounded to the type's smallest steps, once in fp32 and once in
the type, half a step each; for more than eight fp32 tokens sums are made of quarters, whose smallest step is four of the result's, and cut off, not rounded, by
the tensor cores: three parts, with weights 1, 2^-8 and 2^-16, are off by less than 4 (1 + 2^-7) steps, and with the result's rounding by less than five.  Dense sums: (k + 16) 2^-23 of the sum of magnitudes, as anywhere, and the result's rounding.
"""
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


def _near(got, ref, tol, dtype):
    got = got.cpu().double()
    most = torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4)
    over = torch.isinf(got) & (torch.sign(got) == torch.sign(ref)) & (ref.abs() + tol >= most)
    off = torch.where(over, torch.zeros_like(ref), (got - ref).abs())
    assert (off <= tol).all(), f"{int((~(off <= tol)).sum())} of {off.numel()} off, {(off / tol).nan_to_num(1e30).max():.3g} of the tolerance"


def _rounding(ref, dtype, tokens=1):
    f = torch.finfo(dtype)
    steps = 5 if dtype == torch.float32 and tokens > 8 else 1
    return f.eps / 2 * ref.abs() * (1 + 2.0 ** -7) + steps * f.smallest_normal * f.eps


def _diagonal(k, fmt, seed, byte_span, row_span):
    """A matrix with one value a row, on the diagonal: any code, block scales and row scales over the given powers of two."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.zeros(k, k, dtype=torch.int64)
    codes[torch.arange(k), torch.arange(k)] = torch.randint(1, 8, (k,), generator=g) + 8 * torch.randint(0, 2, (k,), generator=g)
    nb = k // P.BLOCK[fmt]
    if fmt == "mxfp4":
        return codes, 127 + torch.randint(byte_span[0], byte_span[1] + 1, (k, nb), generator=g), None
    return codes, torch.randint(1, 0x7F, (k, nb), generator=g), torch.ldexp(torch.ones(k), torch.randint(row_span[0], row_span[1] + 1, (k,), generator=g))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", (1, 8))
@pytest.mark.parametrize("spans", (((-30, 0), (-17, -17)), ((-110, -80), (-110, -60)), ((0, 30), (1, 12)), ((70, 100), (60, 117))))
def test_few_tokens_of_any_size_times_weights_of_any_size(ms, fmt, dtype, m, spans):
    _products(ms, fmt, dtype, m, spans)


def _products(ms, fmt, dtype, m, spans):
    k = 512
    w = _diagonal(k, fmt, m, *spans)
    v = P.values(*w, fmt).diagonal()
    g = torch.Generator().manual_seed(m + 1)
    lo, hi = {torch.float16: (-24, 15), torch.bfloat16: (-133, 127), torch.float32: (-149, 127)}[dtype]
    x = ((1 + torch.rand(m, k, generator=g, dtype=torch.float64)) * torch.ldexp(torch.ones(m, k, dtype=torch.float64), torch.randint(lo, hi, (m, k), generator=g))).to(dtype)
    x[:, ::7] = torch.finfo(dtype).max
    x[:, 3::7] = -torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    ref = x.double() * v
    _near(ms.linear(x.cuda(), P.pack(*w, fmt, "cuda")), ref, _rounding(ref, dtype, m), dtype)


def _dense(ms, fmt, m, n, k, dtype, x_exp, w_exp, seed):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(n, k, generator=g) * 2.0 ** w_exp).cuda()
    x = (torch.randn(m, k, generator=g).double() * 2.0 ** x_exp).to(dtype).cuda()
    q = ms.quantize(w, fmt)
    return x, q, P.values(*P.unpack(q), fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("x_exp,w_exp", ((120, -6), (125, -40), (124, -60), (-120, 100), (-60, 60)))
@pytest.mark.parametrize("m,n,k", ((2, 140, 1024), (8, 300, 4096), (1, 40000, 300)))
def test_few_tokens_sums_far_from_one(ms, fmt, dtype, x_exp, w_exp, m, n, k):
    _sums(ms, fmt, dtype, x_exp, w_exp, m, n, k)


def _sums(ms, fmt, dtype, x_exp, w_exp, m, n, k):
    x, q, wv = _dense(ms, fmt, m, n, k, dtype, x_exp, w_exp, m + n)
    xv = x.cpu().double()
    ref, bound = xv @ wv.t(), xv.abs() @ wv.abs().t()
    _near(ms.linear(x, q), ref, (k + 16) * 2.0 ** -23 * bound + _rounding(ref, dtype, m), dtype)


def test_few_tokens_row_scales_of_any_number(ms):
    """Row scales that are not powers of two, and the smallest and the largest numbers."""
    k = 256
    codes, byte, _ = _diagonal(k, "nvfp4", 5, None, (0, 0))
    row = torch.rand(k, generator=torch.Generator().manual_seed(6)) + 0.5
    row[::5] *= 2.0 ** -120
    row[1::5] = 1e-45
    row[2::5] = 3e38
    v = P.values(codes, byte, row, "nvfp4").diagonal()
    w = P.pack(codes, byte, row, "nvfp4", "cuda")
    for dtype in (torch.float32, torch.bfloat16):
        for m in (1, 5):
            x = torch.randn(m, k, generator=torch.Generator().manual_seed(m))
            x[:, 2::5] *= 2.0 ** -20
            x[:, 1::5] *= 2.0 ** 120
            x = x.to(dtype)
            ref = x.double() * v
            # the row scale's 24 bits: one more rounding in fp32
            _near(ms.linear(x.cuda(), w), ref, _rounding(ref, dtype) + 2.0 ** -23 * ref.abs(), dtype)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", (9, 70, 300))
@pytest.mark.parametrize("spans", (((-30, 0), (-17, -17)), ((-110, -80), (-110, -60)), ((0, 30), (1, 12)), ((70, 100), (60, 117))))
def test_many_tokens_of_any_size_times_weights_of_any_size(ms, fmt, dtype, m, spans):
    _products(ms, fmt, dtype, m, spans)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("x_exp,w_exp", ((120, -6), (125, -40), (124, -60), (-120, 100), (-60, 60)))
@pytest.mark.parametrize("m,n,k", ((9, 140, 1024), (70, 300, 4096), (150, 200, 300)))
def test_many_tokens_sums_far_from_one(ms, fmt, dtype, x_exp, w_exp, m, n, k):
    _sums(ms, fmt, dtype, x_exp, w_exp, m, n, k)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", (1, 9, 100))
def test_fp32_results_just_below_the_largest_number(ms, fmt, m):
    """The parts of an fp32 number times a weight: none leaves the range where the product does not."""
    k = 256
    codes, byte = torch.zeros(k, k, dtype=torch.int64), torch.full((k, k // P.BLOCK[fmt]), 127 if fmt == "mxfp4" else 0x38)
    codes[torch.arange(k), torch.arange(k)] = 7                  # 6 on the diagonal
    w = P.pack(codes, byte, None if fmt == "mxfp4" else torch.ones(k), fmt, "cuda")
    g = torch.Generator().manual_seed(m)
    x = torch.finfo(torch.float32).max / 6 * (1 - torch.rand(m, k, generator=g) * 0.4)
    assert torch.equal(ms.linear(x.cuda(), w).cpu(), (x.double() * 6).float())


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("m,n,k", ((1, 40, 64), (20, 300, 2304), (100, 200, 512), (150, 140, 272), (300, 520, 768)))
@pytest.mark.parametrize("x_exp,w_exp", ((122, -20), (-20, 122), (124, -70), (-60, 123), (-75, 90), (110, -110)))
def test_matmul_of_sides_far_apart(ms, dtype, m, n, k, x_exp, w_exp):
    """One side's row scales huge, the other's tiny: the sum of both sides' codes times one of them leaves the range, the result does not."""
    g = torch.Generator().manual_seed(m)
    x, w = (ms.quantize((torch.randn(r, k, generator=g) * 2.0 ** e).cuda(), "nvfp4") for r, e in ((m, x_exp), (n, w_exp)))
    xv, wv = P.values(*P.unpack(x), "nvfp4"), P.values(*P.unpack(w), "nvfp4")
    ref = xv @ wv.t()
    # (both scales, powers of two, are exact)
    _near(ms.matmul(x, w, dtype), ref, (k + 16) * 2.0 ** -23 * (xv.abs() @ wv.abs().t()) + _rounding(ref, dtype), dtype)


def test_matmul_of_row_scales_of_any_number(ms):
    g = torch.Generator().manual_seed(1)
    for m in (3, 70, 150):
        k, n = 320, 64
        x, w = ([*P.random_matrix(r, k, "nvfp4", g)] for r in (m, n))
        for q, rows in ((x, m), (w, n)):
            q[2] = (torch.rand(rows, generator=g) + 0.5) * torch.ldexp(torch.ones(rows), torch.randint(-63, 64, (rows,), generator=g))
            q[2][::7] = 1e-44
        ref, bound = P.values(*x, "nvfp4") @ P.values(*w, "nvfp4").t(), P.values(*x, "nvfp4").abs() @ P.values(*w, "nvfp4").abs().t()
        got = ms.matmul(P.pack(*x, "nvfp4", "cuda"), P.pack(*w, "nvfp4", "cuda"), torch.float32)
        # three roundings by scales of 24 bits
        _near(got, ref, (k + 16) * 2.0 ** -23 * bound + 3 * 2.0 ** -24 * ref.abs() + _rounding(ref, torch.float32), torch.float32)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("rotate,k", ((16, 48), (32, 96), (64, 192), (128, 256), (128, 33024)))
def test_rotation_of_the_largest_numbers(ms, fmt, dtype, rotate, k):
    """Sums of `rotate` numbers leave the range where the orthonormal transform does not: the codes are those of the same numbers 2^-20 times as large."""
    g = torch.Generator().manual_seed(rotate)
    top = torch.finfo(dtype).max / rotate ** 0.5
    x = (torch.randint(-2, 3, (5, k), generator=g) / 2.0 * top).to(dtype).cuda()
    signs = (torch.randint(0, 2, (k,), generator=g) * 2.0 - 1).cuda()
    a, b = ms.quantize(x, fmt, rotate, signs), ms.quantize(x * 2.0 ** -20, fmt, rotate, signs)
    ca, sa, ra = P.unpack(a)
    cb, sb, rb = P.unpack(b)
    assert torch.equal(ca, cb) and torch.equal(sa, sb if fmt == "nvfp4" else torch.where(sb > 0, sb + 20, sb))
    assert ra is None or torch.equal(ra, rb * 2.0 ** 20)
    assert not torch.isnan(ms.dequantize(b)).any() and not ((sa == (255 if fmt == "mxfp4" else 0x7F)).any())


def test_values_with_row_scales_of_any_number(ms):
    """Code times block scale is exact in fp32, so a row scale rounds once, and a zero stays one however large the scales are."""
    g = torch.Generator().manual_seed(3)
    rows, k = 96, 321
    codes, byte, _ = P.random_matrix(rows, k, "nvfp4", g, spread=6)
    byte[:, 3], byte[:, 4] = 0x7E, 1
    codes[::2, 50:60] = torch.randint(0, 2, (rows // 2, 10), generator=g) * 8
    row = (torch.rand(rows, generator=g) + 0.5) * torch.ldexp(torch.ones(rows), torch.randint(-126, 127, (rows,), generator=g))
    row[:3] = torch.tensor((3.4e38, 1e-45, 2.9e-39))
    v = P.values(codes, byte, row, "nvfp4")                      # (exact in fp64)
    w = P.pack(codes, byte, row, "nvfp4", "cuda")
    for dtype in DTYPES:
        assert torch.equal(ms.dequantize(w, dtype).cpu(), v.float().to(dtype)), dtype
