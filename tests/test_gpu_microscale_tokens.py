"""Few tokens of unlike ranges in one call of ``linear``: a token that takes more parts than another changes nothing for that one."""
import pytest
import torch

from ms_cases import whole_matrix

pytestmark = pytest.mark.gpu


def _tokens(m, k, dtype, seed):
    """m tokens of ordinary numbers, and the same with far smaller ones among those of the odd tokens: 2^-40 in bf16, the smallest numbers in fp16."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    wide = x.clone()
    small = 2.0 ** -40 if dtype == torch.bfloat16 else 2.0 ** -24
    wide[1::2, 5::37] = small
    wide[1::2, 11] = 3e4
    if m > 2:
        wide[2, k // 2:] *= small                                 # ... and of one token in the later columns only
    return x.to(dtype), wide.to(dtype)


@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("m,n,k", ((2, 200, 256), (3, 130, 1111), (8, 300, 4096), (5, 40000, 520), (8, 38000, 4600), (2, 100, 12288)))
def test_tokens_that_take_more_parts_leave_the_others_alone(fmt, dtype, m, n, k):
    from trellis_b200 import microscale as ms
    w, wv = whole_matrix(n, k, fmt, n + k)
    plain, wide = _tokens(m, k, dtype, m)
    a, b = ms.linear(plain, w), ms.linear(wide, w)
    same = (plain == wide).all(1)
    assert same.any() and not same.all() and torch.equal(a[same], b[same])
    # the sum's rounding (fp32, any order) and the result's, half a step
    for x, y in ((plain, a), (wide, b)):
        ref, bound = x.double() @ wv.t(), x.double().abs() @ wv.abs().t()
        tol = (k + 16) * 2.0 ** -23 * bound + torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -10) + torch.finfo(dtype).smallest_normal
        off = (y.double() - ref).abs()
        fits = ref.abs() < torch.finfo(dtype).max / 2
        assert (off <= tol)[fits].all(), f"{(off / tol)[fits].max():.3g} of the tolerance"


@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("span", (3, 30, 60, 200))
@pytest.mark.parametrize("m", (1, 8))
def test_tokens_whose_largest_number_is_anywhere(fmt, dtype, span, m):
    """256 columns of a token at a time with every exponent as their largest, the others up to `span` below: one product a result, which is exact but for its rounding."""
    from trellis_b200 import microscale as ms
    k, b = 2048, ms.BLOCKS[fmt]
    codes = torch.zeros(k, k, dtype=torch.uint8, device="cuda")
    codes[torch.arange(k), torch.arange(k)] = 3                  # 1.5 on the diagonal
    w = ms.from_blocks(codes[:, 0::2] | (codes[:, 1::2] << 4), torch.full((k, k // b), 127 if fmt == "mxfp4" else 0x38, dtype=torch.uint8, device="cuda"),
                       None if fmt == "mxfp4" else 1.0, k, fmt)
    g = torch.Generator(device="cuda").manual_seed(span + m)
    lo, hi = {torch.float32: (-149, 126), torch.float16: (-24, 14), torch.bfloat16: (-133, 126)}[dtype]
    tops = torch.arange(lo, hi + 1, device="cuda")
    for at in range(0, len(tops), 8 * m):
        top = tops[(at + torch.arange(8 * m, device="cuda")) % len(tops)].reshape(m, 8).repeat_interleave(256, 1)
        down = torch.randint(0, span + 1, (m, k), generator=g, device="cuda")
        down[:, 7::256] = 0
        e = (top - down).clamp(min=lo)
        x = ((1 + torch.rand(m, k, generator=g, device="cuda", dtype=torch.float64)) * torch.exp2(e.double())).to(dtype)
        y, want = ms.linear(x, w), (x.double() * 1.5).to(dtype)
        if dtype == torch.float32:
            # 25 bits of a product below 2^-123 reach beyond the smallest step, 2^-149: each of the three parts is rounded there by half a step, and added exactly
            tiny = want.abs() < 2.0 ** -123
            assert ((y.double() - x.double() * 1.5).abs()[tiny] <= 2 * 2.0 ** -149).all(), (at, tops[at])
            y = torch.where(tiny, want, y)
        assert torch.equal(y, want), (at, tops[at])
