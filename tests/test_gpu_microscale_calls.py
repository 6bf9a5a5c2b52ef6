"""Calls of the microscaled operators that go beyond plain matrices: gradients that are asked for, and other programs' matrices."""
import pytest
import torch
from torch.autograd import forward_ad

import ms_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ms():
    from trellis_b200 import microscale
    return microscale


def test_inputs_that_need_a_gradient_on_the_device(ms):
    w = P.pack(*P.random_matrix(20, 64, "nvfp4", torch.Generator().manual_seed(0)), "nvfp4", "cuda")
    x = torch.randn(3, 64, device="cuda")
    q, grown = ms.quantize(x), w._replace(row_scale=w.row_scale.clone().requires_grad_())
    signs = torch.ones(64, device="cuda", requires_grad=True)
    calls = (lambda: ms.quantize(x, rotate=16, signs=signs), lambda: ms.linear(x, grown), lambda: ms.matmul(q, grown), lambda: ms.matmul(grown, q), lambda: ms.dequantize(grown))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        for call in calls:
            call()
        assert torch.equal(ms.linear(x, grown), ms.linear(x, w))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        row = w._replace(row_scale=forward_ad.make_dual(w.row_scale, torch.ones_like(w.row_scale)))
        for call in (lambda: ms.quantize(dual), lambda: ms.linear(dual, w), lambda: ms.linear(x, row), lambda: ms.dequantize(row), lambda: ms.matmul(q, row)):
            with pytest.raises(ValueError, match="gradient"):
                call()
        assert torch.equal(ms.linear(x, w), ms.linear(x.clone(), w))


def test_a_subclass_is_a_matrix_too(ms):
    class Named(ms.Microscaled):
        pass

    for fmt in ("mxfp4", "nvfp4"):
        w = P.pack(*P.random_matrix(20, 64, fmt, torch.Generator().manual_seed(0)), fmt, "cuda")
        x = torch.randn(3, 64, device="cuda")
        q, named = ms.quantize(x, fmt), Named(*w)
        assert torch.equal(ms.linear(x, named), ms.linear(x, w)) and torch.equal(ms.matmul(q, named), ms.matmul(q, w)) and torch.equal(ms.dequantize(named), ms.dequantize(w))
        with pytest.raises(ValueError, match="codes"):
            ms.dequantize(named._replace(codes=w.codes[:, :16]))


@pytest.mark.parametrize("m", (1, 20, 150))
def test_products_of_scales_with_a_sign(ms, m):
    """Scales of another program's matrix that carry a sign: all products take it alike."""
    gen = torch.Generator().manual_seed(m)
    n, k = 70, 96
    codes = torch.randint(0, 16, (n, k), generator=gen)
    byte, sign = torch.full((n, k // 16), 0x38), torch.randint(0, 2, (n, k // 16), generator=gen)
    w = ms.from_blocks((codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8).cuda(), (byte + 128 * sign).to(torch.uint8).cuda(), 0.5, k, "nvfp4")
    wv = P.values(codes, byte, torch.full((n,), 0.5), "nvfp4") * (1 - 2 * sign).repeat_interleave(16, 1)
    x = torch.randint(-4, 5, (m, k), generator=gen).float()      # whole numbers: exact sums, and exact 4-bit values
    q = ms.quantize(x.cuda(), "nvfp4")
    assert torch.equal(ms.dequantize(w).cpu().double(), wv)
    assert torch.equal(ms.linear(x.cuda(), w).cpu().double(), x.double() @ wv.t())
    assert torch.equal(ms.matmul(q, w, torch.float32).cpu().double(), ms.dequantize(q).cpu().double() @ wv.t())


@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
def test_outliers_do_not_set_the_scales_of_a_rotated_matrix(ms, fmt):
    """One channel of 100 among values of at most 1.  Unrotated it is its block's largest value, 100; rotated by 128 no value is above (100 + 127) / 128^(1/2) = 20.1,
    so that the largest scale falls from 2^4 to 2^2 at most (mxfp4), or from at least 100 / 6 (1 - 2^-4) to at most 20.1 / 6 (1 + 2^-4) (nvfp4)."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.rand(200, 512, generator=g, device="cuda") * 2 - 1
    x[:, 17] = 100.0
    signs = torch.randint(0, 2, (512,), generator=g, device="cuda").float() * 2 - 1
    top = []
    for q in (ms.quantize(x, fmt), ms.quantize(x, fmt, 128, signs)):
        s = P.scale_values(ms.block_scales(q).long().cpu(), fmt)
        top.append((s if q.row_scale is None else s * q.row_scale.cpu().double()[:, None]).amax(1))
    assert (top[1] <= top[0] / 4).all()
