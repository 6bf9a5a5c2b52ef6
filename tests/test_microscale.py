"""4-bit microscaled formats, what needs no GPU: refusals, the storage order, argument checks of the C ABI."""
import ctypes

import pytest
import torch

import ms_plain as P
from trellis_b200 import _lib, microscale as ms, quant


def test_plain_forms_round_as_torch_does():
    """The tests' own e4m3 against torch's cast, and their e2m1 against the nearest of all values."""
    t = torch.linspace(0, 448, 20001, dtype=torch.float64)
    t = torch.cat((t, torch.ldexp(t, torch.full((t.numel(),), -12)), torch.arange(0, 449, 0.5, dtype=torch.float64)))
    byte, v = P.nearest_e4m3(t)
    want = t.float().to(torch.float8_e4m3fn)
    assert torch.equal(byte, want.view(torch.uint8).long()) and torch.equal(v, want.double())
    assert torch.equal(P.scale_values(byte, "nvfp4"), v)
    q = torch.linspace(-7, 7, 5001, dtype=torch.float64)
    code = P.nearest_e2m1(q)
    val = P.values(code[None], torch.full((1, 313), 0x38), None, "nvfp4")[0]
    grid = torch.tensor(sorted({s * x for x in P.VALUES for s in (1, -1)}), dtype=torch.float64)
    assert torch.equal((val - q).abs(), (grid[None] - q[:, None]).abs().min(1).values)


@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
@pytest.mark.parametrize("rows,k", ((1, 1), (3, 31), (130, 257), (256, 512)))
def test_storage_of_given_blocks(fmt, rows, k):
    gen = torch.Generator().manual_seed(rows + k)
    codes, byte, row = P.random_matrix(rows, k, fmt, gen)
    odd = torch.nn.functional.pad(codes, (0, k % 2), value=5)          # what a program left in the half behind an odd last column
    q = ms.from_blocks((odd[:, 0::2] | (odd[:, 1::2] << 4)).to(torch.uint8), byte.to(torch.uint8), row, k, fmt)
    got = P.unpack(q)
    assert torch.equal(got[0], codes) and torch.equal(got[1], byte)
    assert (row is None) == (got[2] is None) and (row is None or torch.equal(got[2], row.double()))
    assert torch.equal(ms.block_scales(q).long(), byte)
    assert q.codes.numel() == rows * _lib.lib().tcq_ms_code_pitch(k)
    assert q.scales.numel() == _lib.lib().tcq_ms_scale_bytes(rows, k, ms.FORMATS[fmt])


def test_given_blocks_are_checked():
    c, s = torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    assert ms.from_blocks(c, s, 0.5, 32, "nvfp4").row_scale.tolist() == [0.5, 0.5]
    for bad in ((c, s, None, 32, "nvfp4"), (c, s, 1.0, 32, "mxfp4"), (c, s, 1.0, 33, "nvfp4"), (c.int(), s, 1.0, 32, "nvfp4"),
                (c, s[:1], 1.0, 32, "nvfp4"), (c, s, 1.0, 32, "fp4")):
        with pytest.raises(ValueError):
            ms.from_blocks(*bad)


def test_refusals_before_touching_the_device():
    x = torch.zeros(2, 32)
    for bad in (dict(fmt="int4"), dict(rotate=8, signs=torch.ones(32)), dict(rotate=64, signs=torch.ones(32)), dict(rotate=16),
                dict(signs=torch.ones(32))):
        with pytest.raises(ValueError):
            ms.quantize(x, **bad)
    with pytest.raises(ValueError):
        ms.quantize(torch.zeros(2, 2, 32))
    with pytest.raises(ValueError):
        ms.quantize(x.double())
    with pytest.raises(ValueError, match="gradient"):
        ms.quantize(x.requires_grad_())
    with pytest.raises(ValueError):
        ms.linear(x, x)
    with pytest.raises(ValueError):
        quant.MicroscaleQuantizer("int4")
    with pytest.raises(ValueError):
        quant.MicroscaleQuantizer("nvfp4", rotate=48)
    with pytest.raises(ValueError):
        quant.MicroscaledLinear(torch.zeros(2, 32), rotate=16)
    assert quant.MicroscaleQuantizer("nvfp4").bpw == 4.5 and quant.MicroscaleQuantizer("mxfp4").bpw == 4.25
    q = P.pack(*P.random_matrix(3, 40, "nvfp4", torch.Generator().manual_seed(0)), "nvfp4")
    for bad in (q._replace(codes=q.codes[:, :16]), q._replace(scales=q.scales[:, :2]), q._replace(row_scale=None),
                q._replace(shape=(4, 40)), q._replace(shape=(3, 300)), q._replace(fmt="mxfp4"), q._replace(codes=q.codes.int()),
                q._replace(row_scale=q.row_scale.double()), q._replace(codes=q.codes.t().contiguous().t())):
        with pytest.raises(ValueError):
            ms.dequantize(bad)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the behaviour on a box without a GPU")
def test_no_cpu_fallback():
    q = P.pack(*P.random_matrix(3, 40, "nvfp4", torch.Generator().manual_seed(0)), "nvfp4")
    for call in (lambda: ms.quantize(torch.zeros(2, 32)), lambda: ms.dequantize(q), lambda: ms.linear(torch.zeros(1, 40), q), lambda: ms.matmul(q, q)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_argument_validation_needs_no_gpu():
    L = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    p += (-p) % 256
    Q, D, N, M = L.tcq_ms_quantize, L.tcq_ms_dequantize, L.tcq_ms_linear, L.tcq_ms_matmul
    assert L.tcq_strerror(-12) and L.tcq_ms_code_pitch(33) == 32 and L.tcq_ms_scale_bytes(129, 1, 1) == 4096
    assert L.tcq_ms_scale_bytes(1, 1, 2) == 0 and L.tcq_ms_scale_bytes(-1, 1, 0) == 0 and L.tcq_ms_code_pitch(-1) == 0
    assert Q(p, 0, 1, 16, 16, 2, 0, None, p, p, p, None) == -12         # format
    assert Q(p, 3, 1, 16, 16, 1, 0, None, p, p, p, None) == -12         # type
    assert Q(p, 0, -1, 16, 16, 1, 0, None, p, p, p, None) == -3
    assert Q(p, 0, 1, 16, 15, 1, 0, None, p, p, p, None) == -8          # row stride
    assert Q(p, 0, 1, 48, 48, 1, 32, p, p, p, p, None) == -8            # rotation does not divide k
    assert Q(p, 0, 1, 48, 48, 1, 48, p, p, p, p, None) == -8
    assert Q(p, 0, 1, 48, 48, 1, 16, None, p, p, p, None) == -4         # signs missing
    assert Q(p, 0, 1, 16, 16, 1, 0, None, p, p, None, None) == -4       # row scales missing
    assert Q(p, 0, 1, 16, 16, 0, 0, None, p, p, p, None) == -4          # row scales where there are none
    assert Q(p, 0, 1, 16, 16, 1, 0, None, p + 8, p, p, None) == -5
    assert Q(p + 2, 0, 1, 16, 16, 1, 0, None, p, p, p, None) == -5
    assert Q(p, 0, 0, 16, 16, 1, 0, None, None, None, None, None) == 0  # nothing to do
    assert D(p, p, p, 1, 16, 1, p, 0, 15, None) == -8 and D(p, p, p, 1, 16, 1, None, 0, 16, None) == -4
    assert D(p, p, p, 1, (1 << 24) + 1, 1, p, 0, 1 << 31, None) == -8 and D(p, p, p, 1 << 31, 16, 1, p, 0, 16, None) == -8
    ws = (p, 4096, None)
    assert N(p, 2, 1, 16, p, p, p, 4, 16, 1, p, 3, *ws) == -8           # ldy < n
    assert N(p, 2, 1, 15, p, p, p, 4, 16, 1, p, 4, *ws) == -8           # ldx < k
    assert N(p, 2, 1, 16, p, p, p, 4, 0, 1, p, 4, *ws) == -8            # no columns
    assert N(None, 2, 1, 16, p, p, p, 4, 16, 1, p, 4, *ws) == -4 and N(p, 0, 9, 16, p, p, p, 4, 16, 1, p, 4, None, 0, None) == -4
    assert N(p + 1, 2, 1, 16, p, p, p, 4, 16, 1, p, 4, *ws) == -5 and N(p, 2, 1, 16, p, p, p, 4, 16, 1, p, 4, p + 128, 4096, None) == -5
    assert N(p, 0, 9, 16, p, p, p, 4, 16, 1, p, 4, p, L.tcq_ms_linear_workspace_bytes(9, 4, 16, 0, 1) - 1, None) == -6
    assert L.tcq_ms_linear_workspace_bytes(1, 1, 16, 3, 1) == 0 and L.tcq_ms_linear_workspace_bytes(-1, 1, 16, 0, 1) == 0 and L.tcq_ms_linear_workspace_bytes(1, 1, 16, 0, 2) == 0
    assert N(p, 2, 0, 16, None, None, None, 4, 16, 1, None, 4, None, 0, None) == 0
    assert M(p, p, p, 1, p, p, None, 4, 16, 1, p, 2, 4, None) == -4
    assert M(p, p, p, 1, p, p + 4, p, 4, 16, 1, p, 2, 4, None) == -5
    assert M(p, p, p, -1, p, p, p, 4, 16, 1, p, 2, 4, None) == -3


def test_selftests_of_waits_check_their_arguments():
    L = _lib.lib()
    buf = (ctypes.c_char * 1024)()
    p = ctypes.addressof(buf)
    p += (-p) % 256
    linear, matmul = (p, 2, 1, 16, p, p, p, 4, 16, 1, p, 4, p, 512, None), (p, p, p, 1, p, p, p, 4, 16, 1, p, 2, 4, None)
    for loads in (-1, 2 ** 32 - 1, 2 ** 40):
        assert L.tcq_selftest_ms_linear_waits(loads, *linear) == -3 and L.tcq_selftest_ms_matmul_waits(loads, *matmul) == -3
    assert L.tcq_selftest_ms_linear_waits(0, None, *linear[1:]) == -4 and L.tcq_selftest_ms_matmul_waits(0, None, *matmul[1:]) == -4
    assert L.tcq_selftest_ms_linear_waits(0, p, 2, 0, *linear[3:]) == 0


def test_every_input_that_needs_a_gradient_is_refused():
    """Backward and forward ones, of the input, the signs and the row scales; none where gradients are off."""
    from torch.autograd import forward_ad
    x = torch.zeros(2, 32)
    q = P.pack(*P.random_matrix(3, 32, "nvfp4", torch.Generator().manual_seed(0)), "nvfp4")
    grown = q._replace(row_scale=q.row_scale.clone().requires_grad_())
    for call in (lambda: ms.quantize(x, rotate=16, signs=torch.ones(32, requires_grad=True)), lambda: ms.linear(x, grown), lambda: ms.matmul(q, grown),
                 lambda: ms.dequantize(grown)):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(Exception) as refused:
            call()
        assert "gradient" not in str(refused.value)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(2, 32))
        row = q._replace(row_scale=forward_ad.make_dual(q.row_scale, torch.ones(3)))
        signs = forward_ad.make_dual(torch.ones(32), torch.ones(32))
        for call in (lambda: ms.quantize(dual), lambda: ms.quantize(x, rotate=16, signs=signs), lambda: ms.dequantize(row), lambda: ms.linear(x, row)):
            with pytest.raises(ValueError, match="gradient"):
                call()
        with pytest.raises(Exception) as refused:
            ms.quantize(x)
        assert "gradient" not in str(refused.value)


@pytest.mark.parametrize("rows,k", ((1, 1), (3, 31), (130, 257), (7, 80)))
def test_scales_with_a_sign_go_to_the_codes(rows, k):
    gen = torch.Generator().manual_seed(rows * k)
    codes, byte, row = P.random_matrix(rows, k, "nvfp4", gen)
    sign = torch.randint(0, 2, byte.shape, generator=gen)
    odd = torch.nn.functional.pad(codes, (0, k % 2), value=5)
    packed = (odd[:, 0::2] | (odd[:, 1::2] << 4)).to(torch.uint8)
    want = P.values(codes, byte, row, "nvfp4") * (1 - 2 * sign).repeat_interleave(16, 1)[:, :k]
    for scales in ((byte + 128 * sign).to(torch.uint8), (byte + 128 * sign).to(torch.uint8).view(torch.float8_e4m3fn)):
        q = ms.from_blocks(packed, scales, row, k, "nvfp4")
        got = P.unpack(q)                                        # (checks that nothing stands behind column k)
        assert torch.equal(got[1], byte) and torch.equal(P.values(*got, "nvfp4"), want)
    nan = ms.from_blocks(packed, torch.full_like(byte, 0xFF, dtype=torch.uint8), row, k, "nvfp4")
    assert (ms.block_scales(nan) == 0x7F).all()


def test_scales_of_another_type_are_refused():
    c = torch.zeros(2, 16, dtype=torch.uint8)
    for fmt, row, nb, own, other in (("nvfp4", 1.0, 2, torch.float8_e4m3fn, torch.float8_e8m0fnu), ("mxfp4", None, 1, torch.float8_e8m0fnu, torch.float8_e4m3fn)):
        s = torch.zeros(2, nb, dtype=torch.uint8)
        for good in (s, s.view(torch.int8), s.view(own)):
            assert not ms.block_scales(ms.from_blocks(c, good, row, 32, fmt)).any()
        for bad in (s.view(other), s.view(torch.float8_e5m2), s.bool()):
            with pytest.raises(ValueError, match="scales"):
                ms.from_blocks(c, bad, row, 32, fmt)


@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
def test_blocks_of_matrices_without_rows_or_columns(fmt):
    for rows, k in ((0, 40), (3, 0), (0, 0)):
        nb = -(-k // ms.BLOCKS[fmt])
        q = ms.from_blocks(torch.zeros(rows, -(-k // 2), dtype=torch.uint8), torch.zeros(rows, nb, dtype=torch.uint8), None if fmt == "mxfp4" else 1.0, k, fmt)
        assert ms.block_scales(q).shape == (rows, nb)
