"""4-bit microscaled floating point: quantisation, its inverse, and products (no counterpart in the reference).

The trellis codes next door (``qtip``) store a matrix in 2 to 4 bits a weight and multiply by it one token at a time.
These formats take 4.25 or 4.5 bits a weight and are what the tensor cores multiply directly, so they also serve
prompts and activations:

    quantize(x, fmt)        a matrix -> ``Microscaled`` (codes, block scales, row scales); optionally rotated first
    dequantize(q, dtype)    its values
    linear(x, w)            ``x @ W.T``, x in 16 or 32 bits (weight-only)
    matmul(x, w)            ``X @ W.T``, both in 4 bits

Every value is ``e2m1(code) * block scale``, e2m1 one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign:

    "mxfp4"   blocks of 32 columns, scale 2^(floor(log2 amax) - 2)
    "nvfp4"   blocks of 16 columns, scale e4m3(amax / (6 g)), times a row scale g: the least power of two, from
              2^-80 on, with the row's largest magnitude <= 2688 g (2688 = 6 * 448)

A row scale instead of one for the whole matrix keeps the codes of a token independent of the others in its batch.
Codes are the nearest of the exact quotients, ties to the even code, magnitudes beyond 6 to 6.  A block that holds a
NaN or an infinity becomes all NaN (its scale is), and nothing else changes by it.

All tensors live on one CUDA device; calls are queued on its current stream, nothing synchronises, and every call can
be captured into a graph.  Nothing here has a gradient: a call that would need one, of the input, the signs or the row scales, backward or
forward, is refused.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .qtip import _cuda_device

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCKS = {"mxfp4": 32, "nvfp4": 16}
ROTATIONS = (0, 16, 32, 64, 128)
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Microscaled(NamedTuple):
    """A ``shape`` = (rows, k) matrix in 4 bits, as the kernels read it.

    ``codes``      uint8 ``[rows, 16 * ceil(k / 32)]``: two codes a byte, the even column in the low half; zeros behind column k
    ``scales``     uint8 ``[ceil(rows / 128), atoms, 32, 4, 4]``: block b of row r at ``[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]``;
                   atoms = 2 (mxfp4) or 4 (nvfp4) for every 256 columns begun; zeros behind column k.  The places of rows
                   behind the last one mean nothing (``block_scales`` leaves them out)
    ``row_scale``  fp32 ``[rows]`` for nvfp4, None for mxfp4

    A checkpoint's own codes and scales can be put in this form too (``from_blocks``); any positive row scales go with them.
    """
    codes: torch.Tensor
    scales: torch.Tensor
    row_scale: Optional[torch.Tensor]
    shape: Tuple[int, int]
    fmt: str

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        """torch's functions do not take such a matrix: owners of a layer that look (``nn.TransformerEncoderLayer`` in evaluation) then call the
        layer instead of handing its weight to a function, and those that do not look get a TypeError."""
        return NotImplemented


def _storage(rows: int, k: int, fmt: str):
    """Shapes of codes and scales."""
    return (rows, 16 * -(-k // 32)), (-(-rows // 128), (4 if fmt == "nvfp4" else 2) * -(-k // 256), 32, 4, 4)


def _check_fmt(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f"unknown microscaled format {fmt!r}; expected one of {sorted(FORMATS)}")
    return FORMATS[fmt]


def _check_dtype(dtype) -> int:
    if dtype not in _DTYPES:
        raise ValueError(f"float32, float16 or bfloat16 expected, not {dtype}")
    return _DTYPES[dtype]


def _no_gradient(t: torch.Tensor, name: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"no gradient is defined here: detach {name} or call under torch.no_grad()")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"no gradient is defined here, forward ones neither: {name} has a tangent")


def _check_q(q: Microscaled, name: str) -> int:
    """The CUDA device's number of a well-formed matrix; raises otherwise (the kernels trust its sizes).

    The products of token generation last a few microseconds, so what leads up to them is kept short: one pass over the parts
    where all is well, and the search for what is wrong elsewhere (and results by ``torch.empty_strided``, which is a microsecond
    faster than ``torch.empty``).
    """
    if isinstance(q, Microscaled):
        codes, scales, row, (rows, k), fmt = q
        dev = codes.get_device()
        if (dev >= 0 and codes.dtype is torch.uint8 and scales.dtype is torch.uint8 and scales.get_device() == dev
                and codes.shape == (rows, 16 * -(-k // 32)) and codes.is_contiguous() and scales.is_contiguous()
                and (row.get_device() == dev and row.dtype is torch.float32 and row.shape == (rows,) and row.is_contiguous()
                     and scales.shape == (-(-rows // 128), 4 * -(-k // 256), 32, 4, 4) if fmt == "nvfp4" and row is not None
                     else fmt == "mxfp4" and row is None and scales.shape == (-(-rows // 128), 2 * -(-k // 256), 32, 4, 4))):
            if row is not None and (row.requires_grad or forward_ad._current_level >= 0):
                _no_gradient(row, f"{name}.row_scale")
            return dev
    return _refuse_q(q, name)


def _refuse_q(q, name: str) -> int:
    if not isinstance(q, Microscaled):
        raise ValueError(f"{name} must be a Microscaled matrix, got {type(q).__name__}")
    _check_fmt(q.fmt)
    rows, k = q.shape
    codes, scales = _storage(rows, k, q.fmt)
    dev = q.codes.device
    for part, t, shape, dtype in (("codes", q.codes, codes, torch.uint8), ("scales", q.scales, scales, torch.uint8),
                                  ("row_scale", q.row_scale, (rows,), torch.float32)):
        if part == "row_scale" and q.fmt == "mxfp4":
            if t is not None:
                raise ValueError(f"{name}: mxfp4 has no row scales")
            continue
        if t is None or t.dtype != dtype or tuple(t.shape) != shape or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name}.{part} must be a contiguous {dtype} {list(shape)} tensor on {dev}")
    if q.row_scale is not None:
        _no_gradient(q.row_scale, f"{name}.row_scale")
    _cuda_device()
    raise ValueError(f"{name} must be on a CUDA device")


def _check_x(x: torch.Tensor, name: str) -> torch.Tensor:
    """A matrix with unit column stride and rows that do not overlap, of a type the kernels take, on a CUDA device."""
    if x.dtype not in _DTYPES:
        _check_dtype(x.dtype)
    if x.requires_grad or forward_ad._current_level >= 0:
        _no_gradient(x, name)
    if not x.is_cuda:
        _cuda_device()
        raise ValueError(f"{name} must be on a CUDA device")
    if x.is_contiguous():
        return x
    rows, k = x.shape
    if (x.stride(1) != 1 and k > 1) or (x.stride(0) < k and rows > 1):
        return x.detach().contiguous()
    return x


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _launch(dev: int, name: str, *args) -> None:
    """``qtip._call`` for a device number, by the shortest way to the current device and stream."""
    fn = getattr(_lib.lib(), name)
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, name)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def quantize(x: torch.Tensor, fmt: str = "nvfp4", rotate: int = 0, signs: Optional[torch.Tensor] = None) -> Microscaled:
    """``x [rows, k]`` (fp32, fp16 or bf16; any row stride) to 4 bits.

    ``rotate`` = 16, 32, 64 or 128 (dividing k) first multiplies the columns by ``signs [k]`` (fp32) and transforms every
    ``rotate`` of them by the orthonormal Hadamard matrix, in fp32 within the same kernel: incoherence processing of the input
    axis (``qtip.block_hadamard``).  A product of two matrices rotated alike is the product of the matrices, and outliers
    no longer set the scales.
    """
    _check_fmt(fmt)
    if x.dim() != 2:
        raise ValueError(f"expected a matrix, got {tuple(x.shape)}")
    if rotate not in ROTATIONS or (rotate and x.shape[1] % rotate):
        raise ValueError(f"rotate={rotate} must be one of {ROTATIONS} and divide the {x.shape[1]} columns")
    if (signs is not None) != bool(rotate):
        raise ValueError("signs go with rotate: give both or neither")
    if signs is not None:
        _no_gradient(signs, "signs")
    x = _check_x(x, "x")
    if signs is not None and (signs.dtype != torch.float32 or tuple(signs.shape) != (x.shape[1],) or signs.device != x.device
                              or not signs.is_contiguous()):
        raise ValueError(f"signs must be a contiguous float32 [{x.shape[1]}] tensor on {x.device}")
    rows, k = x.shape
    dev = x.device
    codes_shape, scales_shape = _storage(rows, k, fmt)
    codes = torch.empty_strided(codes_shape, (codes_shape[1], 1), dtype=torch.uint8, device=dev)
    scales = torch.empty_strided(scales_shape, (512 * scales_shape[1], 512, 16, 4, 1), dtype=torch.uint8, device=dev)
    row = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=dev) if fmt == "nvfp4" else None
    if rows and k:
        _launch(dev.index, "tcq_ms_quantize", x.data_ptr(), _DTYPES[x.dtype], rows, k, _pitch(x), FORMATS[fmt], rotate, _ptr(signs),
                codes.data_ptr(), scales.data_ptr(), _ptr(row))
    elif row is not None:
        row.fill_(1.0)                                       # rows without columns
    return Microscaled(codes, scales, row, (rows, k), fmt)


def dequantize(q: Microscaled, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The ``[rows, k]`` values.  Of a matrix quantised here they are exact in fp32, and in bf16 as well; fp16 rounds those out of its range."""
    dev, dt = _check_q(q, "q"), _check_dtype(dtype)
    rows, k = q.shape
    out = torch.empty_strided((rows, k), (k, 1), dtype=dtype, device=q.codes.device)
    if rows and k:
        _launch(dev, "tcq_ms_dequantize", q.codes.data_ptr(), q.scales.data_ptr(), _ptr(q.row_scale), rows, k, FORMATS[q.fmt],
                out.data_ptr(), dt, k)
    return out


def linear(x: torch.Tensor, w: Microscaled) -> torch.Tensor:
    """``x @ W.T``: ``x [..., k]`` (fp32, fp16 or bf16) times a 4-bit ``[n, k]`` matrix -> ``[..., n]`` of x's type.

    Products with the weights' exact values, summed in fp32, rounded once (16-bit results of more than eight rows are summed
    by the tensor cores, which cut fp32 sums off instead of rounding them).  Finite wherever the sum of the products' magnitudes
    is, whatever the size of x and of the weights (mxfp4 block scales up to 2^104).  A row of the result does not depend
    on what the other rows of x hold, and equal calls give equal results.
    """
    dev = _check_q(w, "w")
    codes, scales, row, (n, k), fmt = w
    shape = x.shape
    if not shape or shape[-1] != k:
        raise ValueError(f"x must be [..., {k}], got {tuple(shape)}")
    if x.get_device() != dev:
        raise ValueError(f"x must be on {codes.device}")
    flat = _check_x(x if len(shape) == 2 else x.reshape(math.prod(shape[:-1]), k), "x")
    m = flat.shape[0]
    y = torch.empty_strided((m, n), (n, 1), dtype=flat.dtype, device=flat.device)
    if m and n and k:
        dt, pitch, at = _DTYPES[flat.dtype], _pitch(flat), flat.data_ptr()
        ws = size = None
        if m > 8 and (at % 16 or pitch % 8 or not (dt == 2 or (dt == 1 and fmt == "nvfp4"))):
            size = _lib.lib().tcq_ms_linear_workspace_bytes(m, n, k, dt, FORMATS[fmt])
            ws = torch.empty(size, dtype=torch.uint8, device=flat.device)  # given back when the call is queued: the stream's later work comes after it
        _launch(dev, "tcq_ms_linear", at, dt, m, pitch, codes.data_ptr(), scales.data_ptr(), _ptr(row), n, k, FORMATS[fmt], y.data_ptr(), n,
                _ptr(ws), size or 0)
    elif not k:
        y.zero_()
    return y if len(shape) == 2 else y.view(*shape[:-1], n)


def matmul(x: Microscaled, w: Microscaled, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``X @ W.T`` of two 4-bit matrices ``[m, k]`` and ``[n, k]`` of one format -> ``[m, n]`` of ``dtype``, rounded once.

    The sum is the tensor cores': in fp32 over all of k, cut off where fp32 arithmetic rounds (exact for Gaussian matrices of up to
    12288 columns, whose products have few bits; otherwise up to 2^-23 of the sum of magnitudes a term).
    """
    dev, dt = _check_q(w, "w"), _check_dtype(dtype)
    codes, scales, row, (n, k), fmt = w
    if _check_q(x, "x") != dev or x.fmt != fmt or x.shape[1] != k:
        raise ValueError(f"x and w must have one format, device and number of columns: {x.fmt} {x.shape} on {x.codes.device}, "
                         f"{fmt} {w.shape} on {codes.device}")
    m = x.shape[0]
    y = torch.empty_strided((m, n), (n, 1), dtype=dtype, device=codes.device)
    if m and n and k:
        _launch(dev, "tcq_ms_matmul", x.codes.data_ptr(), x.scales.data_ptr(), _ptr(x.row_scale), m, codes.data_ptr(), scales.data_ptr(), _ptr(row),
                n, k, FORMATS[fmt], y.data_ptr(), dt, n)
    elif not k:
        y.zero_()
    return y


def block_scales(q: Microscaled) -> torch.Tensor:
    """The scale bytes by row and block, uint8 ``[rows, ceil(k / block)]`` (e4m3 for nvfp4, exponents + 127 for mxfp4)."""
    rows, k = q.shape
    s = q.scales.permute(0, 3, 2, 1, 4).reshape(q.scales.shape[0] * 128, q.scales.shape[1] * 4)
    return s[:rows, :-(-k // BLOCKS[q.fmt])].contiguous()


def from_blocks(codes: torch.Tensor, scales: torch.Tensor, row_scale: Optional[torch.Tensor], k: int, fmt: str) -> Microscaled:
    """A matrix from row-major codes ``[rows, >= ceil(k / 2)]`` and scale bytes ``[rows, ceil(k / block)]``, as other programs store them.

    ``row_scale``: fp32 ``[rows]`` or one number for all rows (nvfp4), None (mxfp4).  Done once per matrix, with torch.  Scales are bytes or
    of their own type (float8_e4m3fn, float8_e8m0fnu); the tensor cores take them without a sign, so that of an e4m3 scale goes to its codes.
    """
    _check_fmt(fmt)
    if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[1] < -(-k // 2) or k < 0:
        raise ValueError(f"expected uint8 codes [rows, >= {-(-k // 2)}], got {codes.dtype} {tuple(codes.shape)}")
    rows, nb = codes.shape[0], -(-k // BLOCKS[fmt])
    own = torch.float8_e4m3fn if fmt == "nvfp4" else torch.float8_e8m0fnu
    if tuple(scales.shape) != (rows, nb) or scales.dtype not in (torch.uint8, torch.int8, own):
        raise ValueError(f"expected scales [{rows}, {nb}] of bytes or {own}, got {scales.dtype} {tuple(scales.shape)}")
    if (row_scale is None) != (fmt == "mxfp4"):
        raise ValueError("row scales go with nvfp4, and only with it")
    codes_shape, scales_shape = _storage(rows, k, fmt)
    dev = codes.device
    c = torch.zeros(codes_shape, dtype=torch.uint8, device=dev)
    c[:, :-(-k // 2)] = codes[:, :-(-k // 2)]
    scales = scales.to(dev).view(torch.uint8)
    if fmt == "nvfp4":
        c[:, :-(-k // 2)] ^= ((scales >> 7) * 0x88).repeat_interleave(8, 1)[:, :-(-k // 2)]
        scales = scales & 0x7F
    if k % 2:
        c[:, k // 2] &= 15                                   # the half behind the last column
    full = torch.zeros((scales_shape[0] * 128, scales_shape[1] * 4), dtype=torch.uint8, device=dev)
    full[:rows, :nb] = scales
    tiled = full.reshape(scales_shape[0], 4, 32, scales_shape[1], 4).permute(0, 3, 2, 1, 4).contiguous()
    row = None
    if row_scale is not None:
        row = torch.as_tensor(row_scale, dtype=torch.float32, device=dev).expand(rows).contiguous()
    return Microscaled(c, tiled, row, (rows, k), fmt)
