"""Mixtures of experts whose matrices are in 4-bit microscaled floating point (no counterpart in the reference).

A layer of E experts sends each token to a few of them and adds up what they return, weighted.  Its matrices are most of such a model's bytes, and are
held in the formats of ``microscale``:

    route(logits, top_k)                     -> ``Routing``: each token's experts and weights, and the tokens in order of experts
    grouped_linear(x, w, offsets, tokens)    every expert's rows times that expert's matrix, with bias, activation and gate in the same kernel
    combine(y, routing, residual)            each token's results, weighted and added up

so that a whole layer is

    r = route(x @ router.T, 8)
    h = grouped_linear(x, up, r.offsets, tokens=r.tokens, activation="swiglu")
    out = combine(grouped_linear(h, down, r.offsets, dtype=torch.float32), r, residual)

How many rows an expert has stays on the GPU: nothing here synchronises or depends on it on the host, and every call can be captured into a graph.
All tensors live on one CUDA device; calls are queued on its current stream.  Nothing here has a gradient: a call that would need one is refused.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib
from .microscale import (_DTYPES, FORMATS, Microscaled, _check_act, _check_bias, _check_dtype, _check_fmt, _check_q, _check_x, _grouped, _launch, _no_gradient, _pitch, _ptr,
                         _storage)
from .qtip import _cuda_device

SCORES = {"softmax": 0, "sigmoid": 1}
MOST_EXPERTS, MOST_CHOSEN = 1024, 32


class ExpertMatrices(NamedTuple):
    """``shape`` = (E, n, k): E matrices in 4 bits, each as ``microscale.Microscaled`` holds one, one behind the other.

    ``codes``      uint8 ``[E, n, 16 * ceil(k / 32)]``
    ``scales``     uint8 ``[E, ceil(n / 128), atoms, 32, 4, 4]``
    ``row_scale``  fp32 ``[E, n]`` for nvfp4, None for mxfp4
    """
    codes: torch.Tensor
    scales: torch.Tensor
    row_scale: Optional[torch.Tensor]
    shape: Tuple[int, int, int]
    fmt: str

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        return NotImplemented


class Routing(NamedTuple):
    """Where T tokens go, ``top_k`` experts each.

    ``weights``  fp32 ``[T, top_k]``, in order of falling logits; 0 where there is no expert
    ``experts``  int32 ``[T, top_k]``, -1 where there is none
    ``places``   int32 ``[T, top_k]``: the row of each when all are in order of experts, those of one expert in order of tokens; -1 where there is none
    ``tokens``   int32 ``[T * top_k]``: the token of each of these rows; -1 behind the last
    ``offsets``  int32 ``[E + 1]``: rows ``offsets[e]`` to ``offsets[e + 1] - 1`` are expert e's
    """
    weights: torch.Tensor
    experts: torch.Tensor
    places: torch.Tensor
    tokens: torch.Tensor
    offsets: torch.Tensor


def quantize_experts(w: torch.Tensor, fmt: str = "nvfp4") -> ExpertMatrices:
    """``w [E, n, k]`` (fp32, fp16 or bf16) to 4 bits, matrix by matrix as ``microscale.quantize`` does (a gated product's rows in turn: ``microscale.interleave``)."""
    _check_fmt(fmt)
    if w.dim() != 3:
        raise ValueError(f"expected [experts, n, k], got {tuple(w.shape)}")
    _check_dtype(w.dtype)
    _no_gradient(w, "w")
    if not w.is_cuda:
        _cuda_device()
        raise ValueError("w must be on a CUDA device")
    e, n, k = w.shape
    codes_shape, scales_shape = _storage(n, k, fmt)
    codes = torch.empty((e, *codes_shape), dtype=torch.uint8, device=w.device)
    scales = torch.empty((e, *scales_shape), dtype=torch.uint8, device=w.device)
    row = torch.ones((e, n), dtype=torch.float32, device=w.device) if fmt == "nvfp4" else None
    if n and k:
        for i in range(e):
            x = _check_x(w[i], "w")
            _launch(w.device.index, "tcq_ms_quantize", x.data_ptr(), _DTYPES[x.dtype], n, k, _pitch(x), FORMATS[fmt], 0, None, codes[i].data_ptr(), scales[i].data_ptr(),
                    None if row is None else row[i].data_ptr())
    return ExpertMatrices(codes, scales, row, (e, n, k), fmt)


def stack_experts(matrices: Sequence[Microscaled]) -> ExpertMatrices:
    """E matrices of one shape and format (``microscale.quantize``, ``microscale.from_blocks``) as one; a copy."""
    if not matrices:
        raise ValueError("no matrices")
    for q in matrices:
        dev = _check_q(q, "matrix")
        if q.shape != matrices[0].shape or q.fmt != matrices[0].fmt or dev != matrices[0].codes.get_device():
            raise ValueError("matrices must have one shape, format and device")
    return ExpertMatrices(torch.stack([q.codes for q in matrices]), torch.stack([q.scales for q in matrices]),
                          None if matrices[0].row_scale is None else torch.stack([q.row_scale for q in matrices]), (len(matrices), *matrices[0].shape), matrices[0].fmt)


def expert(w: ExpertMatrices, i: int) -> Microscaled:
    """Expert i's matrix (no copy)."""
    return Microscaled(w.codes[i], w.scales[i], None if w.row_scale is None else w.row_scale[i], tuple(w.shape[1:]), w.fmt)


def _check_e(w: ExpertMatrices, name: str) -> int:
    """The CUDA device's number of well-formed matrices; raises otherwise (the kernels trust their sizes)."""
    if isinstance(w, ExpertMatrices):                        # one short pass where all is well
        codes, scales, row, (e, n, k), fmt = w
        dev = codes.get_device()
        if (dev >= 0 and codes.dtype is torch.uint8 and scales.dtype is torch.uint8 and scales.get_device() == dev and codes.shape == (e, n, 16 * -(-k // 32))
                and codes.is_contiguous() and scales.is_contiguous()
                and (row.get_device() == dev and row.dtype is torch.float32 and row.shape == (e, n) and row.is_contiguous()
                     and scales.shape == (e, -(-n // 128), 4 * -(-k // 256), 32, 4, 4) if fmt == "nvfp4" and row is not None
                     else fmt == "mxfp4" and row is None and scales.shape == (e, -(-n // 128), 2 * -(-k // 256), 32, 4, 4))):
            if row is not None:
                _no_gradient(row, f"{name}.row_scale")
            return dev
    return _refuse_e(w, name)


def _refuse_e(w, name: str) -> int:
    if not isinstance(w, ExpertMatrices):
        raise ValueError(f"{name} must be ExpertMatrices, got {type(w).__name__}")
    _check_fmt(w.fmt)
    e, n, k = w.shape
    codes, scales = _storage(n, k, w.fmt)
    dev = w.codes.device
    if w.fmt == "mxfp4" and w.row_scale is not None:
        raise ValueError(f"{name}: mxfp4 has no row scales")
    for part, t, shape, dtype in (("codes", w.codes, (e, *codes), torch.uint8), ("scales", w.scales, (e, *scales), torch.uint8), ("row_scale", w.row_scale, (e, n), torch.float32)):
        if part == "row_scale" and w.fmt == "mxfp4":
            continue
        if t is None or t.dtype is not dtype or t.shape != shape or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name}.{part} must be a contiguous {dtype} {list(shape)} tensor on {dev}")
    if w.row_scale is not None:
        _no_gradient(w.row_scale, f"{name}.row_scale")
    _cuda_device()
    raise ValueError(f"{name} must be on a CUDA device")


def _check_ints(t: torch.Tensor, name: str, shape: Tuple[int, ...], dev: int) -> None:
    if t.dtype is not torch.int32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor on cuda:{dev}")


def route(logits: torch.Tensor, top_k: int, score: str = "softmax", normalize: bool = True) -> Routing:
    """The ``top_k`` (1 to 32) experts of each token by its ``logits [T, E]`` (fp32, fp16 or bf16; E <= 1024), and all rows in order of experts.

    Chosen are the largest logits; of equal ones the expert with the lower number.  An expert whose logit is -infinity is never chosen, so a token may get fewer than
    ``top_k``, or none (a padded token with such logits alone has no rows and costs nothing).  A NaN is chosen first and makes its token's weights NaN.

    ``score``: "softmax", weights exp(logit) over their sum over all experts, or with ``normalize`` over the chosen ones; "sigmoid", weights
    1 / (1 + exp(-logit)), with ``normalize`` over their sum.  In fp32.
    """
    short = _lib.short()
    parts = short.route(logits, top_k, score, normalize) if short else None
    if parts is not None:
        return Routing(*parts)
    if score not in SCORES:
        raise ValueError(f"unknown score {score!r}; expected one of {sorted(SCORES)}")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, experts], got {tuple(logits.shape)}")
    t, e = logits.shape
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 1 <= top_k <= min(e, MOST_CHOSEN):
        raise ValueError(f"top_k={top_k!r} must be an integer from 1 to {min(e, MOST_CHOSEN)}")
    if e > MOST_EXPERTS:
        raise ValueError(f"at most {MOST_EXPERTS} experts, got {e}")
    logits = _check_x(logits, "logits")
    dev = logits.device
    weights = torch.empty_strided((t, top_k), (top_k, 1), dtype=torch.float32, device=dev)
    chosen = torch.empty_strided((t, top_k), (top_k, 1), dtype=torch.int32, device=dev)
    places = torch.empty_strided((t, top_k), (top_k, 1), dtype=torch.int32, device=dev)
    tokens = torch.empty_strided((t * top_k,), (1,), dtype=torch.int32, device=dev)
    offsets = torch.empty_strided((e + 1,), (1,), dtype=torch.int32, device=dev)
    size = _route_workspace(t, e)
    ws = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=dev) if size else None
    _launch(dev.index, "tcq_route", logits.data_ptr(), _DTYPES[logits.dtype], t, _pitch(logits), e, top_k, SCORES[score], int(normalize), weights.data_ptr(),
            chosen.data_ptr(), places.data_ptr(), tokens.data_ptr(), offsets.data_ptr(), _ptr(ws), size)
    return Routing(weights, chosen, places, tokens, offsets)


@functools.lru_cache(maxsize=4096)
def _route_workspace(t: int, e: int) -> int:
    return _lib.lib().tcq_route_workspace_bytes(t, e)


def grouped_linear(x: torch.Tensor, w: ExpertMatrices, offsets: torch.Tensor, tokens: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   activation: Optional[str] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(x[tokens[i]] @ W[e].T + bias[e])`` for every row i of every expert e, ``offsets[e] <= i < offsets[e + 1]`` -> ``[rows, n]`` of ``dtype`` (x's).

    ``x [T, k]`` in fp16 or bf16.  With ``tokens`` (int32 ``[rows]``), row i is row ``tokens[i]`` of x (one outside x gives NaN); without, row i.  ``offsets``: int32
    ``[E + 1]`` on the GPU; rows of no expert mean nothing in the result, and offsets that fall or leave 0 .. rows are taken as far as they do not.
    ``bias [E, n]``; ``activation`` as ``microscale.linear`` has it (gated ones: n / 2 columns).

    Sums, bias and activation in fp32, rounded once.  The tensor cores multiply 4-bit numbers, so few rows of x are taken as sums of them: every bit of a bf16 number down to 2^-14
    of the largest of its block of 16 (nvfp4) or 32 (mxfp4) columns (fp16: 2^-11), and 2^-22 of that off at most elsewhere (nvfp4: or 2^-39 of the
    row's largest; mxfp4: or 2^-128); many rows are multiplied as they are.  A row of x with a NaN gives NaN, one with an infinity NaN or what its sums have.  A row's result does not depend on what the others hold, and equal calls give equal results.
    """
    short = _lib.short()
    y = short.grouped_linear(x, w, offsets, tokens, bias, activation, dtype) if short and isinstance(w, ExpertMatrices) else None
    if y is not None:
        return y
    dev = _check_e(w, "w")
    e, n, k = w.shape
    act, out = _check_act(activation, n)
    if x.dim() != 2 or x.shape[1] != k or x.dtype not in (torch.float16, torch.bfloat16) or x.get_device() != dev:
        raise ValueError(f"x must be a float16 or bfloat16 [tokens, {k}] matrix on {w.codes.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    if not 1 <= e <= MOST_EXPERTS or not k:
        raise ValueError(f"1 to {MOST_EXPERTS} experts and at least one column expected, got {e} and {k}")
    x = _check_x(x, "x")
    _check_ints(offsets, "offsets", (e + 1,), dev)
    rows = x.shape[0]
    if tokens is not None:
        if tokens.dim() != 1:
            raise ValueError(f"tokens must be [rows], got {tuple(tokens.shape)}")
        rows = tokens.shape[0]
        _check_ints(tokens, "tokens", (rows,), dev)
    bias = _check_bias(bias, (e, n), w.codes.device)
    dtype = x.dtype if dtype is None else dtype
    _check_dtype(dtype)
    y = torch.empty_strided((rows, out), (out, 1), dtype=dtype, device=x.device)
    if rows and n:
        _grouped(dev, x, tokens, offsets, e, rows, w.codes, w.scales, w.row_scale, n, k, w.fmt, bias, act, None, y)
    return y


def combine(y: torch.Tensor, routing: Routing, residual: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``sum_j weights[t, j] * y[places[t, j]] + residual[t]`` -> ``[T, n]`` of ``dtype`` (the residual's, else y's): summed in fp32, rounded once.

    ``y [rows, n]`` and ``residual [T, n]`` in fp32, fp16 or bf16; a choice without an expert adds nothing.  (Of ``routing``, weights and places are read.)
    """
    short = _lib.short()
    out = short.combine(y, routing, residual, dtype) if short else None
    if out is not None:
        return out
    if not isinstance(routing, tuple) or len(routing) != 5:
        raise ValueError(f"routing must be a Routing, or its five parts as a tuple, got {type(routing).__name__}")
    if y.dim() != 2:
        raise ValueError(f"y must be [rows, n], got {tuple(y.shape)}")
    y = _check_x(y, "y")
    dev, n = y.get_device(), y.shape[1]
    weights, _, places, _, _ = routing
    if weights.dim() != 2 or not 1 <= weights.shape[1] <= MOST_CHOSEN:
        raise ValueError(f"routing.weights must be [tokens, 1 to {MOST_CHOSEN}], got {tuple(weights.shape)}")
    if weights.dtype is not torch.float32 or weights.get_device() != dev or not weights.is_contiguous():
        raise ValueError(f"routing.weights must be a contiguous float32 tensor on {y.device}")
    _no_gradient(weights, "routing.weights")
    _check_ints(places, "routing.places", tuple(weights.shape), dev)
    t, top = weights.shape
    if residual is not None:
        if residual.shape != (t, n) or residual.get_device() != dev:
            raise ValueError(f"residual must be a {[t, n]} tensor on {y.device}, got {tuple(residual.shape)} on {residual.device}")
        residual = _check_x(residual, "residual")
        if dtype is not None and dtype != residual.dtype:
            raise ValueError(f"the result has the residual's type, {residual.dtype}, not {dtype}")
        dtype = residual.dtype
    dtype = y.dtype if dtype is None else dtype
    _check_dtype(dtype)
    out = torch.empty_strided((t, n), (n, 1), dtype=dtype, device=y.device)
    if t and n:
        _launch(dev, "tcq_combine", y.data_ptr(), _DTYPES[y.dtype], y.shape[0], _pitch(y), n, weights.data_ptr(), places.data_ptr(), t, top, _ptr(residual),
                0 if residual is None else _pitch(residual), out.data_ptr(), _DTYPES[dtype], n)
    return out
