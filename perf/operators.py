"""What is timed of the 4-bit microscaled operators: their plain forms and the calls that users make, over the sizes they make them at.

Each case is one call, or the few calls that belong together, of ``trellis_b200.microscale``:

    fake      ``dequantize(quantize(w))``: a weight matrix to its 4-bit values and back (``quant.apply_fake_quant`` over a model)
    linear    ``linear(x, w)``: activations in 16 or 32 bits times a 4-bit matrix (weight-only serving)
    product   ``matmul(x, w)``: both operands in 4 bits
    layer     ``matmul(quantize(x, rotated), w)``: what a linear layer with 4-bit activations does for a batch of tokens

Two formats: ``mxfp4`` (blocks of 32, power-of-two scales) and ``nvfp4`` (blocks of 16, e4m3 scales, one more scale a row).  A matrix
of ``rows x k`` values is held as

    codes      uint8 ``[rows, 16 * ceil(k / 32)]``: two e2m1 values a byte, the even column in the low half; zeros behind column k
    scales     uint8 ``[ceil(rows / 128), atoms, 32, 4, 4]``: block b of row r at ``[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]``;
               atoms = 4 (nvfp4) or 2 (mxfp4) for every 256 columns begun; zeros behind column k
    row_scale  fp32 ``[rows]`` (nvfp4), None (mxfp4)
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK = {"mxfp4": 32, "nvfp4": 16}
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # a key / value projection to nvfp4 and back, as a checkpoint's bf16 matrix
        {"name": "fake-1024x4096-nv", "kind": "fake", "n": 1024, "k": 4096, "fmt": "nvfp4", "type": "bfloat16"},
        # a gate / up projection (larger than L2) to mxfp4 and back
        {"name": "fake-12288x4096-mx", "kind": "fake", "n": 12288, "k": 4096, "fmt": "mxfp4", "type": "bfloat16"},
        # an odd fp32 matrix: rows that end inside a block
        {"name": "fake-1000x1111-nv-fp32", "kind": "fake", "n": 1000, "k": 1111, "fmt": "nvfp4", "type": "float32"},
        # token generation, one sequence: a query / output projection, where latency is all
        {"name": "linear-4096x4096-m1-nv", "kind": "linear", "n": 4096, "k": 4096, "m": 1, "fmt": "nvfp4", "type": "bfloat16"},
        # token generation, a few sequences together: the output head, where the weights' bytes are all
        {"name": "linear-151936x4096-m4-mx", "kind": "linear", "n": 151936, "k": 4096, "m": 4, "fmt": "mxfp4", "type": "bfloat16"},
        # fp32 activations, as the trellis product takes them, for a few sequences of a down projection
        {"name": "linear-4096x12288-m7-nv-fp32", "kind": "linear", "n": 4096, "k": 12288, "m": 7, "fmt": "nvfp4", "type": "float32"},
        # a ragged prompt through a gate / up projection
        {"name": "linear-12288x4096-m1000-mx-fp16", "kind": "linear", "n": 12288, "k": 4096, "m": 1000, "fmt": "mxfp4", "type": "float16"},
        # one token, both sides in 4 bits
        {"name": "product-4096x4096-m1-nv", "kind": "product", "n": 4096, "k": 4096, "m": 1, "fmt": "nvfp4", "type": "bfloat16"},
        # a ragged batch through a down projection
        {"name": "product-4096x12288-m777-mx", "kind": "product", "n": 4096, "k": 12288, "m": 777, "fmt": "mxfp4", "type": "float16"},
        # a long prompt through a gate / up projection: the tensor cores' 4-bit rate
        {"name": "product-12288x4096-m8192-nv", "kind": "product", "n": 12288, "k": 4096, "m": 8192, "fmt": "nvfp4", "type": "bfloat16"},
        # eight sequences' tokens, rotated, quantised and multiplied
        {"name": "layer-4096x4096-m8-nv", "kind": "layer", "n": 4096, "k": 4096, "m": 8, "fmt": "nvfp4", "type": "bfloat16", "rotate": 128},
        # a prompt, rotated, quantised and multiplied
        {"name": "layer-12288x4096-m2048-mx", "kind": "layer", "n": 12288, "k": 4096, "m": 2048, "fmt": "mxfp4", "type": "bfloat16", "rotate": 128},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: any number of rows and columns, from one token to a long prompt."""
    kind = rng.choice(("fake", "linear", "linear", "product", "product", "layer"))
    c = {"kind": kind, "fmt": rng.choice(("mxfp4", "nvfp4")), "type": rng.choice(("bfloat16", "bfloat16", "float16", "float32"))}
    if kind == "fake":
        c.update(n=_log_int(rng, 1, 12288), k=_log_int(rng, 16, 12288))
        return c
    if kind in ("product", "layer") and c["type"] == "float32":
        c["type"] = "bfloat16"                              # results of 4-bit operands are asked for in 16 bits
    c["n"] = _log_int(rng, 16, 12288)
    c["k"] = _log_int(rng, 16, 12288)
    # few tokens as often as many; fp32 activations come in small batches
    c["m"] = _log_int(rng, 1, 8) if rng.random() < 0.5 else _log_int(rng, 9, 128 if c["type"] == "float32" else 4096)
    if kind == "layer":
        c["rotate"] = rng.choice((0, 16, 32, 64, 128))
        if c["rotate"]:
            c["k"] = max(1, c["k"] // c["rotate"]) * c["rotate"]
    return c


# ------------------------------------------------------------------------------------------------ the format, plain
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _atoms(k, fmt):
    return (4 if fmt == "nvfp4" else 2) * -(-k // 256)


def _tile_scales(s, k, fmt):
    """``[rows, blocks]`` bytes -> the storage order, zeros in the places behind the last row and block."""
    rows, nb = s.shape
    rt, ka = -(-rows // 128), _atoms(k, fmt)
    full = torch.zeros(rt * 128, ka * 4, dtype=torch.uint8, device=s.device)
    full[:rows, :nb] = s
    return full.reshape(rt, 4, 32, ka, 4).permute(0, 3, 2, 1, 4).contiguous()


def _untile_scales(s, rows, k, fmt):
    return s.permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, -1)[:rows, :-(-k // BLOCK[fmt])]


def _round_e2m1(q):
    """Nearest e2m1 value, ties to the even code, beyond 6 to 6 (fp64)."""
    a = q.abs().clamp(max=6.0)
    step = torch.where(a >= 4, 2.0, torch.where(a >= 2, 1.0, 0.5)).to(q.dtype)
    return torch.copysign(torch.round(a / step) * step, q)


def _blocks(x, fmt):
    """``[rows, k]`` -> fp64 ``[rows, blocks, block]``, zeros behind column k."""
    b = BLOCK[fmt]
    rows, k = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -k % b))
    return x.reshape(rows, -1, b)


def _quantize_plain(x, fmt):
    """fp64 e2m1 values ``[rows, blocks, block]``, scale bytes ``[rows, blocks]``, fp32 row scales or None."""
    v = _blocks(x, fmt)
    fine = torch.isfinite(v)
    ok = fine.all(dim=2)
    amax = torch.where(fine, v, 0.0).abs().amax(dim=2)
    if fmt == "mxfp4":
        e = (torch.frexp(amax)[1] - 1 - 2).clamp(-127, 127)
        e = torch.where(amax > 0, e, -127)
        q = _round_e2m1(v * torch.exp2(-e.double())[..., None])
        byte = torch.where(ok, e + 127, 255).to(torch.uint8)
        row = None
    else:
        top = amax.amax(dim=1)
        f, j = torch.frexp(top)                              # top = f * 2^j, f in [1/2, 1)
        j = torch.where(f <= 0.65625, j - 12, j - 11).clamp(min=-80)      # the least j with top <= 2688 * 2^j
        j = torch.where(top > 0, j, 0)
        row = torch.exp2(j.double())
        s = (amax / row[:, None] / 6).float().to(torch.float8_e4m3fn)
        d = s.double()
        q = torch.where(d[..., None] > 0, v / row[:, None, None] / d[..., None], v * 0.0)
        q = _round_e2m1(q)
        byte = torch.where(ok, s.view(torch.uint8), torch.full_like(s.view(torch.uint8), 0x7F))
        row = row.float()
    return torch.where(ok[..., None], q, 0.0), byte, row


def _scale_values(byte, fmt):
    if fmt == "nvfp4":
        return byte.view(torch.float8_e4m3fn).float()
    return torch.where(byte == 255, math.nan, torch.exp2(byte.float() - 127))


def _pack(q, k):
    """e2m1 values -> packed codes ``[rows, 16 * ceil(k / 32)]``."""
    rows = q.shape[0]
    a = q.abs().float()
    code = torch.bucketize(a, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=q.device)).to(torch.uint8)
    code |= (torch.signbit(q).to(torch.uint8) << 3)
    code = code.reshape(rows, -1)
    code = torch.nn.functional.pad(code, (0, 32 * -(-k // 32) - code.shape[1]))
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _values(t, dtype=torch.float32):
    """The matrix that packed codes stand for (every value is exact in fp32)."""
    codes, scales, row, (rows, k), fmt = t
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=dtype, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), dim=2).reshape(rows, -1)[:, :k]
    s = _scale_values(_untile_scales(scales, rows, k, fmt).contiguous(), fmt).to(dtype).repeat_interleave(BLOCK[fmt], dim=1)[:, :k]
    v = lut[both.int()] * s
    return v if row is None else v * row.to(dtype)[:, None]


def _hadamard(b, dtype=torch.float64):
    h = torch.ones(1, 1, dtype=dtype, device=DEV)
    while h.shape[0] < b:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h


def _rotated(x, rotate, signs):
    """Signs, then an orthonormal Hadamard transform of every ``rotate`` columns; fp64, as borders of the rounding follow."""
    v = x.double()
    if not rotate:
        return v
    v = v * signs.double()
    h = _hadamard(rotate) / math.sqrt(rotate)
    return (v.reshape(x.shape[0], -1, rotate) @ h).reshape(x.shape)


# ------------------------------------------------------------------------------------------------ cases
def _packed(n, k, fmt, g):
    """A matrix of N(0, 0.02^2) weights in 4 bits, in the storage order."""
    codes, scales, rows = [], [], []
    step = 4096
    for r in range(0, n, step):
        w = torch.randn(min(step, n - r), k, generator=g, device=DEV) * 0.02
        q, byte, row = _quantize_plain(w, fmt)
        codes.append(_pack(q, k))
        scales.append(byte)
        rows.append(row)
    row = torch.cat(rows) if fmt == "nvfp4" else None
    return torch.cat(codes), _tile_scales(torch.cat(scales), k, fmt), row, (n, k), fmt


def _activations(m, k, dtype, g):
    """Gaussian activations whose channels differ in scale, log-uniform in [0.1, 10]."""
    scales = torch.exp(torch.empty(k, device=DEV).uniform_(math.log(0.1), math.log(10.0), generator=g))
    return (torch.randn(m, k, generator=g, device=DEV) * scales).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, k, fmt, dtype = case["n"], case["k"], case["fmt"], TYPES[case["type"]]
    s = {"case": case, "dtype": dtype}
    if case["kind"] == "fake":
        # weights N(0, 0.02^2) with 1 % outliers x 20
        w = torch.randn(n, k, generator=g, device=DEV) * 0.02
        s["x"] = torch.where(torch.rand(n, k, generator=g, device=DEV) < 0.01, w * 20, w).to(dtype)
        return s
    s["w"] = _packed(n, k, fmt, g)
    x = _activations(case["m"], k, torch.float32 if case["kind"] == "product" else dtype, g)
    if case["kind"] == "product":
        q, byte, row = _quantize_plain(x, fmt)
        s["x"] = (_pack(q, k), _tile_scales(byte, k, fmt), row, (case["m"], k), fmt)
    else:
        s["x"] = x
    if case.get("rotate"):
        s["signs"] = torch.randint(0, 2, (k,), generator=g, device=DEV).float() * 2 - 1
    return s


def _microscale():
    pkg = os.path.abspath("trellis-everywhere_b200")          # the folder users put on sys.path; the working folder is the repository's root
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from trellis_b200 import microscale
    return microscale


def run(s):
    c, x, dtype = s["case"], s["x"], s["dtype"]
    kind, fmt = c["kind"], c["fmt"]
    if own:
        ms = _microscale()
        if kind == "fake":
            return ms.dequantize(ms.quantize(x, fmt), dtype)
        w = ms.Microscaled(*s["w"])
        if kind == "linear":
            return ms.linear(x, w)
        if kind == "product":
            return ms.matmul(ms.Microscaled(*x), w, dtype)
        return ms.matmul(ms.quantize(x, fmt, rotate=c["rotate"], signs=s.get("signs")), w, dtype)
    if kind == "fake":
        return _fake(x, fmt).to(dtype)
    w = _values(s["w"])
    if kind == "linear":
        return (x.float() @ w.t()).to(dtype)
    if kind == "product":
        return (_values(x) @ w.t()).to(dtype)
    return (_fake(_rotated(x, c["rotate"], s.get("signs")), fmt) @ w.t()).to(dtype)


def _fake(x, fmt):
    """A matrix's 4-bit values (exact in fp32)."""
    rows, k = x.shape
    q, byte, row = _quantize_plain(x, fmt)
    v = q.float() * _scale_values(byte, fmt)[..., None]
    return (v if row is None else v * row[:, None, None]).reshape(rows, -1)[:, :k]


def work(case):
    n, k, fmt, t = case["n"], case["k"], case["fmt"], 4 if case["type"] == "float32" else 2
    if case["kind"] == "fake":
        return {"bytes": 2 * t * n * k, "flops": 8 * n * k}   # a maximum, a quotient, a rounding and the way back
    m = case["m"]
    held = 0.5 + 1 / BLOCK[fmt]                               # bytes a value in 4 bits with its share of a scale
    x = held * m * k if case["kind"] == "product" else t * m * k
    return {"bytes": held * n * k + x + t * m * n, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def _e2m1_by_borders(q):
    """The value whose interval holds |q|: borders half way, a border itself to the side with the even code."""
    a = q.abs()
    v = torch.zeros_like(a)
    for border, up, tie_up in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True), (2.5, 3.0, False), (3.5, 4.0, True), (5.0, 6.0, False)):
        v = torch.where((a >= border) if tie_up else (a > border), up, v)
    return torch.where(q < 0, -v, v)


def _e4m3_nearest(t):
    """Nearest e4m3 number of t >= 0 (t <= 448), ties to even."""
    e = torch.floor(torch.log2(t.clamp(min=1e-300))).clamp(min=-6)
    e = torch.where(torch.exp2(e + 1) <= t, e + 1, torch.where(torch.exp2(e) > t, e - 1, e)).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(t / step) * step


def _fake_exact(x, fmt):
    rows, k = x.shape
    b = BLOCK[fmt]
    out = torch.zeros(rows, -(-k // b) * b, dtype=torch.float64, device=x.device)
    out[:, :k] = x
    v = out.view(rows, -1, b)
    amax = v.abs().max(dim=2, keepdim=True).values
    if fmt == "mxfp4":
        e = torch.floor(torch.log2(amax.clamp(min=1e-300)))
        e = torch.where(torch.exp2(e) > amax, e - 1, torch.where(torch.exp2(e + 1) <= amax, e + 1, e))
        d = torch.exp2((e - 2).clamp(min=-127))
    else:
        top = amax.max(dim=1, keepdim=True).values
        j = torch.ceil(torch.log2((top / 2688).clamp(min=1e-300)))
        j = torch.where(top <= 2688 * torch.exp2(j - 1), j - 1, torch.where(top > 2688 * torch.exp2(j), j + 1, j)).clamp(min=-80)
        d = _e4m3_nearest(amax / torch.exp2(j) / 6) * torch.exp2(j)
    q = _e2m1_by_borders(torch.where(d > 0, v / d.clamp(min=1e-300), torch.zeros_like(v)))
    return (q * d).reshape(rows, -1)[:, :k]


def _values_exact(t):
    """fp64 values of packed codes, from the bits of the two small types."""
    codes, scales, row, (rows, k), fmt = t
    c = torch.empty(rows, 2 * codes.shape[1], dtype=torch.int32, device=codes.device)
    c[:, 0::2] = codes.int() & 15
    c[:, 1::2] = codes.int() >> 4
    e, mant = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, mant / 2, (1 + mant / 2) * torch.exp2((e - 1).double()))
    v = torch.where(c >= 8, -v, v)
    s = scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows].int()
    if fmt == "nvfp4":
        se, sm = s >> 3, (s & 7).double()
        d = torch.where(se == 0, sm / 8 * 2.0 ** -6, (1 + sm / 8) * torch.exp2((se - 7).double())) * row.double()[:, None]
    else:
        d = torch.exp2((s - 127).double())
    b = BLOCK[fmt]
    return (v[:, :k] * d[:, torch.arange(k, device=v.device) // b])


def _rotated_exact(x, rotate, signs):
    v = x.double()
    if not rotate:
        return v
    v = (v * signs.double()).reshape(x.shape[0], -1, rotate)
    h = 1
    while h < rotate:
        v = v.reshape(x.shape[0], -1, 2, h)
        v = torch.stack((v[:, :, 0] + v[:, :, 1], v[:, :, 0] - v[:, :, 1]), dim=2)
        h *= 2
    return v.reshape(x.shape) / math.sqrt(rotate)


def exact(case, seed):
    s = prepare(case, seed)
    x, kind, fmt = s["x"], case["kind"], case["fmt"]
    if kind == "fake":
        return _fake_exact(x.double(), fmt)
    if kind == "product":
        x = _values_exact(x)
    elif kind == "linear":
        x = x.double()
    else:
        x = _fake_exact(_rotated_exact(x, case["rotate"], s.get("signs")), fmt)
    codes, scales, row, (n, k), _ = s["w"]
    parts = []
    for r in range(0, n, 16384):                              # some rows of the matrix at a time (a multiple of the 128 of a scale tile)
        e = min(n, r + 16384)
        parts.append(x @ _values_exact((codes[r:e], scales[r // 128:-(-e // 128)], None if row is None else row[r:e], (e - r, k), fmt)).t())
    return torch.cat(parts, dim=1)
