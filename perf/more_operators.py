"""What is timed of a mixture of experts in 4 bits and of products with an epilogue: their plain forms and the calls that users make.

Each case is one call, or the run of calls that belong together, of ``trellis_b200.microscale`` and ``trellis_b200.experts``:

    linear    ``microscale.linear(x, w, bias, activation, residual)``: a product whose epilogue is part of it
    route     ``experts.route(logits, top_k)``: each token's experts, their weights, and the tokens in order of experts
    experts   ``experts.grouped_linear(x, w, offsets, tokens, bias, activation)``: every expert's rows times that expert's matrix
    combine   ``experts.combine(y, routing, residual)``: a token's results, weighted and added up
    layer     route, the first product with its gate, the second, combine: a whole mixture of experts

A matrix of ``rows x k`` values is held as ``microscale.Microscaled`` describes; E of them as ``experts.ExpertMatrices`` does, the same with
one more axis in front:

    codes      uint8 ``[E, rows, 16 * ceil(k / 32)]``: two e2m1 values a byte, the even column in the low half; zeros behind column k
    scales     uint8 ``[E, ceil(rows / 128), atoms, 32, 4, 4]``: block b of row r at ``[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]``;
               atoms = 4 (nvfp4) or 2 (mxfp4) for every 256 columns begun; zeros behind column k
    row_scale  fp32 ``[E, rows]`` (nvfp4), None (mxfp4)

"swiglu" and "geglu" take rows in pairs: the even one is the gate, the odd one what it multiplies, and half as many results come out.
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
GATED = ("swiglu", "geglu")


def listed():
    return [
        # token generation, one sequence: an attention's output projection, added to the residual stream
        {"name": "linear-4096x4096-m1-nv", "kind": "linear", "n": 4096, "k": 4096, "m": 1, "fmt": "nvfp4", "type": "bfloat16", "bias": False, "act": "", "res": True},
        # token generation, a batch of sequences: gate and up projection of 12288 as one matrix, with the gate in the epilogue
        {"name": "linear-24576x4096-m12-mx", "kind": "linear", "n": 24576, "k": 4096, "m": 12, "fmt": "mxfp4", "type": "bfloat16", "bias": False, "act": "swiglu", "res": False},
        # a ragged prompt through a layer with a bias and GELU
        {"name": "linear-12288x4096-m2000-nv-fp16", "kind": "linear", "n": 12288, "k": 4096, "m": 2000, "fmt": "nvfp4", "type": "float16", "bias": True, "act": "gelu_tanh", "res": False},
        # fp32 activations of a small, odd layer, with everything that an epilogue does
        {"name": "linear-1000x1111-m37-mx-fp32", "kind": "linear", "n": 1000, "k": 1111, "m": 37, "fmt": "mxfp4", "type": "float32", "bias": True, "act": "relu", "res": True},
        # token generation, one sequence: eight experts of 128
        {"name": "route-t1-e128-k8", "kind": "route", "t": 1, "e": 128, "top": 8, "type": "bfloat16", "score": "softmax", "norm": True},
        # a prompt: two experts of 61, each weighted by itself
        {"name": "route-t5000-e61-k2-fp32", "kind": "route", "t": 5000, "e": 61, "top": 2, "type": "float32", "score": "sigmoid", "norm": False},
        # token generation, one sequence: the gated first product of eight experts of 64, where latency is all
        {"name": "experts-t1-e64-k8-nv", "kind": "experts", "t": 1, "e": 64, "top": 8, "n": 2048, "k": 2048, "fmt": "nvfp4", "type": "bfloat16", "bias": False, "act": "swiglu", "gather": True},
        # token generation, 48 sequences: the second product, where the bytes of all experts' weights are all
        {"name": "experts-t48-e64-k8-mx", "kind": "experts", "t": 48, "e": 64, "top": 8, "n": 4096, "k": 1024, "fmt": "mxfp4", "type": "bfloat16", "bias": True, "act": "", "gather": False},
        # a ragged prompt: the gated first product, where products are all
        {"name": "experts-t2040-e64-k8-nv", "kind": "experts", "t": 2040, "e": 64, "top": 8, "n": 2816, "k": 2048, "fmt": "nvfp4", "type": "bfloat16", "bias": False, "act": "swiglu", "gather": True},
        # one sequence's eight results
        {"name": "combine-t1-k8", "kind": "combine", "t": 1, "e": 64, "top": 8, "n": 2048, "type": "bfloat16", "res": True},
        # a prompt's results, of an odd width
        {"name": "combine-t4000-k4-odd", "kind": "combine", "t": 4000, "e": 16, "top": 4, "n": 2035, "type": "float16", "res": False},
        # a batch of 200 tokens through a whole mixture of experts of an odd inner width
        {"name": "layer-t200-e32-k4-mx-fp16", "kind": "layer", "t": 200, "e": 32, "top": 4, "n": 1000, "k": 2048, "fmt": "mxfp4", "type": "float16", "act": "swiglu"},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: from one token to a prompt, any number of experts, rows and columns."""
    kind = rng.choice(("linear", "linear", "route", "experts", "experts", "experts", "combine", "layer"))
    c = {"kind": kind, "type": rng.choice(("bfloat16", "bfloat16", "float16"))}
    if kind == "linear":
        act = rng.choice(("", "relu", "gelu", "gelu_tanh", "silu", "swiglu", "geglu"))
        # few tokens as often as many; fp32 activations come in small batches
        if rng.random() < 0.2:
            c["type"] = "float32"
        m = _log_int(rng, 1, 16) if rng.random() < 0.5 else _log_int(rng, 17, 64 if c["type"] == "float32" else 2048)
        n = _log_int(rng, 16, 8192)
        c.update(n=n + n % 2, k=_log_int(rng, 16, 4096), m=m, fmt=rng.choice(("mxfp4", "nvfp4")), bias=rng.random() < 0.5, act=act, res=rng.random() < 0.5)
        return c
    e = _log_int(rng, 2, 128)
    c.update(e=e, top=min(e, rng.randint(1, 8)), t=_log_int(rng, 1, 16) if rng.random() < 0.5 else _log_int(rng, 17, 1024 if kind in ("experts", "layer") else 4096))
    if kind == "route":
        if rng.random() < 0.3:
            c["type"] = "float32"
        c.update(score=rng.choice(("softmax", "sigmoid")), norm=rng.random() < 0.5)
        return c
    c["n"] = 2 * _log_int(rng, 8, 1024)
    if kind == "combine":
        c["n"] += rng.randint(0, 1)
        c["res"] = rng.random() < 0.5
        return c
    c.update(k=_log_int(rng, 16, 2048), fmt=rng.choice(("mxfp4", "nvfp4")), act=rng.choice(("", "relu", "gelu", "gelu_tanh", "silu", "swiglu", "geglu")))
    if kind == "experts":
        c.update(bias=rng.random() < 0.5, gather=rng.random() < 0.5)
    else:
        c.update(act=rng.choice(GATED), n=max(16, c["n"] // 2))
    return c


# ------------------------------------------------------------------------------------------------ the format, plain
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantize_plain(w, fmt):
    """A matrix ``[rows, k]`` as packed codes, tiled scales, row scales."""
    rows, k = w.shape
    b = BLOCK[fmt]
    v = torch.nn.functional.pad(w.double(), (0, -k % 256)).reshape(rows, -1, b)
    amax = v.abs().amax(dim=2)
    if fmt == "mxfp4":
        e = (torch.frexp(amax)[1] - 3).clamp(-127, 127)
        byte, d, row = e + 127, torch.exp2(e.double()), None
        byte = torch.where(amax > 0, byte, 0)
    else:
        top = amax.amax(dim=1).clamp(min=1e-20)
        j = torch.ceil(torch.log2(top / 2688))
        s = (amax / torch.exp2(j)[:, None] / 6).float().clamp(max=448.0).to(torch.float8_e4m3fn)
        byte, d, row = s.view(torch.uint8), s.double() * torch.exp2(j)[:, None], torch.exp2(j).float()
    a = (v / torch.where(d > 0, d, 1.0)[..., None]).clamp(-6, 6).float()
    code = torch.bucketize(a.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)).to(torch.uint8)
    code = (code | (torch.signbit(a).to(torch.uint8) << 3)).reshape(rows, -1)
    code[:, k:] = 0
    code = code[:, :32 * -(-k // 32)]
    full = torch.zeros(-(-rows // 128) * 128, byte.shape[1], dtype=torch.uint8, device=w.device)
    full[:rows, :-(-k // b)] = byte[:, :-(-k // b)].to(torch.uint8)
    tiled = full.reshape(-1, 4, 32, byte.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return code[:, 0::2] | (code[:, 1::2] << 4), tiled, row


def _values(codes, scales, row, n, k, fmt):
    """fp32 ``[..., n, k]`` that packed codes stand for (every value is exact), of one matrix or of E."""
    lut = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    v = lut[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)[..., :k].int()]
    s = scales.movedim(-2, -4).movedim(-2, -3)                # [..., tiles, 4, 32, atoms, 4]
    s = s.reshape(*s.shape[:-5], s.shape[-5] * 128, -1)[..., :n, :-(-k // BLOCK[fmt])].contiguous()
    s = s.view(torch.float8_e4m3fn).float() if fmt == "nvfp4" else torch.exp2(s.float() - 127)
    v = v * s.repeat_interleave(BLOCK[fmt], dim=-1)[..., :k]
    return v if row is None else v * row[..., None]


def _epilogue(h, bias, act, residual):
    """Bias, activation and residual in fp32."""
    if bias is not None:
        h = h + bias.float()
    if act in GATED:
        h, up = h[..., 0::2], h[..., 1::2]
    if act == "relu":
        h = torch.where(h < 0, 0.0, h)
    elif act in ("gelu", "geglu"):
        h = 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
    elif act == "gelu_tanh":
        h = 0.5 * h * (1 + torch.tanh(math.sqrt(2 / math.pi) * (h + 0.044715 * h * h * h)))
    elif act in ("silu", "swiglu"):
        h = h / (1 + torch.exp(-h))
    if act in GATED:
        h = h * up
    return h if residual is None else h + residual.float()


def _route(logits, top, score, norm):
    """(weights, experts, places, tokens, offsets) of a batch, in fp32; ties go to the expert with the lower number."""
    t, e = logits.shape
    v = logits.float()
    best, chosen = torch.sort(v, dim=1, descending=True, stable=True)
    best, chosen = best[:, :top], chosen[:, :top]
    if score == "softmax":
        p = torch.exp(best - best[:, :1])
        w = p / (p.sum(1, keepdim=True) if norm else torch.exp(v - best[:, :1]).sum(1, keepdim=True))
    else:
        w = 1 / (1 + torch.exp(-best))
        w = w / w.sum(1, keepdim=True) if norm else w
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True)[1]
    places = torch.empty_like(order)
    places[order] = torch.arange(t * top, device=flat.device)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = (flat[:, None] == torch.arange(e, device=flat.device)).sum(0).cumsum(0)
    return w, chosen.int(), places.reshape(t, top).int(), (order // top).int(), offsets


def _grouped(x, w, offsets, room, bias, act):
    """Rows in order of experts times their expert's matrix: each expert's rows in a padded place of their own, one product of them all."""
    e = offsets.shape[0] - 1
    i = torch.arange(x.shape[0], device=x.device)
    of = torch.searchsorted(offsets[1:].contiguous().long(), i, right=True)
    at = i - offsets.long()[of]
    padded = torch.zeros(e, room, x.shape[1], device=x.device)
    padded[of, at] = x.float()
    h = (padded @ w.transpose(1, 2))[of, at]
    return _epilogue(h if bias is None else h + bias.float()[of], None, act, None)


def _combine(y, weights, places, residual):
    out = (y.float()[places.long()] * weights[..., None]).sum(1)
    return out if residual is None else out + residual.float()


# ------------------------------------------------------------------------------------------------ cases
def _weights(n, k, fmt, g, count=0, scale=0.02):
    """A matrix of N(0, scale^2) weights in 4 bits, or ``count`` of them with one more axis in front."""
    parts = [_quantize_plain(torch.randn(n, k, generator=g, device=DEV) * scale, fmt) for _ in range(count or 1)]
    return tuple(None if p[0] is None else torch.stack(p) if count else p[0] for p in zip(*parts))


def _activations(m, k, dtype, g):
    """Gaussian activations whose channels differ in scale, log-uniform in [0.1, 10]."""
    scales = torch.exp(torch.empty(k, device=DEV).uniform_(math.log(0.1), math.log(10.0), generator=g))
    return (torch.randn(m, k, generator=g, device=DEV) * scales).to(dtype)


def _logits(t, e, dtype, g):
    """Gaussian logits; some experts are asked more often than others."""
    return (torch.randn(t, e, generator=g, device=DEV) * 1.5 + torch.randn(e, generator=g, device=DEV) * 0.5).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["type"]]
    s = {"case": case, "dtype": dtype, "bias": None, "res": None}
    if kind == "linear":
        n, k, m = case["n"], case["k"], case["m"]
        s["w"] = _weights(n, k, case["fmt"], g)
        s["x"] = _activations(m, k, dtype, g)
        if case["bias"]:
            s["bias"] = torch.randn(n, generator=g, device=DEV).to(dtype)
        if case["res"]:
            s["res"] = (torch.randn(m, n // 2 if case["act"] in GATED else n, generator=g, device=DEV) * 3).to(dtype)
        return s
    t, e, top = case["t"], case["e"], case["top"]
    s["logits"] = _logits(t, e, dtype, g)
    if kind == "route":
        return s
    s["routing"] = _route(s["logits"], top, "softmax", True)
    s["room"] = int(s["routing"][4].diff().max())            # rows of the expert with most of them
    n = case["n"]
    if kind == "combine":
        s["y"] = torch.randn(t * top, n, generator=g, device=DEV).to(dtype)
        if case["res"]:
            s["res"] = (torch.randn(t, n, generator=g, device=DEV) * 3).to(dtype)
        return s
    k = case["k"]
    if kind == "experts":
        s["w"] = _weights(n, k, case["fmt"], g, e)
        s["x"] = _activations(t if case["gather"] else t * top, k, dtype, g)
        if case["bias"]:
            s["bias"] = torch.randn(e, n, generator=g, device=DEV).to(dtype)
        return s
    s["w"] = _weights(2 * n, k, case["fmt"], g, e)
    s["down"] = _weights(k, n, case["fmt"], g, e)
    s["x"] = _activations(t, k, dtype, g)
    s["res"] = (torch.randn(t, k, generator=g, device=DEV) * 3).to(dtype)
    return s


def _package():
    pkg = os.path.abspath("trellis-everywhere_b200")          # the folder users put on sys.path; the working folder is the repository's root
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from trellis_b200 import experts, microscale
    return microscale, experts


def run(s):
    c = s["case"]
    return _run_own(c, s) if own else _run_plain(c, s)


def _run_own(c, s):
    ms, ex = _package()
    kind = c["kind"]
    if kind == "linear":
        return ms.linear(s["x"], ms.Microscaled(*s["w"], (c["n"], c["k"]), c["fmt"]), bias=s["bias"], activation=c["act"] or None, residual=s["res"])
    if kind == "route":
        return tuple(ex.route(s["logits"], c["top"], score=c["score"], normalize=c["norm"]))
    if kind == "combine":
        return ex.combine(s["y"], ex.Routing(*s["routing"]), residual=s["res"])
    if kind == "experts":
        w = ex.ExpertMatrices(*s["w"], (c["e"], c["n"], c["k"]), c["fmt"])
        return ex.grouped_linear(s["x"], w, s["routing"][4], tokens=s["routing"][3] if c["gather"] else None, bias=s["bias"], activation=c["act"] or None)
    r = ex.route(s["logits"], c["top"])
    up = ex.ExpertMatrices(*s["w"], (c["e"], 2 * c["n"], c["k"]), c["fmt"])
    down = ex.ExpertMatrices(*s["down"], (c["e"], c["k"], c["n"]), c["fmt"])
    h = ex.grouped_linear(s["x"], up, r.offsets, tokens=r.tokens, activation=c["act"])
    return ex.combine(ex.grouped_linear(h, down, r.offsets, dtype=torch.float32), r, residual=s["res"])


def _run_plain(c, s):
    kind, dtype = c["kind"], s["dtype"]
    if kind == "route":
        return _route(s["logits"], c["top"], c["score"], c["norm"])
    if kind == "combine":
        return _combine(s["y"], s["routing"][0], s["routing"][2], s["res"]).to(dtype)
    w = _values(*s["w"], 2 * c["n"] if kind == "layer" else c["n"], c["k"], c["fmt"])
    if kind == "linear":
        return _epilogue(s["x"].float() @ w.t(), s["bias"], c["act"], s["res"]).to(dtype)
    if kind == "experts":
        x = s["x"][s["routing"][3].long()] if c["gather"] else s["x"]
        return _grouped(x, w, s["routing"][4], s["room"], s["bias"], c["act"]).to(dtype)
    weights, _, places, tokens, offsets = _route(s["logits"], c["top"], "softmax", True)
    h = _grouped(s["x"][tokens.long()], w, offsets, s["room"], None, c["act"])
    y = _grouped(h, _values(*s["down"], c["k"], c["n"], c["fmt"]), offsets, s["room"], None, "")
    return _combine(y, weights, places, s["res"]).to(dtype)


def work(case):
    kind, t = case["kind"], 4 if case["type"] == "float32" else 2
    held = lambda n, k: (0.5 + 1 / BLOCK[case["fmt"]]) * n * k  # noqa: E731  bytes in 4 bits with their share of scales
    if kind == "linear":
        n, k, m = case["n"], case["k"], case["m"]
        out = n // 2 if case["act"] in GATED else n
        return {"bytes": held(n, k) + t * m * (k + out * (2 if case["res"] else 1)) + t * n * case["bias"], "flops": 2 * m * n * k}
    tokens, e, top = case["t"], case["e"], case["top"]
    rows = tokens * top
    if kind == "route":
        return {"bytes": t * tokens * e + 16 * rows + 4 * (e + 1), "flops": 4 * tokens * e}
    n = case["n"]
    if kind == "combine":
        return {"bytes": t * n * (rows + tokens * (2 if case["res"] else 1)) + 8 * rows, "flops": 2 * rows * n}
    k, used = case["k"], min(e, rows)                         # no more experts than rows have weights to be read
    if kind == "experts":
        out = n // 2 if case["act"] in GATED else n
        return {"bytes": used * held(n, k) + t * (k * (tokens if case["gather"] else rows) + rows * out), "flops": 2 * rows * n * k}
    return {"bytes": used * 3 * held(n, k) + t * tokens * (3 * k + e), "flops": 6 * rows * n * k}


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def _values_exact(codes, scales, row, n, k, fmt):
    """fp64 values of one matrix, from the bits of the two small types."""
    c = torch.empty(n, 2 * codes.shape[1], dtype=torch.int32, device=codes.device)
    c[:, 0::2] = codes.int() & 15
    c[:, 1::2] = codes.int() >> 4
    e, mant = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, mant / 2, (1 + mant / 2) * torch.exp2((e - 1).double()))
    v = torch.where(c >= 8, -v, v)
    r, b = torch.arange(n, device=codes.device)[:, None], (torch.arange(k, device=codes.device) // BLOCK[fmt])[None, :]
    s = scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4].int()
    if fmt == "nvfp4":
        se, sm = s >> 3, (s & 7).double()
        d = torch.where(se == 0, sm / 8 * 2.0 ** -6, (1 + sm / 8) * torch.exp2((se - 7).double())) * row.double()[:, None]
    else:
        d = torch.exp2((s - 127).double())
    return v[:, :k] * d


def _act_exact(h, act):
    if act in GATED:
        return _act_exact(h[:, 0::2], {"swiglu": "silu", "geglu": "gelu"}[act]) * h[:, 1::2]
    if act == "relu":
        return h.clamp(min=0)
    if act == "gelu":
        return h * torch.special.ndtr(h)
    if act == "gelu_tanh":
        return h * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (h + 0.044715 * h ** 3))
    return h * torch.sigmoid(h) if act == "silu" else h


def _grouped_exact(x, w, offsets, n, k, fmt, bias, act):
    out = []
    bounds = offsets.tolist()
    for i, (a, b) in enumerate(zip(bounds, bounds[1:])):
        if b > a:
            h = x[a:b] @ _values_exact(w[0][i], w[1][i], None if w[2] is None else w[2][i], n, k, fmt).t()
            out.append(_act_exact(h if bias is None else h + bias[i].double(), act))
    return torch.cat(out)


def _route_exact(logits, top, score, norm):
    """Chosen one after the other: the largest that is left, of equal ones the first."""
    t, e = logits.shape
    v = logits.double()
    w = torch.softmax(v, 1) if score == "softmax" else torch.sigmoid(v)
    left, experts = v.clone(), []
    number = torch.arange(e, device=v.device)
    for _ in range(top):
        first = torch.where(left == left.amax(1, keepdim=True), number, e).amin(1)
        experts.append(first)
        left[torch.arange(t, device=v.device), first] = -math.inf
    experts = torch.stack(experts, 1)
    weights = w.gather(1, experts)
    if norm:
        weights = weights / weights.sum(1, keepdim=True)
    flat = experts.flatten()
    count = torch.bincount(flat, minlength=e)
    key = flat * (t * top) + torch.arange(t * top, device=v.device)
    order = torch.argsort(key)
    places = torch.argsort(order)
    offsets = torch.cat((count.new_zeros(1), torch.cumsum(count, 0)))
    return weights, experts.int(), places.reshape(t, top).int(), torch.div(order, top, rounding_mode="floor").int(), offsets.int()


def _combine_exact(y, weights, places, residual):
    out = torch.einsum("tkn,tk->tn", y.double()[places.long()], weights.double())
    return out if residual is None else out + residual.double()


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _route_exact(s["logits"], case["top"], case["score"], case["norm"])
    if kind == "combine":
        return _combine_exact(s["y"], s["routing"][0], s["routing"][2], s["res"])
    n, k, fmt, act = case["n"], case["k"], case["fmt"], case["act"]
    x = s["x"].double()
    if kind == "linear":
        h = x @ _values_exact(*s["w"], n, k, fmt).t()
        h = _act_exact(h if s["bias"] is None else h + s["bias"].double(), act)
        return h if s["res"] is None else h + s["res"].double()
    if kind == "experts":
        if case["gather"]:
            x = x[s["routing"][3].long()]
        return _grouped_exact(x, s["w"], s["routing"][4], n, k, fmt, s["bias"], act)
    weights, _, places, tokens, offsets = _route_exact(s["logits"], case["top"], "softmax", True)
    h = _grouped_exact(x[tokens.long()], s["w"], offsets, 2 * n, k, fmt, None, act)
    return _combine_exact(_grouped_exact(h, s["down"], offsets, k, n, fmt, None, ""), weights, places, s["res"])
