"""Products with an epilogue, routing and combining from their definitions, in 64 bits, with bounds of what a kernel that rounds where it may is off by."""
import math

import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
GATED = {"swiglu": "silu", "geglu": "gelu"}


def activate(h, act):
    if act is None:
        return h
    if act == "relu":
        return h.clamp(min=0)
    if act == "gelu":
        return h * 0.5 * torch.special.erfc(-h * math.sqrt(0.5))
    if act == "gelu_tanh":
        return h * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (h + 0.044715 * h ** 3))
    assert act == "silu"
    return h * torch.sigmoid(h)


def sums_bound(x, w, fmt):
    """Of fp32 sums of x's 4-bit parts times w (fp64 [m, k], [n, k]).  With s of a block, 1.7 s <= amax: x / s is rounded to 15 binary places, 2^-16 s <= 2^-16.7 amax off.  nvfp4
    leaves digits out whose scale is below 2^-17 of the row's largest scale S, 1.7 S <= the row's largest: 4 (1/8 + 1/64 + ...) 2^-17 S <= 0.572 2^-17 / 1.7 = 2^-18.5 of the row's largest.
    For every 64 columns 2^-22 of the sum of the parts' magnitudes: the first is |x| + 0.572 s at most and the others 0.572 s together, |x| + 1.15 s <= 1.7 amax."""
    b, k = BLOCK[fmt], x.shape[1]
    amax = torch.nn.functional.pad(x.abs(), (0, -k % b)).reshape(x.shape[0], -1, b).amax(2).repeat_interleave(b, 1)[:, :k]
    a = amax @ w.abs().t()
    bound = a * (2.0 ** -16.7 + 1.7 * (k / 64 + 8) * 2.0 ** -22)
    if fmt == "nvfp4":
        bound = bound + 2.0 ** -18.5 * x.abs().amax(1, keepdim=True) * w.abs().sum(1)[None]
    return bound


def fp32_bound(x, w, parts=True):
    """Of fp32 sums: 2^-24 of the sum of magnitudes for each of up to k additions is far more than pairs of them make; a tree of 256s has k / 256 + 32 steps."""
    return (x.abs() @ w.abs().t()) * (x.shape[1] / 64 + 32) * 2.0 ** -23


def epilogue(h, bound, bias, act, residual, dtype):
    """(y, bound): activations grow an error by at most 1.13 (the steepest slope of GELU and SiLU) and add 2^-20 of their value (fp32 functions of a few ulp, and of arguments that
    are rounded), the residual 2^-24; the result is rounded by half a step at most, or half the least number."""
    if bias is not None:
        h = h + bias.double()
        bound = bound + h.abs() * 2.0 ** -24
    if act in GATED:
        g, u, bg, bu = h[:, 0::2], h[:, 1::2], bound[:, 0::2], bound[:, 1::2]
        a = activate(g, GATED[act])
        y = a * u
        slack = 2.0 ** -20 * (a.abs() + g.abs() * 2.0 ** -4)
        bound = (1.13 * bg + slack) * (u.abs() + bu) + a.abs() * bu + y.abs() * 2.0 ** -23
    else:
        y = activate(h, act)
        bound = bound if act in (None, "relu") else 1.13 * bound + 2.0 ** -20 * (y.abs() + h.abs() * 2.0 ** -4)
    if residual is not None:
        y = y + residual.double()
        bound = bound + y.abs() * 2.0 ** -24
    info = torch.finfo(dtype)
    return y, bound + (y.abs() + bound) * info.eps / 2 + info.smallest_normal * info.eps / 2


def route(logits, top, score, normalize):
    """(weights fp64, experts, places, tokens, offsets), one token after the other on the CPU."""
    v = logits.double().cpu()
    t, e = v.shape
    weights, experts = torch.zeros(t, top, dtype=torch.float64), torch.full((t, top), -1, dtype=torch.int64)
    for i in range(t):
        row = v[i].tolist()
        order = sorted((n for n in range(e) if row[n] != -math.inf), key=lambda n: (-(math.inf if math.isnan(row[n]) else row[n]), 0 if math.isnan(row[n]) else 1, n))[:top]
        if not order:
            continue
        c = v[i][order]
        if score == "softmax":
            top_value = c[0]
            w = torch.exp(c - top_value) / (torch.exp(c - top_value).sum() if normalize else torch.exp(v[i] - top_value).sum())
        else:
            w = torch.sigmoid(c)
            if normalize:
                w = torch.softmax(torch.nn.functional.logsigmoid(c), 0)
        weights[i, :len(order)], experts[i, :len(order)] = w, torch.tensor(order)
    flat = experts.flatten()
    rows = sorted((j for j in range(t * top) if flat[j] >= 0), key=lambda j: (int(flat[j]), j))
    places, tokens = torch.full((t * top,), -1, dtype=torch.int64), torch.full((t * top,), -1, dtype=torch.int64)
    for place, j in enumerate(rows):
        places[j], tokens[place] = place, j // top
    counts = torch.bincount(flat[flat >= 0], minlength=e)
    return weights, experts, places.reshape(t, top), tokens, torch.cat((torch.zeros(1, dtype=torch.int64), counts.cumsum(0)))
