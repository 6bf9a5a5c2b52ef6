"""Quantizer plug-in interface (``src/trellis/quant.py:20-26`` of the reference) for the B200 codec.

The reference's model-level drivers walk ``nn.Linear`` modules and call
``Quantizer.quantize_weight(w) -> w_fake``; ``TrellisQuantizer`` is that interface
on top of the CUDA encoder, with or without LDLQ feedback.  ``MicroscaleQuantizer`` is the
same for the 4-bit microscaled formats, and ``MicroscaledLinear`` / ``apply_microscaled`` keep
the weights in 4 bits and multiply by them there, ``MicroscaledExperts`` those of a mixture of experts (no counterpart in the reference).
"""
from __future__ import annotations

import math
import zlib
from typing import Callable, Optional

import torch
import torch.nn as nn

from . import experts, microscale
from .ldlq import tcq_quantize_weight_ldlq
from .qtip import CodebookLike, _cuda_device, block_hadamard, tcq_quantize_weight


class Quantizer:
    """Interface: map a weight matrix ``[out, in]`` to its fake-quantised version."""
    name: str = "identity"
    bpw: float = 16.0

    def quantize_weight(self, w: torch.Tensor) -> torch.Tensor:  # pragma: no cover - interface
        return w


class TrellisQuantizer(Quantizer):
    """Tail-biting trellis-coded quantisation at K bits per weight on the B200 encoder.

    ``hessian`` (optional): callable ``name -> H`` or a tensor; when given, LDLQ
    feedback is used for that matrix, as ``scripts/run_tcq_eval.py:113-127`` does.
    ``seed_from_name`` reproduces the driver's ``seed = crc32(name)``.
    """

    def __init__(self, K: int = 3, codebook: CodebookLike = "mcg", seed: int = 0, sigma_reg: float = 0.025):
        self.K, self.codebook, self.seed, self.sigma_reg = K, codebook, seed, sigma_reg
        self.name = f"tcq-b200-k{K}"
        self.bpw = float(K)

    def quantize_weight(self, w: torch.Tensor, H: Optional[torch.Tensor] = None, seed: Optional[int] = None) -> torch.Tensor:
        s = self.seed if seed is None else seed
        if H is None:
            return tcq_quantize_weight(w, self.K, self.codebook, seed=s, backend="b200")
        return tcq_quantize_weight_ldlq(w, self.K, self.codebook, H, seed=s, sigma_reg=self.sigma_reg, backend="b200")


def _signs(k: int, seed: int, device) -> torch.Tensor:
    """+-1 for every input channel, from the CPU generator (as ``qtip.IPContext`` draws its signs)."""
    gen = torch.Generator(device="cpu").manual_seed(seed)
    return torch.empty(k, dtype=torch.float32).random_(0, 2, generator=gen).mul_(2).sub_(1).to(device)


class MicroscaleQuantizer(Quantizer):
    """4-bit microscaled floating point (``microscale.quantize``), optionally in a rotated space of the input channels.

    ``rotate`` (16 to 128, dividing the matrix's input channels; 0: none) applies seeded signs and a block Hadamard
    transform before the quantisation and takes them back after it.
    """

    def __init__(self, fmt: str = "nvfp4", rotate: int = 0, seed: int = 0):
        if fmt not in microscale.FORMATS:
            raise ValueError(f"unknown microscaled format {fmt!r}; expected one of {sorted(microscale.FORMATS)}")
        if rotate not in microscale.ROTATIONS:
            raise ValueError(f"rotate={rotate} must be one of {microscale.ROTATIONS}")
        self.fmt, self.rotate, self.seed = fmt, rotate, seed
        self.name = f"{fmt}-b200" + (f"-h{rotate}" if rotate else "")
        self.bpw = 4.0 + 8.0 / microscale.BLOCKS[fmt]

    @torch.no_grad()
    def quantize_weight(self, w: torch.Tensor, seed: Optional[int] = None) -> torch.Tensor:
        wd = w.to(_cuda_device(w))
        if not self.rotate:
            back = microscale.dequantize(microscale.quantize(wd, self.fmt), w.dtype)
        else:
            signs = _signs(w.shape[1], self.seed if seed is None else seed, wd.device)
            z = microscale.dequantize(microscale.quantize(wd, self.fmt, self.rotate, signs))
            back = block_hadamard(z, 1, self.rotate) * signs
        return back.to(dtype=w.dtype, device=w.device)


def _apply_in_fp32(module: nn.Module, names, apply) -> nn.Module:
    """``nn.Module._apply`` of a module whose buffers of these names stay fp32 whatever type it is given."""
    kept = {name: t for name in names if (t := getattr(module, name)) is not None}
    apply()
    for name, t in kept.items():
        now = getattr(module, name)
        if now.dtype != torch.float32:
            setattr(module, name, t.to(now.device))
    return module


class MicroscaledLinear(nn.Module):
    """``nn.Linear`` for inference with its weight in 4 bits (no gradient: inputs that need one are refused).

    ``activations=16``: inputs stay as they are (``microscale.linear``).  ``activations=4``: inputs are quantised token by
    token (``microscale.quantize``) and both sides multiplied in 4 bits (``microscale.matmul``); ``rotate`` then puts both
    sides in a rotated space of the input channels, which leaves the product what it is.

    ``activation`` ("relu", "gelu", "gelu_tanh", "silu", or gated by pairs of rows, "geglu", "swiglu": ``microscale.linear``) and the ``residual`` that ``forward`` may be given are
    applied to the sums of the product, bias included, before they are rounded (``activations=16``).
    """

    activation: Optional[str] = None                        # (of modules that were saved without one)

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, fmt: str = "nvfp4", activations: int = 16,
                 rotate: int = 0, seed: int = 0, activation: Optional[str] = None):
        super().__init__()
        if activations not in (4, 16):
            raise ValueError("activations must be 4 or 16")
        if rotate and activations == 16:
            raise ValueError("rotate needs activations=4: inputs are rotated as they are quantised")
        if activation is not None and activations == 4:
            raise ValueError("an activation in the product needs activations=16")
        microscale._check_act(activation, weight.shape[0])
        self.fmt, self.activations, self.rotate, self.activation = fmt, activations, rotate, activation
        self.out_features, self.in_features = weight.shape
        wd = weight.detach().to(_cuda_device(weight))
        signs = _signs(self.in_features, seed, wd.device) if rotate else None
        q = microscale.quantize(wd, fmt, rotate, signs)
        for name, t in (("codes", q.codes), ("scales", q.scales), ("row_scale", q.row_scale), ("signs", signs),
                        ("bias", None if bias is None else bias.detach().to(wd.device))):
            self.register_buffer(name, t)

    def _apply(self, fn, recurse: bool = True):
        """Moves with the module, but the scales and signs stay fp32 whatever type the module is given."""
        return _apply_in_fp32(self, ("row_scale", "signs"), lambda: super(MicroscaledLinear, self)._apply(fn, recurse))

    @property
    def weight(self) -> "microscale.Microscaled":
        return microscale.Microscaled(self.codes, self.scales, self.row_scale, (self.out_features, self.in_features), self.fmt)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.activation is not None or residual is not None:
            if self.activations == 4:
                raise ValueError("a residual in the product needs activations=16")
            return microscale.linear(x, self.weight, self.bias, self.activation, residual)
        if self.activations == 16:
            y = microscale.linear(x, self.weight)
        else:
            if not x.dim() or x.shape[-1] != self.in_features:
                raise ValueError(f"x must be [..., {self.in_features}], got {tuple(x.shape)}")
            q = microscale.quantize(x.reshape(math.prod(x.shape[:-1]), self.in_features), self.fmt, self.rotate, self.signs)
            y = microscale.matmul(q, self.weight, x.dtype).reshape(*x.shape[:-1], self.out_features)
        return y if self.bias is None else y + self.bias.to(y.dtype)

    def extra_repr(self) -> str:
        then = "" if self.activation is None else f", {self.activation}"
        return f"{self.in_features} -> {self.out_features}, {self.fmt}, activations={self.activations}, rotate={self.rotate}{then}"


class MicroscaledExperts(nn.Module):
    """A mixture of experts for inference with its matrices in 4 bits: ``sum_e weight_e * (act(x @ gate_e.T) * (x @ up_e.T)) @ down_e.T`` over each token's ``top_k`` experts.

    ``up [E, n, k]`` and ``down [E, k_out, n]``; ``gate`` like ``up`` with a gated ``activation`` ("swiglu", "geglu"), None with another (``act(x @ up_e.T)``).  Biases ``[E, n]``,
    ``[E, n]``, ``[E, k_out]`` or None.  The experts and their weights come of logits (``experts.route`` with ``score`` and ``normalize``): ``router(x)``, where one is given, or what
    ``forward`` is handed.  Sums between the products stay fp32 but for the rounding of the second one's input to ``inner``, x's type where that is None: fp16 holds inner results up to 65504,
    beyond which they are infinite, and bfloat16 any.
    """

    inner: Optional[torch.dtype] = None                     # (of modules that were saved without one)

    def __init__(self, up: torch.Tensor, down: torch.Tensor, top_k: int, gate: Optional[torch.Tensor] = None, fmt: str = "nvfp4", activation: str = "swiglu",
                 score: str = "softmax", normalize: bool = True, router: Optional[nn.Module] = None, up_bias: Optional[torch.Tensor] = None,
                 gate_bias: Optional[torch.Tensor] = None, down_bias: Optional[torch.Tensor] = None, inner: Optional[torch.dtype] = None):
        super().__init__()
        if inner not in (None, torch.float16, torch.bfloat16):
            raise ValueError(f"inner={inner}: expected None, float16 or bfloat16")
        if up.dim() != 3 or down.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[2] != up.shape[1]:
            raise ValueError(f"up must be [experts, n, k] and down [experts, k_out, n], got {tuple(up.shape)} and {tuple(down.shape)}")
        if (gate is not None) != (activation in microscale.GATED):
            raise ValueError(f"activation {activation!r} {'takes' if gate is None else 'does not take'} a gate")
        if gate is not None and gate.shape != up.shape:
            raise ValueError(f"gate must be like up, {list(up.shape)}, got {list(gate.shape)}")
        if gate_bias is not None and (gate is None or up_bias is None) or (gate is not None and up_bias is not None and gate_bias is None):
            raise ValueError("gate_bias goes with a gate and up_bias, and up_bias of a gated layer with gate_bias")
        microscale._check_act(activation, 2)
        if score not in experts.SCORES or not 1 <= top_k <= min(up.shape[0], experts.MOST_CHOSEN):
            raise ValueError(f"score={score!r}, top_k={top_k}: expected one of {sorted(experts.SCORES)} and 1 to {min(up.shape[0], experts.MOST_CHOSEN)}")
        self.fmt, self.activation, self.top_k, self.score, self.normalize, self.router, self.inner = fmt, activation, top_k, score, normalize, router, inner
        self.shape = tuple(up.shape) + (down.shape[1],)     # experts, inner, in and out features
        dev = _cuda_device(up)
        with torch.no_grad():
            first = up.detach().to(dev)
            if gate is not None:
                first = microscale.interleave(gate.detach().to(dev), first)
            q, r = experts.quantize_experts(first, fmt), experts.quantize_experts(down.detach().to(dev), fmt)
            del first
            if gate_bias is not None:
                up_bias = torch.stack((gate_bias.detach(), up_bias.detach()), -1).flatten(-2)
        for name, t in (("up_codes", q.codes), ("up_scales", q.scales), ("up_row_scale", q.row_scale), ("down_codes", r.codes), ("down_scales", r.scales), ("down_row_scale", r.row_scale),
                        ("up_bias", None if up_bias is None else up_bias.detach().to(dev)), ("down_bias", None if down_bias is None else down_bias.detach().to(dev))):
            self.register_buffer(name, t)

    def _apply(self, fn, recurse: bool = True):
        """Moves with the module, but the row scales stay fp32 whatever type the module is given."""
        return _apply_in_fp32(self, ("up_row_scale", "down_row_scale"), lambda: super(MicroscaledExperts, self)._apply(fn, recurse))

    @property
    def up(self) -> "experts.ExpertMatrices":
        e, n, k, _ = self.shape
        return experts.ExpertMatrices(self.up_codes, self.up_scales, self.up_row_scale, (e, 2 * n if self.activation in microscale.GATED else n, k), self.fmt)

    @property
    def down(self) -> "experts.ExpertMatrices":
        e, n, _, out = self.shape
        return experts.ExpertMatrices(self.down_codes, self.down_scales, self.down_row_scale, (e, out, n), self.fmt)

    def forward(self, x: torch.Tensor, logits: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x [..., k]`` in fp16 or bf16, ``logits [..., E]`` where there is no router, ``residual [..., k_out]`` of x's type added in the same pass."""
        e, _, k, out = self.shape
        if not x.dim() or x.shape[-1] != k:
            raise ValueError(f"x must be [..., {k}], got {tuple(x.shape)}")
        if (logits is None) == (self.router is None):
            raise ValueError("logits come either from the router or with the call")
        tokens = math.prod(x.shape[:-1])
        flat = x.reshape(tokens, k)
        r = experts.route((self.router(flat) if logits is None else logits).reshape(tokens, e), self.top_k, self.score, self.normalize)
        h = experts.grouped_linear(flat, self.up, r.offsets, r.tokens, self.up_bias, self.activation, self.inner)
        y = experts.grouped_linear(h, self.down, r.offsets, bias=self.down_bias, dtype=torch.float32)
        return experts.combine(y, r, None if residual is None else residual.reshape(tokens, out), x.dtype).reshape(*x.shape[:-1], out)

    def extra_repr(self) -> str:
        e, n, k, out = self.shape
        return f"{e} experts, {self.top_k} a token, {k} -> {n} -> {out}, {self.activation}, {self.fmt}"


def seed_from_name(name: str) -> int:
    """Per-matrix seed of the reference driver (``zlib.crc32(name)``, run_tcq_eval.py:115)."""
    return zlib.crc32(name.encode())


@torch.no_grad()
def apply_fake_quant(model: nn.Module, quantizer: Quantizer, skip: Callable[[str], bool] = lambda n: False) -> int:
    """Replace every ``nn.Linear`` weight by its fake-quantised version (quant.py:72-85). Returns the count."""
    count = 0
    for name, mod in model.named_modules():
        if isinstance(mod, nn.Linear) and not skip(name):
            mod.weight.data = quantizer.quantize_weight(mod.weight.data).to(mod.weight.dtype)
            count += 1
    return count


_FORWARD_HOOKS = ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks", "_forward_pre_hooks_with_kwargs")
_STATE_HOOKS = ("_state_dict_hooks", "_state_dict_pre_hooks", "_load_state_dict_pre_hooks", "_load_state_dict_post_hooks")


def _check_replaceable(name: str, layer: nn.Linear) -> None:
    """Refuses a layer that is more than its weight and bias (backward hooks are left out: no gradient passes its replacement)."""
    if "weight" not in layer._parameters or "forward" in layer.__dict__ or any(getattr(layer, h) for h in _STATE_HOOKS):
        raise ValueError(f"{name}: its weight is computed, its forward is its own or hooks read its state: take that off first, or skip it")
    if layer.weight.is_meta or (layer.bias is not None and layer.bias.is_meta):
        raise ValueError(f"{name}: its weight or bias has no values yet (meta device)")


@torch.no_grad()
def apply_microscaled(model: nn.Module, fmt: str = "nvfp4", activations: int = 16, rotate: int = 0,
                      skip: Callable[[str], bool] = lambda n: False) -> int:
    """Replace every ``nn.Linear`` below ``model`` by a ``MicroscaledLinear`` (seeds by name, as ``seed_from_name``). Returns the count.

    A layer that stands under several names is replaced under each that is not skipped, by one ``MicroscaledLinear``.  Subclasses of
    ``nn.Linear`` stay: they may do more than its product, or their owner may read their weight (``nn.MultiheadAttention`` does).
    A layer's mode (``training``) and its forward hooks go to its replacement; a layer with a computed weight (weight norm, pruning),
    a forward of its own or hooks on its state is refused.  All is checked before the first layer is replaced.
    """
    microscale._check_fmt(fmt)
    layers = {}                                              # layer -> its names
    for name, mod in model.named_modules(remove_duplicate=False):
        if type(mod) is nn.Linear and name and not skip(name):
            layers.setdefault(mod, []).append(name)
    for mod, names in layers.items():
        if rotate and mod.in_features % rotate:
            raise ValueError(f"{names[0]}: rotate={rotate} does not divide its {mod.in_features} input channels")
        microscale._check_dtype(mod.weight.dtype)
        _check_replaceable(names[0], mod)
    count = len(layers)
    while layers:                                            # a layer's own weight goes before the next one's 4 bits are made
        mod = next(iter(layers))
        names = layers.pop(mod)
        new = MicroscaledLinear(mod.weight.data, mod.bias, fmt, activations, rotate, seed_from_name(names[0])).train(mod.training)
        for hooks in _FORWARD_HOOKS:                         # (the same dict: a handle from the layer still removes its hook)
            setattr(new, hooks, getattr(mod, hooks))
        for name in names:
            parent, _, leaf = name.rpartition(".")
            setattr(model.get_submodule(parent), leaf, new)
    return count
