"""Quantizer plug-in interface (``src/trellis/quant.py:20-26`` of the reference) for the B200 codec.

The reference's model-level drivers walk ``nn.Linear`` modules and call
``Quantizer.quantize_weight(w) -> w_fake``; ``TrellisQuantizer`` is that interface
on top of the CUDA encoder, with or without LDLQ feedback.  ``MicroscaleQuantizer`` is the
same for the 4-bit microscaled formats, and ``MicroscaledLinear`` / ``apply_microscaled`` keep
the weights in 4 bits and multiply by them there (no counterpart in the reference).
"""
from __future__ import annotations

import math
import zlib
from typing import Callable, Optional

import torch
import torch.nn as nn

from . import microscale
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


class MicroscaledLinear(nn.Module):
    """``nn.Linear`` for inference with its weight in 4 bits (no gradient: inputs that need one are refused).

    ``activations=16``: inputs stay as they are (``microscale.linear``).  ``activations=4``: inputs are quantised token by
    token (``microscale.quantize``) and both sides multiplied in 4 bits (``microscale.matmul``); ``rotate`` then puts both
    sides in a rotated space of the input channels, which leaves the product what it is.
    """

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, fmt: str = "nvfp4", activations: int = 16,
                 rotate: int = 0, seed: int = 0):
        super().__init__()
        if activations not in (4, 16):
            raise ValueError("activations must be 4 or 16")
        if rotate and activations == 16:
            raise ValueError("rotate needs activations=4: inputs are rotated as they are quantised")
        self.fmt, self.activations, self.rotate = fmt, activations, rotate
        self.out_features, self.in_features = weight.shape
        wd = weight.detach().to(_cuda_device(weight))
        signs = _signs(self.in_features, seed, wd.device) if rotate else None
        q = microscale.quantize(wd, fmt, rotate, signs)
        for name, t in (("codes", q.codes), ("scales", q.scales), ("row_scale", q.row_scale), ("signs", signs),
                        ("bias", None if bias is None else bias.detach().to(wd.device))):
            self.register_buffer(name, t)

    def _apply(self, fn, recurse: bool = True):
        """Moves with the module, but the scales and signs stay fp32 whatever type the module is given."""
        kept = {name: t for name in ("row_scale", "signs") if (t := getattr(self, name)) is not None}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            now = getattr(self, name)
            if now.dtype != torch.float32:
                setattr(self, name, t.to(now.device))
        return self

    @property
    def weight(self) -> "microscale.Microscaled":
        return microscale.Microscaled(self.codes, self.scales, self.row_scale, (self.out_features, self.in_features), self.fmt)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.activations == 16:
            y = microscale.linear(x, self.weight)
        else:
            if not x.dim() or x.shape[-1] != self.in_features:
                raise ValueError(f"x must be [..., {self.in_features}], got {tuple(x.shape)}")
            q = microscale.quantize(x.reshape(math.prod(x.shape[:-1]), self.in_features), self.fmt, self.rotate, self.signs)
            y = microscale.matmul(q, self.weight, x.dtype).reshape(*x.shape[:-1], self.out_features)
        return y if self.bias is None else y + self.bias.to(y.dtype)

    def extra_repr(self) -> str:
        return f"{self.in_features} -> {self.out_features}, {self.fmt}, activations={self.activations}, rotate={self.rotate}"


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
