"""A splat refiner: a small sequence model whose tokens are Gaussians.

The Gaussians of a scene, in an order that keeps neighbours together
(:func:`morton_order`), follow a few learned scene tokens; blocks of windowed
attention and a gated recurrence along the order predict an update of every
parameter, and the refined splats go through the rasterizer like any others, so
the refiner trains on rendered images. Scenes of different sizes are packed
into one batch. This module runs the sequence operators of the package together
as they are meant to be used:

* training and whole-scene inference: :meth:`SplatRefiner.forward`
* one new Gaussian at a time (a scene that arrives as a stream):
  :meth:`SplatRefiner.stream` and :meth:`SplatRefiner.step`, for a causal refiner
  (``right=0``)
* 8-bit products for serving: :meth:`SplatRefiner.quantize`

Activations are bfloat16, the residual stream float32.
"""

from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch
from torch import nn

from .attention import window_attention, window_attention_step, window_cache
from .norm import rms_norm, rms_norm_e4m3
from .recurrence import gated_scan, gated_scan_step
from .sequences import PackedSequences
from .splats import GaussianSplat

_NAMES = ("mean", "rotation", "scale", "opacity", "color")
_DEAD_OPACITY = 0.005  # as relocation counts splats as dead


def morton_order(points: torch.Tensor, bits: int = 16) -> torch.Tensor:
    """The order of ``points`` [N, 3] along a Z-curve through their bounding box
    cut into ``2**bits`` cells a side: indices, ties by index."""
    if points.dim() != 2 or points.shape[1] != 3 or not 1 <= bits <= 20:
        raise ValueError(f"morton_order takes [N, 3] points and 1 to 20 bits, got "
                         f"{tuple(points.shape)} and {bits}")
    if len(points) == 0:
        return torch.empty(0, dtype=torch.int64, device=points.device)
    points = points.detach().double()
    low, high = points.amin(0), points.amax(0)
    cells = 2 ** bits
    cell = ((points - low) / (high - low).clamp(min=1e-30) * cells).long().clamp(0, cells - 1)
    code = torch.zeros(len(points), dtype=torch.int64, device=points.device)
    for bit in range(bits):
        for axis in range(3):
            code |= (cell[:, axis] >> bit & 1) << (3 * bit + axis)
    return torch.argsort(code, stable=True)


def _alive(splats: GaussianSplat) -> torch.Tensor:
    """Which splats the others' attention may see."""
    return splats.opacity.detach()[:, 0].sigmoid() >= _DEAD_OPACITY


class _Product(nn.Linear):
    """A bfloat16 linear layer that can be switched to 8-bit products."""

    def __init__(self, inputs: int, outputs: int, device=None):
        super().__init__(inputs, outputs, bias=False, device=device, dtype=torch.bfloat16)
        # Made from the weight: they move with the module, but are not saved.
        self.register_buffer("codes", None, persistent=False)
        self.register_buffer("scales", None, persistent=False)
        self.rounded = None

    def _changes(self) -> int | None:
        """The count of the weight's changes in place (inference tensors have none)."""
        return None if self.weight.is_inference() else self.weight._version

    def quantize(self) -> None:
        """e4m3 weights with one scale an output, of the weight as it is now."""
        self.rounded = self._changes()
        w = self.weight.detach().float()
        self.scales = (w.abs().amax(1) / 448.0).clamp(min=1e-12)
        self.codes = (w / self.scales[:, None]).to(torch.float8_e4m3fn)

    def eight_bit(self, codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        if self.rounded != self._changes():  # an optimizer's step, a loaded checkpoint
            self.quantize()
        return torch._scaled_mm(codes, self.codes.t(), scale[:, None], self.scales[None],
                                out_dtype=torch.bfloat16)


@dataclass(frozen=True)
class RefinerShape:
    """Sizes of a refiner. ``left`` and ``right``: the attention's window along
    the order; ``first``: scene tokens, which stay visible."""

    width: int = 256
    blocks: int = 2
    heads: int = 4
    kv_heads: int = 2
    left: int = 256
    right: int = 256
    first: int = 4


class _Block(nn.Module):
    def __init__(self, shape: RefinerShape, device=None):
        super().__init__()
        self.shape = shape
        dim = shape.width // shape.heads
        self.split = [shape.heads * dim, shape.kv_heads * dim, shape.kv_heads * dim]
        self.dim = dim

        def ones():
            return nn.Parameter(torch.ones(shape.width, device=device, dtype=torch.bfloat16))

        self.norm_attend, self.norm_mix = ones(), ones()
        self.qkv = _Product(shape.width, sum(self.split), device)
        self.attend_out = _Product(self.split[0], shape.width, device)
        self.mix = _Product(shape.width, 2 * shape.width, device)
        self.mix_out = _Product(shape.width, shape.width, device)

    def _normed(self, x, residual, weight, product):
        """The product of the norm of ``x + residual``, and the sum."""
        if product.codes is not None and not torch.is_grad_enabled():
            codes, scale, residual = rms_norm_e4m3(x, weight, residual)
            return product.eight_bit(codes, scale), residual
        y, residual = rms_norm(x, weight, residual)
        return product(y), residual

    def _heads(self, qkv):
        return (t.unflatten(-1, (-1, self.dim)) for t in qkv.split(self.split, -1))

    def forward(self, x, residual, packed, valid):
        s = self.shape
        qkv, residual = self._normed(x, residual, self.norm_attend, self.qkv)
        x = window_attention(*self._heads(qkv), packed, left=s.left, right=s.right, first=s.first,
                             valid=valid)
        x = self.attend_out(x.flatten(1))
        mix, residual = self._normed(x, residual, self.norm_mix, self.mix)
        x, _ = gated_scan(*mix.chunk(2, -1), packed)
        return self.mix_out(x), residual

    def step(self, x, residual, positions, cache, state, valid, cache_valid):
        qkv, residual = self._normed(x, residual, self.norm_attend, self.qkv)
        x = window_attention_step(*self._heads(qkv), *cache, positions, first=self.shape.first,
                                  valid=valid, cache_valid=cache_valid)
        x = self.attend_out(x.flatten(1))
        mix, residual = self._normed(x, residual, self.norm_mix, self.mix)
        x = gated_scan_step(*mix.chunk(2, -1), state)
        return self.mix_out(x), residual


class SplatRefiner(nn.Module):
    """Predicts updates of Gaussians of one SH degree (see the module's text).
    The output layer starts at zero, so an untrained refiner changes nothing."""

    def __init__(self, sh_degree: int = 0, shape: RefinerShape = RefinerShape(), device="cuda"):
        super().__init__()
        if shape.width % shape.heads or shape.heads % shape.kv_heads:
            raise ValueError(f"width, heads and kv_heads do not divide: {shape}")
        self.sh_degree, self.shape = sh_degree, shape
        self.features = 11 + 3 * (sh_degree + 1) ** 2
        self.scene = nn.Parameter(0.02 * torch.randn(shape.first, shape.width, device=device))
        self.embed = nn.Linear(self.features, shape.width, device=device)
        self.blocks = nn.ModuleList(_Block(shape, device) for _ in range(shape.blocks))
        self.norm = nn.Parameter(torch.ones(shape.width, device=device, dtype=torch.bfloat16))
        self.head = nn.Linear(shape.width, self.features, device=device)
        nn.init.zeros_(self.head.weight)
        nn.init.zeros_(self.head.bias)

    def quantize(self) -> None:
        """Switches the products behind a norm to 8 bits for calls without
        gradients. Their weights are rounded here, and again by the first such call
        after they have changed in place; training goes on in bfloat16, and what
        ``state_dict`` saves is the bfloat16 weights."""
        for block in self.blocks:
            block.qkv.quantize()
            block.mix.quantize()

    def _features(self, splats: GaussianSplat) -> torch.Tensor:
        features = torch.cat([getattr(splats, name).flatten(1) for name in _NAMES], 1)
        if features.shape[1] != self.features:
            raise ValueError(f"a refiner of SH degree {self.sh_degree} cannot take splats with "
                             f"{features.shape[1]} parameters each")
        return features

    def _update(self, x, residual):
        # Over the width: an optimizer step that moves every weight by its learning
        # rate then moves a splat's parameters by about as much.
        y, _ = rms_norm(x, self.norm, residual)
        return self.head(y.float()) / self.shape.width

    def forward(self, scenes: Sequence[GaussianSplat]) -> list[dict[str, torch.Tensor]]:
        """The refined parameters of each scene (a dict of mean, rotation, scale,
        opacity, color), differentiable in the refiner and the scenes."""
        first, tokens, alive, orders = self.shape.first, [], [], []
        for splats in scenes:
            features = self._features(splats)
            order = morton_order(splats.mean)
            orders.append((features, order))
            tokens += [self.scene, self.embed(features[order])]
            alive += [torch.ones(first, dtype=torch.bool, device=order.device),
                      _alive(splats)[order]]
        packed = PackedSequences([first + len(order) for _, order in orders],
                                 device=self.scene.device)
        residual, valid = torch.cat(tokens), torch.cat(alive)
        x = torch.zeros(residual.shape, dtype=torch.bfloat16, device=residual.device)
        for block in self.blocks:
            x, residual = block(x, residual, packed, valid)
        update = self._update(x, residual)
        refined, at = [], 0
        for features, order in orders:
            rows = update[at + first:at + first + len(order)]
            refined.append(self._unpack(features.index_add(0, order, rows)))
            at += first + len(order)
        return refined

    def _unpack(self, features: torch.Tensor) -> dict[str, torch.Tensor]:
        parts = features.split([3, 4, 3, 1, self.features - 11], 1)
        out = {name: part.contiguous() for name, part in zip(_NAMES, parts)}
        out["color"] = out["color"].unflatten(1, (-1, 3))
        return out

    # ------------------------------------------------------------- streams

    @torch.no_grad()
    def stream(self, batch: int) -> dict:
        """The state of ``batch`` streams that have seen the scene tokens."""
        if self.shape.right:
            raise ValueError("only a causal refiner (right=0) takes splats one by one")
        s, device = self.shape, self.scene.device
        alive = torch.zeros(batch, s.first + s.left + 1, dtype=torch.bool, device=device)
        state = {"length": 0, "alive": alive, "blocks": [
            (window_cache(batch, s.left, s.first, s.kv_heads, block.dim, device=device),
             torch.zeros(batch, s.width, device=device)) for block in self.blocks]}
        for token in self.scene:
            self._advance(token.expand(batch, -1).contiguous(), None, state)
        return state

    def _advance(self, residual, alive, state):
        positions = torch.full((len(residual),), state["length"], dtype=torch.int64,
                               device=residual.device)
        x = torch.zeros(residual.shape, dtype=torch.bfloat16, device=residual.device)
        for block, (cache, scan) in zip(self.blocks, state["blocks"]):
            x, residual = block.step(x, residual, positions, cache, scan, alive, state["alive"])
        state["length"] += 1
        return x, residual

    @torch.no_grad()
    def step(self, splats: GaussianSplat, state: dict) -> dict[str, torch.Tensor]:
        """The refined parameters of one new splat of each stream (``splats`` holds
        one a stream), given those that came before it; advances ``state``."""
        features = self._features(splats)
        x, residual = self._advance(self.embed(features), _alive(splats), state)
        return self._unpack(features + self._update(x, residual))
