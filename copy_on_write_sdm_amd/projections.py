"""A stack's attention blocks and MLPs from their weights, over ``linear``: the
callables that ``PagedAttention`` and the stack's prefill and decode take.

The reference runs these in its model (CausalSelfAttention and ResidualMLP,
copy_on_write_sdm/model.py:25-189).  What norms a block's input stays the
caller's.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Mapping

import torch

from .linear import linear

Norm = Callable[[torch.Tensor], torch.Tensor]


@dataclass
class ResidualMLP:
    """tokens + down(activation(up(norm(tokens)))), weights [out, in] and
    biases as ``nn.Linear`` holds them; ``norm`` is the block's input norm."""

    up_weight: torch.Tensor
    down_weight: torch.Tensor
    up_bias: torch.Tensor | None = None
    down_bias: torch.Tensor | None = None
    activation: str | None = "gelu"
    norm: Norm | None = None

    @torch.no_grad()
    def __call__(self, tokens: torch.Tensor) -> torch.Tensor:
        x = tokens if self.norm is None else self.norm(tokens)
        inner = linear(x, self.up_weight, self.up_bias, activation=self.activation)
        return linear(inner, self.down_weight, self.down_bias, residual=tokens)


@dataclass
class AttentionLayer:
    """One attention block's weights, [out, in] as ``nn.Linear`` holds them:
    the query's, key's and value's projections as one matrix of (heads + 2
    kv_heads) * head_width rows in that order, and the output projection.
    ``norm`` is the block's input norm, ``tail`` what follows its residual add
    (a ``ResidualMLP``)."""

    input_weight: torch.Tensor
    output_weight: torch.Tensor
    input_bias: torch.Tensor | None = None
    output_bias: torch.Tensor | None = None
    norm: Norm | None = None
    tail: Callable[[torch.Tensor], torch.Tensor] | None = None


class AttentionProjections:
    """``project`` and ``finish`` of a ``PagedAttention`` from its layers'
    weights, by the layers' positions in the layout."""

    def __init__(self, layers: Mapping[int, AttentionLayer], *, heads: int, kv_heads: int,
                 head_width: int):
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
            raise ValueError("query heads must be a multiple of the key heads")
        rows = (heads + 2 * kv_heads) * head_width
        for at, layer in layers.items():
            if layer.input_weight.ndim != 2 or layer.input_weight.shape[0] != rows:
                raise ValueError(f"attention layer {at}'s input projection must have {rows} rows")
            if layer.output_weight.shape != (layer.input_weight.shape[1], heads * head_width):
                raise ValueError(f"attention layer {at}'s output projection does not match")
        self.layers = dict(layers)
        self.heads, self.kv_heads, self.head_width = heads, kv_heads, head_width

    @torch.no_grad()
    def project(self, layer: int, tokens: torch.Tensor, positions: torch.Tensor
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        weights = self.layers[layer]
        x = tokens if weights.norm is None else weights.norm(tokens)
        heads, end = self.heads, self.heads + self.kv_heads
        x = linear(x, weights.input_weight, weights.input_bias)
        x = x.view(x.shape[0], end + self.kv_heads, self.head_width)
        return x[:, :heads], x[:, heads:end], x[:, end:]

    @torch.no_grad()
    def finish(self, layer: int, tokens: torch.Tensor, mixed: torch.Tensor) -> torch.Tensor:
        weights = self.layers[layer]
        out = linear(mixed.reshape(mixed.shape[0], self.heads * self.head_width),
                     weights.output_weight, weights.output_bias, residual=tokens)
        return out if weights.tail is None else weights.tail(out)
