"""SwiGLU feed-forward: down(silu(gate(x)) * up(x)).

gate and up run as one product (src/torchinferno/models/llama3/tensor_parallel.py:4398, 3170 concatenates
them, gate first); here their rows are interleaved instead (row 2i = gate i, row 2i + 1 = up i), so that one
tile of the product holds both and the few-rows kernel of a decode step can apply the activation in its
epilogue;
silu(g) = g / (1 + exp(-g)) with g in fp32
(src/torchinferno/kernels/triton_ops.py:29-32); no bias
(src/torchinferno/models/llama3/pipeline.py:247-250).
"""
from __future__ import annotations

from typing import Mapping

import torch

from torchinferno_b200.kernels import ops
from torchinferno_b200.kernels.block_scaled import BlockScaledWeight
from torchinferno_b200.kernels.gemm import LinearWeight, gated_projection, linear, linear_swiglu, projection
from torchinferno_b200.parts.base import FeedForward, LayerContext, WeightSpec, register_part


class SwiGLUFeedForward(FeedForward):
    def __init__(self, *, hidden_size: int, intermediate_size: int, gate_name: str = "gate_proj.weight",
                 up_name: str = "up_proj.weight", down_name: str = "down_proj.weight",
                 dtype: torch.dtype, device: torch.device) -> None:
        super().__init__(dtype=dtype, device=device)
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self.names = (gate_name, up_name, down_name)
        self.gate_up_weight: LinearWeight | BlockScaledWeight | None = None
        self.down_weight: LinearWeight | BlockScaledWeight | None = None

    def weight_specs(self) -> list[WeightSpec]:
        g, u, d = self.names
        return [WeightSpec(g, (self.intermediate_size, self.hidden_size), block_scaled=True),
                WeightSpec(u, (self.intermediate_size, self.hidden_size), block_scaled=True),
                WeightSpec(d, (self.hidden_size, self.intermediate_size), block_scaled=True)]

    def bind(self, weights: Mapping[str, torch.Tensor]) -> None:
        g, u, d = self.names
        self.gate_up_weight, self.down_weight = gated_projection(weights[g], weights[u]), projection(weights[d])

    def forward(self, x: torch.Tensor, ctx: LayerContext) -> torch.Tensor:
        return linear(linear_swiglu(x, self.gate_up_weight), self.down_weight)


register_part("feed_forward", "swiglu", SwiGLUFeedForward)


class DenseFeedForward(FeedForward):
    """down(act(up(x))) without a gate: act = relu squared (``relu2``; the square in fp32).  No biases."""

    def __init__(self, *, hidden_size: int, intermediate_size: int, activation: str = "relu2", up_name: str = "up",
                 down_name: str = "down", dtype: torch.dtype, device: torch.device) -> None:
        super().__init__(dtype=dtype, device=device)
        if activation != "relu2":
            raise ValueError(f"unknown activation {activation!r}; known: ['relu2']")
        self.hidden_size, self.intermediate_size, self.activation = hidden_size, intermediate_size, activation
        self.names = (up_name, down_name)
        self.up_weight: LinearWeight | BlockScaledWeight | None = None
        self.down_weight: LinearWeight | BlockScaledWeight | None = None

    def weight_specs(self) -> list[WeightSpec]:
        u, d = self.names
        return [WeightSpec(u, (self.intermediate_size, self.hidden_size), std=self.hidden_size ** -0.5, block_scaled=True),
                WeightSpec(d, (self.hidden_size, self.intermediate_size), std=self.intermediate_size ** -0.5, block_scaled=True)]

    def bind(self, weights: Mapping[str, torch.Tensor]) -> None:
        u, d = self.names
        self.up_weight, self.down_weight = projection(weights[u]), projection(weights[d])

    def forward(self, x: torch.Tensor, ctx: LayerContext) -> torch.Tensor:
        hidden = linear(x, self.up_weight)
        return linear(ops.relu_squared(hidden, hidden), self.down_weight)


register_part("feed_forward", "dense", DenseFeedForward)
