"""The typed operators of an MLP block: `linear` (a matrix product with bias,
activation and residual in its epilogue) and `layer_norm`, differentiable, in
fp32, bf16 or fp16 (include/sgnn.h, "Typed operators").

They are what a block of the reference is made of (build_mlp + LayerNorm +
residual, graph_network.py:7-45, :86-96, :176), for any sizes, leading
dimensions and alignment.  autograd.mlp runs the modules that the fp32 ReLU
chain there does not cover on them: 16-bit parameters and other activations.

Forward and backward run in libsgnn_hip.so on the caller's stream; every sum
and statistic is held in fp32 and a 16-bit result is rounded once.  Everything
is deterministic.  Backward passes are differentiable once; forward-mode
derivatives are refused.  To capture a backward pass into a graph, take the
gradients with torch.autograd.grad (it needs no accumulation node of a leaf,
which belongs to the stream that first used it).
Checks, allocation and the autograd nodes are csrc/torch_ops.cpp.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._hip import ACTIVATIONS, torch_ops


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual.

    x [..., K], weight [N, K] (nn.Linear's layout), bias [N], residual [..., N]; one
    type for all.  activation: "none", "relu", "gelu" (erf), "gelu_tanh" or "silu".
    Differentiable in x, weight, bias and residual."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return torch_ops().linear(x, weight, bias, residual, act)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias (+ residual) over the last dimension
    (biased variance, as nn.LayerNorm).

    x [..., W] (W up to 2^23); weight and bias [W] of x's type or float32 (both of one); residual
    of x's shape and type.  Differentiable in x, weight, bias and residual."""
    return torch_ops().layer_norm(x, weight, bias, residual, eps)
