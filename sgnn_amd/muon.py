"""Orthogonalised updates of weight matrices: `newton_schulz` (include/sgnn.h,
sgnn_newton_schulz)."""
from __future__ import annotations

from typing import List, Sequence, Tuple, Union

import torch

from ._hip import torch_ops

QUINTIC = (3.4445, -4.7750, 2.0315)


def newton_schulz(g: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5,
                  coefficients: Tuple[float, float, float] = QUINTIC,
                  eps: float = 1e-7) -> Union[torch.Tensor, List[torch.Tensor]]:
    """The orthogonalised g: X = g / (|g|_F + eps), then `steps` times
    X <- a X + (b X X^T + c (X X^T)^2) X with (a, b, c) = coefficients.

    g: a matrix [m, n], a batch [b, m, n], or a sequence of these (of one type and
    device; any shapes: matrices of one shape next to each other share launches).
    Returns new tensors of g's shapes and type.  Not differentiable."""
    if isinstance(g, torch.Tensor):
        return torch_ops().newton_schulz([g], steps, *coefficients, eps)[0]
    return torch_ops().newton_schulz(list(g), steps, *coefficients, eps)
