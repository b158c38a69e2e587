"""Orthogonalised updates of weight matrices: `newton_schulz` (include/sgnn.h,
sgnn_newton_schulz)."""
from __future__ import annotations

from typing import List, Sequence, Tuple, Union

import torch

from ._hip import DTYPES, SgnnMatrix, check, lib, require_gpu_tensor, stream_ptr
from .functional import _on_device, _ptr, _workspace

QUINTIC = (3.4445, -4.7750, 2.0315)
_MAX_DIM = 2 ** 31 - 1


def _matrices(ins: Sequence[torch.Tensor], outs: Sequence[torch.Tensor]):
    """The host array of sgnn_matrix over [m, n] and [b, m, n] tensors with unit column stride."""
    views = []
    for g, o in zip(ins, outs):
        m, n = g.shape[-2:]
        size = g.element_size()
        for i in range(g.shape[0] if g.dim() == 3 else 1):
            step = (i * g.stride(0), i * o.stride(0)) if g.dim() == 3 else (0, 0)
            views.append((g.data_ptr() + size * step[0], o.data_ptr() + size * step[1], max(g.stride(-2), n),
                          max(o.stride(-2), n), m, n))
    mats = (SgnnMatrix * len(views))()
    for t, v in zip(mats, views):
        t.in_, t.out, t.ld_in, t.ld_out, t.rows, t.cols = v
    return mats


def newton_schulz(g: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5,
                  coefficients: Tuple[float, float, float] = QUINTIC,
                  eps: float = 1e-7) -> Union[torch.Tensor, List[torch.Tensor]]:
    """The orthogonalised g: X = g / (|g|_F + eps), then `steps` times
    X <- a X + (b X X^T + c (X X^T)^2) X with (a, b, c) = coefficients.

    g: a matrix [m, n], a batch [b, m, n], or a sequence of these (of one type and
    device; any shapes: matrices of one shape next to each other share launches).
    Returns new tensors of g's shapes and type.  Not differentiable."""
    single = isinstance(g, torch.Tensor)
    ins = [g] if single else list(g)
    a, b, c = (float(v) for v in coefficients)
    if steps < 0 or not eps >= 0.0:
        raise ValueError(f"newton_schulz: steps {steps}, eps {eps}")
    for t in ins:
        require_gpu_tensor(t, "g")
        if t.dtype not in DTYPES or t.dtype != ins[0].dtype or t.device != ins[0].device:
            raise ValueError(f"newton_schulz: {t.dtype} on {t.device} next to {ins[0].dtype} on {ins[0].device} "
                             "(float32, bfloat16 or float16, one for all)")
        if t.dim() not in (2, 3) or max(t.shape[-2:]) > _MAX_DIM:
            raise ValueError(f"newton_schulz: a matrix [m, n] or a batch [b, m, n], got {tuple(t.shape)}")
    with torch.no_grad():
        ins = [t if t.stride(-1) == 1 and t.stride(-2) >= t.shape[-1] else t.contiguous() for t in ins]
        outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in ins]
        mats = _matrices(ins, outs)
        if len(mats):
            L, like = lib(), ins[0]
            nws = L.sgnn_newton_schulz_workspace_bytes(mats, len(mats))
            ws = _workspace(nws, like)
            with _on_device(like.device):
                check(L.sgnn_newton_schulz(DTYPES[like.dtype], mats, len(mats), int(steps), a, b, c, float(eps),
                                           _ptr(ws), nws, stream_ptr(like.device)), "sgnn_newton_schulz")
    return outs[0] if single else outs
