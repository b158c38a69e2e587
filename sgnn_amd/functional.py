"""The typed operators of an MLP block: `linear` (a matrix product with bias,
activation and residual in its epilogue) and `layer_norm`, differentiable, in
fp32, bf16 or fp16 (include/sgnn.h, "Typed operators").

They are what a block of the reference is made of (build_mlp + LayerNorm +
residual, graph_network.py:7-45, :86-96, :176), for any sizes, leading
dimensions and alignment.  autograd.mlp runs the modules that the fp32 ReLU
chain there does not cover on them: 16-bit parameters and other activations.

Forward and backward run in libsgnn_hip.so on the caller's stream; every sum
and statistic is held in fp32 and a 16-bit result is rounded once.  Everything
is deterministic.  Backward passes are differentiable once.  To capture one
into a graph, take the gradients with torch.autograd.grad (it needs no
accumulation node of a leaf, which belongs to the stream that first used it).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ._hip import ACTIVATIONS, DTYPES, check, lib, require_gpu_tensor, stream_ptr


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _operand(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A GPU tensor of a supported type (and of `like`'s type and device)."""
    require_gpu_tensor(t, name)
    if like is None:
        if t.dtype not in DTYPES:
            raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    elif t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {like.dtype} on {like.device}")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, width] with unit column stride and rows that do not overlap (copied only where it is not)."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1] or t.is_contiguous():
        return t
    return t.contiguous()


def _ld(t: torch.Tensor) -> int:
    """The leading dimension of _rows' result (a single row's stride says nothing)."""
    return max(t.stride(0), t.shape[1])


def _workspace(nbytes: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


class _on_device:
    """The tensor's device made current for the launch (where it is not)."""

    def __init__(self, device: torch.device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


# ----------------------------------------------------------------------------- linear
def _linear_forward(x, weight, bias, residual, act: int, need_z: bool):
    M, K = x.shape
    N = weight.shape[0]
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    z = torch.empty(M, N, dtype=x.dtype, device=x.device) if need_z else None
    if M == 0 or N == 0:
        return y, z
    L, dt = lib(), DTYPES[x.dtype]
    nws = L.sgnn_linear_workspace_bytes(dt, M, N, K)
    ws = _workspace(nws, x)
    with _on_device(x.device):
        check(L.sgnn_linear(dt, M, N, K, x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight), _ptr(bias), act,
                            _ptr(residual), _ld(residual) if residual is not None else 0, _ptr(z), y.data_ptr(), N,
                            _ptr(ws), nws, stream_ptr(x.device)), "sgnn_linear")
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int):
        # the slope of ReLU shows in y where no residual was added to it; the others need z itself
        need_z = act > 1 or (act == 1 and residual is not None)
        y, z = _linear_forward(x, weight, bias, residual, act, need_z)
        ctx.act, ctx.has_bias = act, bias is not None
        ctx.save_for_backward(x, weight, y if act == 1 and z is None else z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dres = dy if need_r else None
        M, K = x.shape
        N = weight.shape[0]
        dy = _rows(dy)
        dx = torch.empty(M, K, dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty(N, K, dtype=x.dtype, device=x.device) if need_w else None
        db = torch.empty(N, dtype=x.dtype, device=x.device) if need_b else None
        if need_x or need_w or need_b:
            L, dt = lib(), DTYPES[x.dtype]
            nws = L.sgnn_linear_bwd_workspace_bytes(dt, M, N, K, ctx.act)
            ws = _workspace(nws, x)
            with _on_device(x.device):
                check(L.sgnn_linear_bwd(dt, M, N, K, dy.data_ptr(), _ld(dy), _ptr(z), ctx.act, x.data_ptr(), _ld(x),
                                        weight.data_ptr(), _ld(weight), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nws,
                                        stream_ptr(x.device)), "sgnn_linear_bwd")
        return dx, dw, db, dres, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual.

    x [..., K], weight [N, K] (nn.Linear's layout), bias [N], residual [..., N]; one
    type for all.  activation: "none", "relu", "gelu" (erf), "gelu_tanh" or "silu".
    Differentiable in x, weight, bias and residual; a 16-bit type keeps the
    pre-activation values for the backward pass in that type."""
    _operand(x, "x")
    _operand(weight, "weight", x)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    N = weight.shape[0]
    shape = (*x.shape[:-1], N)
    if bias is not None:
        _operand(bias, "bias", x)
        if tuple(bias.shape) != (N,):
            raise ValueError(f"linear: bias {tuple(bias.shape)} does not fit weight {tuple(weight.shape)}")
        bias = bias.contiguous()
    if residual is not None:
        _operand(residual, "residual", x)
        if tuple(residual.shape) != shape:
            raise ValueError(f"linear: residual {tuple(residual.shape)}, the output is {shape}")
        residual = _rows(residual)
    act = ACTIVATIONS[activation]
    args = (_rows(x), _rows(weight), bias, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        y = _Linear.apply(*args, act)
    else:
        y = _linear_forward(*args, act, False)[0]
    return y if len(shape) == 2 else y.view(shape)


# ----------------------------------------------------------------------------- layer norm
def _norm_forward(x, weight, bias, residual, eps: float, need_stats: bool):
    n, width = x.shape
    y = torch.empty(n, width, dtype=x.dtype, device=x.device)
    stats = torch.empty(2, n, dtype=torch.float32, device=x.device) if need_stats else None
    if n:
        affine = weight if weight is not None else bias
        dt = DTYPES[x.dtype]
        with _on_device(x.device):
            check(lib().sgnn_norm(dt, DTYPES[affine.dtype] if affine is not None else dt, x.data_ptr(), _ld(x), n,
                                  width, _ptr(weight), _ptr(bias), _ptr(residual),
                                  _ld(residual) if residual is not None else 0, eps, y.data_ptr(), _ptr(stats),
                                  stats.data_ptr() + 4 * n if need_stats else None, stream_ptr(x.device)), "sgnn_norm")
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps: float):
        y, stats = _norm_forward(x, weight, bias, residual, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_type = bias.dtype if bias is not None else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dres = dy if need_r else None
        n, width = x.shape
        dy = _rows(dy)
        dx = torch.empty(n, width, dtype=x.dtype, device=x.device) if need_x else None
        wtype = weight.dtype if weight is not None else ctx.bias_type or x.dtype
        dw = torch.empty(width, dtype=wtype, device=x.device) if need_w else None
        db = torch.empty(width, dtype=wtype, device=x.device) if need_b else None
        if need_x or need_w or need_b:
            L = lib()
            nws = L.sgnn_norm_bwd_workspace_bytes(n, width) if need_w or need_b else 0
            ws = _workspace(nws, x)
            with _on_device(x.device):
                check(L.sgnn_norm_bwd(DTYPES[x.dtype], DTYPES[wtype], dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x),
                                      stats.data_ptr(), stats.data_ptr() + 4 * n, _ptr(weight), n, width, _ptr(dx),
                                      _ptr(dw), _ptr(db), _ptr(ws), nws, stream_ptr(x.device)), "sgnn_norm_bwd")
        return dx, dw, db, dres, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias (+ residual) over the last dimension
    (biased variance, as nn.LayerNorm).

    x [..., W]; weight and bias [W] of x's type or float32 (both of one); residual
    of x's shape and type.  Differentiable in x, weight, bias and residual."""
    _operand(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x {tuple(x.shape)} has no last dimension to normalise over")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps {eps}")
    width = x.shape[-1]
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        require_gpu_tensor(t, name)
        if t.device != x.device or t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {x.dtype} or float32 on {x.device}")
        if tuple(t.shape) != (width,):
            raise ValueError(f"layer_norm: {name} {tuple(t.shape)}, x is {tuple(x.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    if residual is not None:
        _operand(residual, "residual", x)
        if residual.shape != x.shape:
            raise ValueError(f"layer_norm: residual {tuple(residual.shape)}, x is {tuple(x.shape)}")
        residual = _rows(residual)
    shape = x.shape
    args = (_rows(x), weight.contiguous() if weight is not None else None,
            bias.contiguous() if bias is not None else None, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        y = _LayerNorm.apply(*args, eps)
    else:
        y = _norm_forward(*args, eps, False)[0]
    return y if len(shape) == 2 else y.view(shape)
