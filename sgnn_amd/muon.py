"""The Muon optimiser: `newton_schulz` orthogonalises the updates of weight
matrices (include/sgnn.h, sgnn_newton_schulz), `Muon` applies them to a
FlatParams buffer, with the fused Adam step for every other parameter.

The reference trains with torch.optim.Adam (train.py:199); this is an
alternative behind the same Trainer (`optimizer="muon"`).
"""
from __future__ import annotations

from typing import List, Sequence, Tuple, Union

import torch
import torch.nn as nn

from ._hip import SgnnMuonSeg, check, lib, stream_ptr, torch_ops

QUINTIC = (3.4445, -4.7750, 2.0315)
MIN_SIDE = 16   # Linear weights narrower than this (raw features in, positions out) keep Adam


def newton_schulz(g: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5,
                  coefficients: Tuple[float, float, float] = QUINTIC, eps: float = 1e-7,
                  out: Union[None, torch.Tensor, Sequence[torch.Tensor]] = None) -> Union[torch.Tensor, List[torch.Tensor]]:
    """The orthogonalised g: X = g / (|g|_F + eps), then `steps` times
    X <- a X + (b X X^T + c (X X^T)^2) X with (a, b, c) = coefficients.

    g: a matrix [m, n], a batch [b, m, n], or a sequence of these (of one type and
    device; any shapes: matrices of one shape next to each other share launches).
    Returns new tensors of g's shapes and type, or writes `out` (likewise; rows of
    unit stride).  A matrix of `out` may be its own g; it may overlap nothing else
    of g or `out`.  Not differentiable."""
    single = isinstance(g, torch.Tensor)
    outs = [] if out is None else [out] if single else list(out)
    got = torch_ops().newton_schulz([g] if single else list(g), outs, steps, *coefficients, eps)
    return got[0] if single else got


def hidden_matrices(module: nn.Module) -> List[nn.Parameter]:
    """The weights Muon orthogonalises: those of nn.Linear with at least MIN_SIDE rows and columns."""
    return [m.weight for m in module.modules() if isinstance(m, nn.Linear) and min(m.weight.shape) >= MIN_SIDE]


class Muon:
    """One step: m = momentum m + grad, u = grad + momentum m (nesterov; else m),
    W -= lr (0.2 sqrt(max(rows, cols)) newton_schulz(u) + weight_decay W) for the
    hidden matrices of `module` -- the factor gives the update Adam's typical root
    mean square, 0.2, so that both share one `lr` and schedule -- and the fused Adam
    step for the other parameters.  `lr` may be changed between steps."""

    def __init__(self, flat, module: nn.Module, lr: float, momentum: float = 0.95, nesterov: bool = True,
                 steps: int = 5, weight_decay: float = 0.0, betas=(0.9, 0.999), eps: float = 1e-8):
        self.flat, self.lr, self.momentum, self.nesterov = flat, lr, momentum, nesterov
        self.steps, self.weight_decay, self.betas, self.eps = steps, weight_decay, betas, eps
        chosen = {flat.offsets[id(p)][0] for p in hidden_matrices(module)}
        self.is_matrix = [off in chosen for off, _, _ in flat.order]
        self.exp_avg = torch.zeros_like(flat.param)      # the matrices' momentum, the others' first moment
        self.exp_avg_sq = torch.zeros_like(flat.param)
        self.update = torch.zeros_like(flat.param)
        self.step_count = 0
        segs = (SgnnMuonSeg * len(flat.order))()
        mats = []
        for s, m, (off, n, shape) in zip(segs, self.is_matrix, flat.order):
            s.offset, s.numel, s.matrix = off, n, int(m)
            s.scale = 0.2 * max(shape) ** 0.5 if m else 0.0
            if m:
                mats.append(self.update[off:off + n].view(shape))
        self.mats = sorted(mats, key=lambda t: tuple(t.shape))   # one shape next to each other
        self.segs = torch.frombuffer(bytearray(segs), dtype=torch.uint8).to(flat.param.device)

    def step(self) -> None:
        self.step_count += 1
        f, L = self.flat, lib()
        n, s = len(f.order), stream_ptr(f.param.device)
        check(L.sgnn_muon_moments(self.segs.data_ptr(), n, f.param.data_ptr(), f.grad.data_ptr(),
                                  self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.update.data_ptr(),
                                  float(self.momentum), int(self.nesterov), float(self.lr), float(self.betas[0]),
                                  float(self.betas[1]), float(self.eps), self.step_count, s), "sgnn_muon_moments")
        if not self.mats:
            return
        newton_schulz(self.mats, steps=self.steps, out=self.mats)
        check(L.sgnn_muon_apply(self.segs.data_ptr(), n, f.param.data_ptr(), self.update.data_ptr(), float(self.lr),
                                float(self.weight_decay), s), "sgnn_muon_apply")

    def state_dict(self) -> dict:
        """torch.optim's layout: per parameter (module.parameters() order) `step` and
        `momentum_buffer` (matrices) or `exp_avg` / `exp_avg_sq` (the others)."""
        f = self.flat
        group = {"lr": self.lr, "momentum": self.momentum, "nesterov": self.nesterov, "steps": self.steps,
                 "weight_decay": self.weight_decay, "betas": tuple(self.betas), "eps": self.eps,
                 "params": list(range(len(f.order)))}
        state = {}
        if self.step_count > 0:
            for i, (m, (off, n, shape)) in enumerate(zip(self.is_matrix, f.order)):
                of = lambda t: t[off:off + n].view(shape).detach().clone()
                state[i] = {"step": torch.tensor(float(self.step_count))}
                state[i].update({"momentum_buffer": of(self.exp_avg)} if m else
                                {"exp_avg": of(self.exp_avg), "exp_avg_sq": of(self.exp_avg_sq)})
        return {"state": state, "param_groups": [group]}

    def load_state_dict(self, sd: dict) -> None:
        f = self.flat
        groups = sd["param_groups"]
        if len(groups) != 1 or len(groups[0]["params"]) != len(f.order) or "momentum" not in groups[0]:
            raise ValueError(f"not the state of a Muon optimiser over {len(f.order)} parameters in one group")
        g = groups[0]
        parts = []
        for slot, pid in enumerate(g["params"]):
            st = sd["state"].get(pid)
            if st is None:
                continue
            keys = {"momentum_buffer": self.exp_avg} if self.is_matrix[slot] else {"exp_avg": self.exp_avg,
                                                                                   "exp_avg_sq": self.exp_avg_sq}
            off, n, shape = f.order[slot]
            for k, to in keys.items():
                if k not in st or tuple(st[k].shape) != tuple(shape):
                    raise ValueError(f"optimizer state {pid}: no {k} of shape {tuple(shape)}")
                parts.append((to[off:off + n], st[k], int(float(st["step"]))))
        counts = {c for _, _, c in parts}
        if len(counts) > 1:
            raise ValueError(f"parameters at different steps {sorted(counts)}: one fused update cannot resume them")
        with torch.no_grad():
            self.exp_avg.zero_()
            self.exp_avg_sq.zero_()
            for to, value, _ in parts:
                to.copy_(value.reshape(-1))
        self.lr, self.momentum, self.nesterov = float(g["lr"]), float(g["momentum"]), bool(g["nesterov"])
        self.steps, self.weight_decay = int(g["steps"]), float(g["weight_decay"])
        self.betas, self.eps = tuple(g["betas"]), float(g["eps"])
        self.step_count = counts.pop() if counts else 0


def make_optimizer(name: str, flat, module: nn.Module, lr: float):
    """The optimiser of a Trainer: "adam" (the reference's) or "muon"."""
    if name == "adam":
        from .training import Adam
        return Adam(flat, lr)
    if name == "muon":
        return Muon(flat, module, lr)
    raise ValueError(f'optimizer must be "adam" or "muon", got {name!r}')
