"""Muon: momentum whose direction is orthogonalised by Newton-Schulz products, over flat buffers.

Every matrix parameter W (a convolution weight counts as ``[cout, everything else]``) takes

    M <- mu M + G,   U = G + mu M (Nesterov) or M,
    W <- (1 - lr wd) W - lr f(shape) NewtonSchulz(U)

with ``f = sqrt(max(1, rows / cols))`` ("original") or ``0.2 sqrt(max(rows, cols))``
("match_rms_adamw"); all other parameters take the SGD of :class:`.fused_sgd.FusedSGD`.  One step
is one native call for the whole model: the matrices share every kernel launch and the last
product of each writes the weights.  On the CPU the same formulas run as torch operations.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from ..ops import native
from ..parallel.flat import FlatModule

ADJUST_LR = ("original", "match_rms_adamw")


def lr_factor(rows: int, cols: int, adjust_lr_fn: str = "original") -> float:
    if adjust_lr_fn == "original":
        return math.sqrt(max(1.0, rows / cols))
    if adjust_lr_fn == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    raise ValueError(f"muon: adjust_lr_fn must be one of {ADJUST_LR}, got {adjust_lr_fn!r}")


def _orthogonalize_cpu(x: torch.Tensor, coef: Sequence[float], eps: float) -> torch.Tensor:
    y = x.double()
    y = (y / (y.square().sum(dim=(-2, -1), keepdim=True).sqrt() + eps)).float()
    tall = y.shape[-2] > y.shape[-1]
    if tall:
        y = y.transpose(-2, -1)
    for k in range(0, len(coef), 3):
        a = y @ y.transpose(-2, -1)
        y = coef[k] * y + (coef[k + 1] * a + coef[k + 2] * (a @ a)) @ y
    return (y.transpose(-2, -1) if tall else y).to(x.dtype)


@torch.no_grad()
def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients=native.NS_COEFFICIENTS,
                  eps: float = 1e-7, precision: Optional[str] = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of ``[..., m, n]`` matrices (:func:`..ops.native.newton_schulz`
    has the formula, the layouts, ``precision`` and what is refused).  An update has no gradient: the
    result is detached from ``x``, and an ``x`` with a forward-mode tangent is refused."""
    if x.is_cuda:
        return native.newton_schulz(x, steps, coefficients, eps, precision)
    native.ns_check(x, eps, precision)
    return _orthogonalize_cpu(x, native.ns_coefficients(steps, coefficients), float(eps))


class Muon:
    """``sgd_params`` names matrix parameters that take SGD all the same (default: the classifier
    ``fc1.weight``, where there is one); parameters of fewer than two dimensions always do."""

    def __init__(self, module_or_flat, lr: float = 0.02, momentum: float = 0.95,
                 weight_decay: float = 0.0, nesterov: bool = True, ns_steps: int = 5,
                 ns_coefficients=native.NS_COEFFICIENTS, eps: float = 1e-7,
                 adjust_lr_fn: str = "original", precision: str = "fp32",
                 sgd_params: Optional[Sequence[str]] = None, sgd_lr: float = 0.1,
                 sgd_momentum: float = 0.9, sgd_weight_decay: float = 1e-4):
        if precision not in native.NS_PRECISIONS:
            raise ValueError(f"muon: precision must be one of {native.NS_PRECISIONS}, got {precision!r}")
        self.flat = module_or_flat if isinstance(module_or_flat, FlatModule) \
            else FlatModule(module_or_flat)
        self.lr, self.momentum, self.weight_decay, self.nesterov = lr, momentum, weight_decay, nesterov
        self.sgd_lr, self.sgd_momentum, self.sgd_weight_decay = sgd_lr, sgd_momentum, sgd_weight_decay
        native.ns_check_eps(eps)
        self.eps, self.precision = float(eps), precision
        self.coefficients = native.ns_coefficients(ns_steps, ns_coefficients)
        self.matrices, self.segments = split_slots(self.flat.slots, sgd_params, adjust_lr_fn)
        self.buf = torch.zeros_like(self.flat.params)
        self.steps = 0
        self._plan = self._workspace = None
        if self.flat.params.is_cuda:
            triples = [self.coefficients[k:k + 3] for k in range(0, len(self.coefficients), 3)]
            self._plan = native.MuonPlan(self.matrices, self.segments, len(triples), triples, self.eps,
                                         precision)
            self._workspace = torch.empty(self._plan.workspace_bytes, dtype=torch.uint8,
                                          device=self.flat.params.device)

    def zero_grad(self) -> None:
        self.flat.zero_grad()

    @torch.no_grad()
    def step(self, grad_scale: float = 1.0) -> None:
        p, g, m = self.flat.params, self.flat.grads, self.buf
        if self._plan is not None:
            native.muon_step_(self._plan, p, g, m, self.lr, self.momentum, self.weight_decay,
                              self.nesterov, self.sgd_lr, self.sgd_momentum, self.sgd_weight_decay,
                              grad_scale, self._workspace)
        else:
            muon_step_cpu_(self, p, g, m, grad_scale)
        self.steps += 1


def split_slots(slots, sgd_params: Optional[Sequence[str]], adjust_lr_fn: str):
    """``(matrices, segments)`` of a flat layout, as :class:`..ops.native.MuonPlan` takes them."""
    named = set(sgd_params) if sgd_params is not None else {"fc1.weight"}
    unknown = named - {s.name for s in slots}
    if sgd_params is not None and unknown:
        raise ValueError(f"muon: sgd_params names no parameter of the model: {sorted(unknown)}")
    matrices, segments = [], []
    for s in slots:
        if s.numel == 0:
            continue
        if len(s.shape) >= 2 and s.name not in named:
            rows = int(s.shape[0])
            cols = s.numel // rows
            matrices.append((s.offset, rows, cols, lr_factor(rows, cols, adjust_lr_fn)))
        else:
            segments.append((s.offset, s.numel))
    return matrices, segments


def muon_step_cpu_(o: Muon, p: torch.Tensor, g: torch.Tensor, m: torch.Tensor, grad_scale: float) -> None:
    for at, rows, cols, factor in o.matrices:
        w, gr, mo = (t[at:at + rows * cols].view(rows, cols) for t in (p, g, m))
        gr = gr * grad_scale
        mo.mul_(o.momentum).add_(gr)
        u = gr + o.momentum * mo if o.nesterov else mo
        w.mul_(1 - o.lr * o.weight_decay).sub_(
            o.lr * factor * _orthogonalize_cpu(u, o.coefficients, o.eps))
    for at, n in o.segments:
        w, gr, mo = (t[at:at + n] for t in (p, g, m))
        mo.mul_(o.sgd_momentum).add_(gr * grad_scale + o.sgd_weight_decay * w)
        w.sub_(o.sgd_lr * mo)
